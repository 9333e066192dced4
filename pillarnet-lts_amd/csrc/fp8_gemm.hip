// out[m][n] = act(sum over k blocks b of 2^(sx[m][b] + sw[n][b]) * sum_{k in b} x[m][k] w[n][k] + bias[n]),  x, w e4m3.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes a whole block of 128 in one instruction, with the two scales as byte operands:
// the blocks' scales cost no vector instruction and the partial sums stay in fp32 accumulators.  The order of k inside a
// block does not matter as long as both operands agree, so a lane simply holds 32 consecutive bytes of its row.
#include "ffn_common.h"

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) float fp8_f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 fp8_bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 fp8_bf16x2;

struct Fp8GemmArgs {
  const unsigned char *x, *w;        // [M][kp], [N][kp]
  const uint32_t *xs, *ws;           // [ceil(kblocks / 4)][M], [..][N]
  long long M;
  int N, kblocks;
  const void* bias;
  int bias_dtype, act, out_dtype;
  void* out;
  long long ldo;
};

__device__ __forceinline__ fp8_f32x4 mfma_fp8(i32x8 a, i32x8 b, fp8_f32x4 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, (int)sa, 0, (int)sb);
}

// eight bytes widened to bf16 and multiplied by their block's scale, both exact
__device__ __forceinline__ fp8_bf16x8 widen8(int lo, int hi, float scale) {
  const fp8_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const fp8_bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return fp8_bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float scale_of(uint32_t word) { return __uint_as_float((word & 0xffu) << 23); }

// 128 x 128 tile, four waves of 64 x 64, one block of 128 per step staged through LDS (16-byte chunks of a row
// exchanged by (row >> 1) & 7, so that the 16 rows a fragment read covers fall on different banks).
template <bool WIDE>
__global__ __launch_bounds__(256) void fp8_gemm_kernel(Fp8GemmArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned char lx[128 * 128], lw[128 * 128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lk = lane >> 4;
  const long long m0 = (long long)blockIdx.x * 128;
  const int n0 = blockIdx.y * 128, wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
  const long long kp = (long long)a.kblocks * 128;
  fp8_f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = fp8_f32x4{0.f, 0.f, 0.f, 0.f};
  for (int kb = 0; kb < a.kblocks; ++kb) {
    uint4 rx[4], rw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int id = tid + i * 256, r = id >> 3, ch = id & 7;
      const long long m = m0 + r < a.M ? m0 + r : a.M - 1;
      const long long n = n0 + r < a.N ? n0 + r : a.N - 1;
      rx[i] = *reinterpret_cast<const uint4*>(a.x + m * kp + kb * 128 + ch * 16);
      rw[i] = *reinterpret_cast<const uint4*>(a.w + n * kp + kb * 128 + ch * 16);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int id = tid + i * 256, r = id >> 3, ch = (id & 7) ^ ((r >> 1) & 7);
      *reinterpret_cast<uint4*>(lx + r * 128 + ch * 16) = rx[i];
      *reinterpret_cast<uint4*>(lw + r * 128 + ch * 16) = rw[i];
    }
    __syncthreads();
    i32x8 fx[4], fw[4];
    uint32_t sx[4], sw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = wm + i * 16 + lr, q = wn + i * 16 + lr;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const i32x4 vx = *reinterpret_cast<const i32x4*>(lx + r * 128 + (((lk * 2 + h) ^ ((r >> 1) & 7)) * 16));
        const i32x4 vw = *reinterpret_cast<const i32x4*>(lw + q * 128 + (((lk * 2 + h) ^ ((q >> 1) & 7)) * 16));
#pragma unroll
        for (int e = 0; e < 4; ++e) { fx[i][h * 4 + e] = vx[e]; fw[i][h * 4 + e] = vw[e]; }
      }
      const long long m = m0 + r < a.M ? m0 + r : a.M - 1;
      const int n = n0 + q < a.N ? n0 + q : a.N - 1;
      sx[i] = a.xs[(long long)(kb >> 2) * a.M + m] >> (8 * (kb & 3));
      sw[i] = a.ws[(long long)(kb >> 2) * a.N + n] >> (8 * (kb & 3));
    }
    if (WIDE) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        fp8_bf16x8 bx[4], bw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bx[i] = widen8(fx[i][2 * e], fx[i][2 * e + 1], scale_of(sx[i]));
          bw[i] = widen8(fw[i][2 * e], fw[i][2 * e + 1], scale_of(sw[i]));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bw[j], bx[i], acc[i][j], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mfma_fp8(fw[j], fx[i], acc[i][j], sw[j], sx[i]);   // D[n][m]
    }
  }
  // lane holds n = 4 * lk .. +3 of m = lr: four consecutive outputs of a row
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long m = m0 + wm + i * 16 + lr;
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + wn + j * 16 + lk * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (n + e >= a.N) continue;
        float v = acc[i][j][e];
        if (a.bias) v += a.bias_dtype == PN_DTYPE_F32 ? reinterpret_cast<const float*>(a.bias)[n + e]
                                                      : (float)reinterpret_cast<const __bf16*>(a.bias)[n + e];
        v = act_f(v, a.act);
        if (a.out_dtype == PN_DTYPE_F32) reinterpret_cast<float*>(a.out)[m * a.ldo + n + e] = v;
        else reinterpret_cast<__bf16*>(a.out)[m * a.ldo + n + e] = (__bf16)v;
      }
    }
  }
}

extern "C" int pn_fp8_gemm(const void* x, const void* x_scale, long long m, const void* w, const void* w_scale, int n, int k,
                           const void* bias, int bias_dtype, int act, int out_dtype, void* out, long long ldo, void* stream) {
  PN_CHECK_ARG(m >= 0 && n >= 1 && k >= 1, "pn_fp8_gemm: %lld x %d x %d", m, n, k);
  PN_CHECK_ARG(act >= PN_ACT_NONE && act <= PN_ACT_GELU, "pn_fp8_gemm: activation %d", act);
  PN_CHECK_ARG((out_dtype == PN_DTYPE_F32 || out_dtype == PN_DTYPE_BF16) && (!bias || bias_dtype == PN_DTYPE_F32 || bias_dtype == PN_DTYPE_BF16),
               "pn_fp8_gemm: output type %d, bias type %d (fp32 or bf16)", out_dtype, bias_dtype);
  if (m == 0) return PN_OK;
  PN_CHECK_ARG(x && x_scale && w && w_scale && out, "pn_fp8_gemm: null pointer");
  PN_CHECK_ARG((((uintptr_t)x | (uintptr_t)w | (uintptr_t)x_scale | (uintptr_t)w_scale) & 15) == 0,
               "pn_fp8_gemm: operands must be 16-byte aligned");
  PN_CHECK_ARG(ldo >= n, "pn_fp8_gemm: output row stride %lld below %d", ldo, n);
  PN_CHECK_ARG(m < (1ll << 31) * 128 && n <= 65535 * 128, "pn_fp8_gemm: too many rows");
  Fp8GemmArgs a = {(const unsigned char*)x, (const unsigned char*)w, (const uint32_t*)x_scale, (const uint32_t*)w_scale, m, n,
                   (k + 127) / 128, bias, bias_dtype, act, out_dtype, out, ldo};
  const dim3 grid((unsigned)((m + 127) / 128), (n + 127) / 128), wg(256);
  if (out_dtype == PN_DTYPE_F32) hipLaunchKernelGGL(fp8_gemm_kernel<true>, grid, wg, 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(fp8_gemm_kernel<false>, grid, wg, 0, (hipStream_t)stream, a);
  PN_CHECK_LAUNCH("fp8_gemm_kernel");
  return PN_OK;
}
