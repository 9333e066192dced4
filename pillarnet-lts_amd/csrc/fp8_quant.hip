// fp32 / bf16 rows -> e4m3 bytes with one power-of-two scale for each block of 128 along the contraction.
//
// scale of a block = 2^e, e the smallest exponent >= -126 with amax <= 448 * 2^e (448: e4m3's largest value), q = x / 2^e
// rounded to nearest even.  A power of two scales without rounding, is one byte (e + 127), and is what the block-scaled
// matrix instruction multiplies by on its own.  amax is taken over the finite elements; infinities and NaN become the
// type's NaN (it has no infinity) and so mark every product they enter.
//
// One 128 x 128 tile per workgroup, read once; from its registers come the bytes along the rows (blocks 1 x 128), along the
// columns (the transposed operand of a weight gradient, blocks 128 x 1), both with one scale for the whole tile
// (BLOCK: weights), and the tile's column sums (bias gradients).
#include "ffn_common.h"

struct QuantArgs {
  const void* x;
  long long rows, ldx;
  int cols;
  unsigned char* q;          // [rows][kp], kp = cols rounded up to 128
  unsigned char* q_scale;    // dwords [ceil(kp / 512)][rows], byte (k block & 3)
  unsigned char* qt;         // [cols][mp], mp = rows rounded up to 128
  unsigned char* qt_scale;   // dwords [ceil(mp / 512)][cols]
  float* colsum;             // [ceil(rows / 128)][cols]
};

// e + 127 of a block with largest finite magnitude `bits` (as an integer: magnitudes order like their bit patterns)
__device__ __forceinline__ int block_scale(uint32_t bits) {
  const int b = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b < 1 ? 1 : b;
}
__device__ __forceinline__ float inv_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }   // 2^(127 - byte)
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

template <typename T, bool BLOCK>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(QuantArgs a) {
  constexpr int PITCH = 136;                          // LDS row of a column's 128 bytes, 8-byte aligned
  __shared__ __attribute__((aligned(16))) unsigned char tile[128 * PITCH];
  __shared__ uint32_t wave_max[4][128];
  __shared__ float wave_sum[4][128];
  const int tid = threadIdx.x, wave = tid >> 6, c8 = tid & 15, r8 = tid >> 4;
  const int kb = blockIdx.x, col0 = kb * 128 + c8 * 8;
  const long long mb = blockIdx.y, row0 = mb * 128 + r8 * 8;
  const T* X = reinterpret_cast<const T*>(a.x);
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) load8(X + (row0 + i) * a.ldx + col0, row0 + i < a.rows ? a.cols - col0 : 0, v[i]);

  uint32_t rmax[8], cmax[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) cmax[j] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    rmax[i] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t m = finite_bits(v[i][j]);
      rmax[i] = umax(rmax[i], m);
      cmax[j] = umax(cmax[j], m);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) rmax[i] = umax(rmax[i], (uint32_t)__shfl_xor((int)rmax[i], o));
  }
  if (BLOCK) {                                        // one scale for the tile
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = umax(m, rmax[i]);
    m = umax(m, (uint32_t)__shfl_xor((int)m, 16));
    m = umax(m, (uint32_t)__shfl_xor((int)m, 32));
    if ((tid & 63) == 0) wave_max[wave][0] = m;
    __syncthreads();
    m = umax(umax(wave_max[0][0], wave_max[1][0]), umax(wave_max[2][0], wave_max[3][0]));
#pragma unroll
    for (int i = 0; i < 8; ++i) rmax[i] = cmax[i] = m;
  } else if (a.qt) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      cmax[j] = umax(cmax[j], (uint32_t)__shfl_xor((int)cmax[j], 16));
      cmax[j] = umax(cmax[j], (uint32_t)__shfl_xor((int)cmax[j], 32));
      if ((tid & 48) == 0) wave_max[wave][c8 * 8 + j] = cmax[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = c8 * 8 + j;
      cmax[j] = umax(umax(wave_max[0][c], wave_max[1][c]), umax(wave_max[2][c], wave_max[3][c]));
    }
  }
  if (a.q) {
    const long long kp = (long long)gridDim.x * 128;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (row0 + i >= a.rows) continue;
      const int sc = block_scale(rmax[i]);
      const float f = inv_scale(sc);
      const uint2 o = make_uint2(pack4(v[i][0] * f, v[i][1] * f, v[i][2] * f, v[i][3] * f),
                                 pack4(v[i][4] * f, v[i][5] * f, v[i][6] * f, v[i][7] * f));
      *reinterpret_cast<uint2*>(a.q + (row0 + i) * kp + col0) = o;
      if (c8 == 0) a.q_scale[(((long long)(kb >> 2) * a.rows) + row0 + i) * 4 + (kb & 3)] = (unsigned char)sc;
    }
  }
  if (a.qt) {
    const long long mp = (long long)gridDim.y * 128;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int sc = block_scale(cmax[j]);
      const float f = inv_scale(sc);
      const uint2 o = make_uint2(pack4(v[0][j] * f, v[1][j] * f, v[2][j] * f, v[3][j] * f),
                                 pack4(v[4][j] * f, v[5][j] * f, v[6][j] * f, v[7][j] * f));
      *reinterpret_cast<uint2*>(tile + (c8 * 8 + j) * PITCH + r8 * 8) = o;
      if (r8 == 0 && col0 + j < a.cols) a.qt_scale[((mb >> 2) * a.cols + col0 + j) * 4 + (mb & 3)] = (unsigned char)sc;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = i * 16 + r8;
      if (kb * 128 + c < a.cols)
        *reinterpret_cast<uint2*>(a.qt + (long long)(kb * 128 + c) * mp + mb * 128 + c8 * 8) =
            *reinterpret_cast<const uint2*>(tile + c * PITCH + c8 * 8);
    }
  }
  if (a.colsum) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i][j];
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      if ((tid & 48) == 0) wave_sum[wave][c8 * 8 + j] = s;
    }
    __syncthreads();
    if (tid < 128 && kb * 128 + tid < a.cols)
      a.colsum[mb * a.cols + kb * 128 + tid] = (wave_sum[0][tid] + wave_sum[1][tid]) + (wave_sum[2][tid] + wave_sum[3][tid]);
  }
}

extern "C" int pn_fp8_quantize(int dtype, const void* x, long long rows, int cols, long long ldx, int block_rows, void* q,
                               void* q_scale, void* qt, void* qt_scale, float* colsum, void* stream) {
  PN_CHECK_ARG(dtype == PN_DTYPE_F32 || dtype == PN_DTYPE_BF16, "pn_fp8_quantize: element type %d (fp32 or bf16)", dtype);
  PN_CHECK_ARG(block_rows == 1 || block_rows == 128, "pn_fp8_quantize: blocks of %d rows (1 or 128)", block_rows);
  PN_CHECK_ARG(rows >= 0 && cols >= 1 && rows <= 65535ll * 128, "pn_fp8_quantize: %lld x %d elements", rows, cols);
  if (rows == 0) return PN_OK;
  PN_CHECK_ARG(x && (rows == 1 || ldx >= cols), "pn_fp8_quantize: x missing or its row stride below the row length");
  PN_CHECK_ARG((q && q_scale) || (qt && qt_scale), "pn_fp8_quantize: output missing");
  PN_CHECK_ARG((!q || q_scale) && (!qt || qt_scale), "pn_fp8_quantize: bytes without scales");
  PN_CHECK_ARG((((uintptr_t)q | (uintptr_t)qt | (uintptr_t)q_scale | (uintptr_t)qt_scale) & 15) == 0,
               "pn_fp8_quantize: outputs must be 16-byte aligned");
  QuantArgs a = {x, rows, ldx, cols, (unsigned char*)q, (unsigned char*)q_scale, (unsigned char*)qt, (unsigned char*)qt_scale, colsum};
  const dim3 grid((cols + 127) / 128, (unsigned)((rows + 127) / 128)), wg(256);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PN_DTYPE_F32) {
    if (block_rows == 1) hipLaunchKernelGGL((fp8_quantize_kernel<float, false>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL((fp8_quantize_kernel<float, true>), grid, wg, 0, s, a);
  } else {
    if (block_rows == 1) hipLaunchKernelGGL((fp8_quantize_kernel<__bf16, false>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL((fp8_quantize_kernel<__bf16, true>), grid, wg, 0, s, a);
  }
  PN_CHECK_LAUNCH("fp8_quantize_kernel");
  return PN_OK;
}

// out[c] = sum of colsum over the row blocks, in a fixed order
__global__ __launch_bounds__(256) void fp8_colsum_kernel(const float* partial, long long blocks, int cols, void* out, int out_dtype) {
  __shared__ float lds[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < cols)
    for (long long i = w; i < blocks; i += 4) s += partial[i * cols + c];
  lds[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < cols) {
    s = (lds[0][lane] + lds[1][lane]) + (lds[2][lane] + lds[3][lane]);
    if (out_dtype == PN_DTYPE_F32) reinterpret_cast<float*>(out)[c] = s;
    else reinterpret_cast<__bf16*>(out)[c] = (__bf16)s;
  }
}
extern "C" int pn_fp8_colsum(const float* partial, long long rows, int cols, int out_dtype, void* out, void* stream) {
  PN_CHECK_ARG(out_dtype == PN_DTYPE_F32 || out_dtype == PN_DTYPE_BF16, "pn_fp8_colsum: output type %d (fp32 or bf16)", out_dtype);
  PN_CHECK_ARG(rows >= 0 && cols >= 1 && out && (partial || rows == 0), "pn_fp8_colsum: null pointer or empty row");
  hipLaunchKernelGGL(fp8_colsum_kernel, dim3((cols + 63) / 64), dim3(256), 0, (hipStream_t)stream, partial, (rows + 127) / 128, cols, out,
                     out_dtype);
  PN_CHECK_LAUNCH("fp8_colsum_kernel");
  return PN_OK;
}
