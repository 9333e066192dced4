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
//
// Bound by memory: 8200 x 4096 bf16 into both operands 32 us (4.2 TB/s), 16384 x 4096 along the rows alone 31 - 50 us (4 - 6.5
// TB/s).  Small matrices are bound by a tile's way through LDS (512 x 3136 fp32, both operands: 100 tiles, 15 us).
#include "ffn_common.h"

struct QuantArgs {
  const void* x;
  long long rows, ldx;
  int cols, col_blocks;
  unsigned char *q, *q_scale, *qt, *qt_scale;
  float* colsum;             // [ceil(rows / 128)][cols]
};

// The tile's 128 x 128 bytes, rows of PITCH in LDS, to eight tiles of an operand: whole 2 KB runs.
template <int PITCH>
__device__ __forceinline__ void write_tiles(const unsigned char* lds, unsigned char* q, long long group0, int groups, long long blocks, long long block) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int u = (int)threadIdx.x + i * 256, g = u >> 7, h = (u >> 6) & 1, l = u & 63;
    const unsigned char* src = lds + (g * 16 + (l & 15)) * PITCH + (l >> 4) * 32 + h * 16;
    const uint2 a = *reinterpret_cast<const uint2*>(src), b = *reinterpret_cast<const uint2*>(src + 8);
    if (g < groups) *reinterpret_cast<uint4*>(q + ((group0 + g) * blocks + block) * 2048 + (u & 127) * 16) = make_uint4(a.x, a.y, b.x, b.y);
  }
}

template <typename T, bool BLOCK>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(QuantArgs a) {
  typedef Raw8<T> R;
  constexpr int PITCH = 136, MAGS = R::MAGS;          // LDS row of a column's 128 bytes, 8-byte aligned
  __shared__ __attribute__((aligned(16))) unsigned char tile[128 * PITCH];
  __shared__ uint32_t wave_max[4][16 * MAGS];
  __shared__ float wave_sum[4][128];
  const int tid = threadIdx.x, wave = tid >> 6, c8 = tid & 15, r8 = tid >> 4;
  const int kb = (int)(blockIdx.x % (unsigned)a.col_blocks), col0 = kb * 128 + c8 * 8;
  const long long mb = blockIdx.x / (unsigned)a.col_blocks, row0 = mb * 128 + r8 * 8;
  const T* X = reinterpret_cast<const T*>(a.x);
  // All eight loads before anything that waits for one: no branch between them but the tile's own (a load behind a branch of
  // its own waits for the one before: eight trips to memory instead of one).
  R v[8];
  if (kb * 128 + 128 <= a.cols) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].load(X + (row0 + i < a.rows ? row0 + i : a.rows - 1) * a.ldx + col0);
  } else {
    const int n = a.cols - col0, first = n > 0 ? col0 : a.cols - 1;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].load_part(X + (row0 + i < a.rows ? row0 + i : a.rows - 1) * a.ldx + first, n > 0 ? (n < 8 ? n : 8) : 1);
    if (n <= 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i].clear();
    }
  }
  if (mb * 128 + 128 > a.rows) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (row0 + i >= a.rows) v[i].clear();
  }

  uint32_t rmax[8], cmax[MAGS], any = 0;
#pragma unroll
  for (int j = 0; j < MAGS; ++j) cmax[j] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    rmax[i] = v[i].template row_mag<false>();
    any = R::mag_max(any, rmax[i]);
#pragma unroll
    for (int j = 0; j < MAGS; ++j) cmax[j] = R::mag_max(cmax[j], v[i].template mag<false>(j));
  }
  if (R::mag_inf(any)) {                              // rare: leave out what is not finite
#pragma unroll
    for (int j = 0; j < MAGS; ++j) cmax[j] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      rmax[i] = v[i].template row_mag<true>();
#pragma unroll
      for (int j = 0; j < MAGS; ++j) cmax[j] = R::mag_max(cmax[j], v[i].template mag<true>(j));
    }
  }
  if (BLOCK) {                                        // one scale for the tile
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = R::mag_max(m, rmax[i]);
    m = R::mag_bits(mag_max16<R>(m));
    m = umax(m, (uint32_t)__shfl_xor((int)m, 16));
    m = umax(m, (uint32_t)__shfl_xor((int)m, 32));
    if ((tid & 63) == 0) wave_max[wave][0] = m;
    __syncthreads();
    m = umax(umax(wave_max[0][0], wave_max[1][0]), umax(wave_max[2][0], wave_max[3][0]));
#pragma unroll
    for (int i = 0; i < 8; ++i) rmax[i] = m;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) rmax[i] = R::mag_bits(mag_max16<R>(rmax[i]));
    if (a.qt) {
#pragma unroll
      for (int j = 0; j < MAGS; ++j) {
        cmax[j] = R::mag_max(cmax[j], (uint32_t)__shfl_xor((int)cmax[j], 16));
        cmax[j] = R::mag_max(cmax[j], (uint32_t)__shfl_xor((int)cmax[j], 32));
        if ((tid & 48) == 0) wave_max[wave][c8 * MAGS + j] = cmax[j];
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < MAGS; ++j) {
        const int c = c8 * MAGS + j;
        cmax[j] = R::mag_max(R::mag_max(wave_max[0][c], wave_max[1][c]), R::mag_max(wave_max[2][c], wave_max[3][c]));
      }
    }
  }
  const long long row_blocks = (a.rows + 127) / 128;
  if (a.q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int sc = block_scale(rmax[i]);
      *reinterpret_cast<uint2*>(tile + (r8 * 8 + i) * PITCH + c8 * 8) = v[i].quant(scale_value(sc));
      if (c8 == 0 && row0 + i < a.rows) a.q_scale[(((long long)(kb >> 2) * a.rows) + row0 + i) * 4 + (kb & 3)] = (unsigned char)sc;
    }
    __syncthreads();
    const long long left = a.rows - mb * 128;
    write_tiles<PITCH>(tile, a.q, mb * 8, left < 128 ? (int)(left + 15) / 16 : 8, a.col_blocks, kb);
    if (a.qt) __syncthreads();
  }
  if (a.qt) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int sc = block_scale(BLOCK ? rmax[0] : R::col_bits(cmax, j));
      *reinterpret_cast<uint2*>(tile + (c8 * 8 + j) * PITCH + r8 * 8) = R::quant_col(v, j, scale_value(sc));
      if (r8 == 0 && col0 + j < a.cols) a.qt_scale[((mb >> 2) * a.cols + col0 + j) * 4 + (mb & 3)] = (unsigned char)sc;
    }
    __syncthreads();
    const int left = a.cols - kb * 128;
    write_tiles<PITCH>(tile, a.qt, (long long)kb * 8, left < 128 ? (left + 15) / 16 : 8, row_blocks, mb);
  }
  if (a.colsum) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i].get(j);
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      if ((tid & 48) == 0) wave_sum[wave][c8 * 8 + j] = s;
    }
    __syncthreads();
    if (tid < 128 && kb * 128 + tid < a.cols)
      a.colsum[mb * a.cols + kb * 128 + tid] = (wave_sum[0][tid] + wave_sum[1][tid]) + (wave_sum[2][tid] + wave_sum[3][tid]);
  }
}

int fp8_quantize_launch(const Fp8QuantJob& j, hipStream_t s) {
  // (a launch holds less than 2^32 threads; many rows of few columns get there within the card's memory)
  const long long tiles = (j.rows + 127) / 128 * ((j.cols + 127ll) / 128);
  PN_CHECK_ARG(tiles < 1ll << 24, "fp8 quantiser: %lld x %d elements are more than one launch takes", j.rows, j.cols);
  const Fp8Operand q = fp8_operand(j.q, j.rows, j.cols), qt = fp8_operand(j.qt, j.cols, j.rows);
  const int col_blocks = (j.cols + 127) / 128;
  QuantArgs a = {j.x, j.rows, j.rows == 1 ? 0 : j.ldx, j.cols, col_blocks, (unsigned char*)q.q, (unsigned char*)q.scale,
                 (unsigned char*)qt.q, (unsigned char*)qt.scale, j.colsum};
  const dim3 grid((unsigned)tiles), wg(256);
  if (j.dtype == PN_DTYPE_F32) {
    if (j.block_rows == 1) hipLaunchKernelGGL((fp8_quantize_kernel<float, false>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL((fp8_quantize_kernel<float, true>), grid, wg, 0, s, a);
  } else {
    if (j.block_rows == 1) hipLaunchKernelGGL((fp8_quantize_kernel<__bf16, false>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL((fp8_quantize_kernel<__bf16, true>), grid, wg, 0, s, a);
  }
  PN_CHECK_LAUNCH("fp8_quantize_kernel");
  return PN_OK;
}

extern "C" size_t pn_fp8_operand_bytes(long long rows, long long cols) { return rows < 0 || cols < 1 ? 0 : fp8_bytes(rows, cols); }

extern "C" int pn_fp8_quantize(int dtype, const void* x, long long rows, int cols, long long ldx, int block_rows, void* q, void* qt,
                               float* colsum, void* stream) {
  PN_CHECK_ARG(dtype == PN_DTYPE_F32 || dtype == PN_DTYPE_BF16, "pn_fp8_quantize: element type %d (fp32 or bf16)", dtype);
  PN_CHECK_ARG(block_rows == 1 || block_rows == 128, "pn_fp8_quantize: blocks of %d rows (1 or 128)", block_rows);
  PN_CHECK_ARG(rows >= 0 && cols >= 1 && rows < (1ll << 40) / cols, "pn_fp8_quantize: %lld x %d elements", rows, cols);
  if (rows == 0) return PN_OK;
  PN_CHECK_ARG(x && (rows == 1 || ldx >= cols), "pn_fp8_quantize: x missing or its row stride below the row length");
  PN_CHECK_ARG(q || qt || colsum, "pn_fp8_quantize: output missing");
  PN_CHECK_ARG((((uintptr_t)q | (uintptr_t)qt) & 255) == 0, "pn_fp8_quantize: operands must be 256-byte aligned");
  return fp8_quantize_launch(Fp8QuantJob{x, dtype, block_rows, rows, ldx, cols, q, qt, colsum}, (hipStream_t)stream);
}

// out[c] = sum of colsum over the row blocks, in a fixed order
__global__ __launch_bounds__(256) void fp8_colsum_kernel(const float* partial, long long blocks, int cols, void* out, int out_dtype) {
  __shared__ float lds[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (long long i = w; i < blocks; i += 4) s += partial[i * cols + c];
  }
  lds[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < cols) {
    s = (lds[0][lane] + lds[1][lane]) + (lds[2][lane] + lds[3][lane]);
    if (out_dtype == PN_DTYPE_F32) reinterpret_cast<float*>(out)[c] = s;
    else reinterpret_cast<__bf16*>(out)[c] = (__bf16)s;
  }
}
int fp8_colsum_launch(const float* partial, long long rows, int cols, int out_dtype, void* out, hipStream_t s) {
  hipLaunchKernelGGL(fp8_colsum_kernel, dim3((cols + 63) / 64), dim3(256), 0, s, partial, (rows + 127) / 128, cols, out, out_dtype);
  PN_CHECK_LAUNCH("fp8_colsum_kernel");
  return PN_OK;
}
