// out[m][n] = act(sum over k blocks b of 2^(sx[m][b] + sw[n][b]) * sum_{k in b} x[m][k] w[n][k] + bias[n]),  x, w e4m3.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes a whole block of 128 in one instruction, with the two scales as byte operands:
// the blocks' scales cost no vector instruction and the partial sums stay in fp32 accumulators.  The order of k inside a
// block does not matter as long as both operands agree, so a lane simply holds 32 bytes of its row as they lie in the operand's tile.
//
// The instruction rounds the products of eight neighbouring k to 16 bits below the largest of them before it adds (measured with
// single pairs of products: 1.4e-5 relative at worst).  That is far below a bf16 result's own rounding and far above an fp32
// result's: for fp32 outputs (WIDE) the same bytes are widened to bf16 and multiplied by v_mfma_f32_16x16x32_bf16.  That is exact down
// to bf16's smallest step, 2^-133: in blocks of an exponent below -124 (no element over 1.1e-35) a value may be off by half of that.
// Measured (from card to card): 8192^3 386 - 436 us into bf16 (2.5 - 2.8 PFLOP/s), 836 - 944 into fp32 (1.2 - 1.3 PFLOP/s, the bf16
// instruction's own bound with the widening beside it); 16384 x 4096 x 8192 with bias and GELU 455 - 470 us; one row of 8192 x 8192 15 us
// (4.4 TB/s).
#include "ffn_common.h"
#include <type_traits>

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef __attribute__((ext_vector_type(4))) float fp8_f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 fp8_bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 fp8_bf16x2;

struct Fp8GemmArgs {
  const unsigned char *x, *w;        // tiles of 2 KB: [ceil(M / 16)][kblocks], [ceil(N / 16)][kblocks]
  const uint32_t *xs, *ws;           // [kquads][x_rows], [kquads][N]
  long long M, x_rows;               // rows of this launch, rows of the operand that they are part of
  int N, kblocks, kquads;            // blocks of 128, words of four scales
  int tiles_m, tiles_n;
  const void* bias;
  int bias_dtype, act, out_dtype;
  void* out;
  long long ldo;
};

__device__ __forceinline__ fp8_f32x4 mfma_fp8(i32x8 a, i32x8 b, fp8_f32x4 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, (int)sa, 0, (int)sb);
}

// eight bytes widened to bf16 and multiplied by their block's scale, both exact down to 2^-133
__device__ __forceinline__ fp8_bf16x8 widen8(int lo, int hi, float scale) {
  const fp8_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const fp8_bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return fp8_bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float scale_of(uint32_t word) { return __uint_as_float((word & 0xffu) << 23); }

// Tile order: workgroups are dealt to the 8 XCDs round robin, so XCD x takes the x-th eighth of the order, and the order
// runs through blocks of 8 x-tiles before the next w-tile: the 32 workgroups of an XCD then share 8 + 4 operand strips in
// its L2 instead of 32 + 1.
struct TileAt { int m, n; };
__device__ __forceinline__ TileAt tile_at(int lin, int tiles_m, int tiles_n) {
  constexpr int G = 8;
  const int group = lin / (G * tiles_n), in = lin - group * G * tiles_n, gm = min(G, tiles_m - group * G);
  return TileAt{group * G + in % gm, in / gm};
}
__device__ __forceinline__ float load_bias(const Fp8GemmArgs& a, int n) {
  if (!a.bias || n >= a.N) return 0.f;
  return a.bias_dtype == PN_DTYPE_F32 ? reinterpret_cast<const float*>(a.bias)[n] : (float)reinterpret_cast<const __bf16*>(a.bias)[n];
}

// BM x BN tiles, WM x WN waves, blocks of 128 in a ring of RING stages in LDS: while block b is multiplied, the blocks up to
// b + RING - 1 are on their way by direct loads; one barrier a block.
//
// A workgroup goes on from tile to tile: the first blocks of the next tile are on their way before the outputs of the last one
// are written.  bf16 outputs leave through a part of LDS of the wave's own, as whole 128-byte runs: from the accumulators'
// layout they would be 32 bytes of sixteen rows each (measured on 256 x 256 tiles: 32 us a tile that way, 23 blocks' worth).
template <int BM, int BN, int WM, int WN, int RING, bool WIDE> struct Fp8Tile {
  static constexpr int NW = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16, PX = BM / 8 / NW, PW = BN / 8 / NW;
  static constexpr int XBYTES = BM * 128, BUF = (BM + BN) * 128;
  static constexpr int CN = BN / WN, PROWS = FM * 16 < 32 ? FM * 16 : 32, PARK = WIDE ? 0 : PROWS * CN * 2;   // a wave's output rows
  static constexpr int LDS = RING * BUF + NW * PARK;
  static_assert(PX * 8 * NW == BM && PW * 8 * NW == BN && NW % 2 == 0, "every wave stages the same number of 1 KB planes, of one parity");
  static_assert(LDS <= 163840 && RING >= 2, "160 KB");
};

// vmcnt(N) lgkmcnt(15) expcnt(7): the counter of vector memory operations is split over bits 0-3 and 14-15
template <int N> __device__ __forceinline__ void wait_vmcnt() { __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14); }

template <int BM, int BN, int WM, int WN, int RING, bool WIDE>
__global__ __launch_bounds__(WM * WN * 64) void fp8_tile_kernel(Fp8GemmArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef Fp8Tile<BM, BN, WM, WN, RING, WIDE> C;
  constexpr int NW = C::NW, FM = C::FM, FN = C::FN, PX = C::PX, PW = C::PW, BUF = C::BUF, XBYTES = C::XBYTES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, lk = lane >> 4;
  const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
  const int total = a.tiles_m * a.tiles_n, per = (total + 7) / 8;
  const int end = min((int)(blockIdx.x & 7) * per + per, total), step = (int)gridDim.x >> 3;
  int lin = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if (lin >= end) return;                                 // the whole workgroup

  // Operands of the tile that is being staged: a wave's pieces are planes of 1 KB, NW planes apart.  Groups of 16 rows past
  // an operand's end lie past the descriptor's range and come as zeros; their outputs are not stored.
  const unsigned strip = (unsigned)a.kblocks * 2048u;     // bytes of a group of 16 rows
  long long m0;
  int n0, rows_m, rows_n;
  __amdgpu_buffer_rsrc_t rx, rw;
  const unsigned voff = (unsigned)lane * 16 + (unsigned)(wave & 1) * 1024 + (unsigned)(wave >> 1) * strip;
  const unsigned vsx = (unsigned)(wm + lr) * 4, vsw = (unsigned)(wn + lr) * 4;
  auto enter = [&](int at) {
    const TileAt t = tile_at(at, a.tiles_m, a.tiles_n);
    m0 = (long long)t.m * BM;
    n0 = t.n * BN;
    rows_m = a.M - m0 < BM ? (int)(a.M - m0) : BM;
    rows_n = a.N - n0 < BN ? a.N - n0 : BN;
    rx = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x + (m0 >> 4) * strip), 0, (int)((unsigned)(rows_m + 15) / 16 * strip), 0x00020000);
    rw = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + (long long)(n0 >> 4) * strip), 0, (int)((unsigned)(rows_n + 15) / 16 * strip),
                                           0x00020000);
  };
  auto stage = [&](int kb) {
    char* base = smem + kb % RING * BUF + wave * 1024;
#pragma unroll
    for (int j = 0; j < PX; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (__attribute__((address_space(3))) void*)(base + j * NW * 1024), 16,
                                               voff + j * (NW / 2) * strip, kb * 2048, 0, 0);
#pragma unroll
    for (int j = 0; j < PW; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (__attribute__((address_space(3))) void*)(base + XBYTES + j * NW * 1024), 16,
                                               voff + j * (NW / 2) * strip, kb * 2048, 0, 0);
  };
  uint32_t sx[FM], sw[FN], nx[FM], nw[FN];                // scale words of this lane's rows (four blocks each), and the next ones
  auto scales = [&](int q) {
    const __amdgpu_buffer_rsrc_t x = __builtin_amdgcn_make_buffer_rsrc((void*)(a.xs + (long long)q * a.x_rows + m0), 0, rows_m * 4, 0x00020000);
    const __amdgpu_buffer_rsrc_t w = __builtin_amdgcn_make_buffer_rsrc((void*)(a.ws + (long long)q * a.N + n0), 0, rows_n * 4, 0x00020000);
#pragma unroll
    for (int i = 0; i < FM; ++i) nx[i] = __builtin_amdgcn_raw_buffer_load_b32(x, vsx + i * 64, 0, 0);
#pragma unroll
    for (int j = 0; j < FN; ++j) nw[j] = __builtin_amdgcn_raw_buffer_load_b32(w, vsw + j * 64, 0, 0);
  };
  auto open = [&]() {                                     // the first blocks of the tile just entered
    scales(0);
#pragma unroll
    for (int k = 0; k < RING - 1; ++k)
      if (k < a.kblocks) stage(k);
  };

  enter(lin);
  open();
  bool stores_behind = false;                             // STORES stores were issued behind the staged blocks' loads
  constexpr int STORES = WIDE ? FM * FN : FM * 16 * C::CN / 512, AHEAD = (RING - 2) * (PX + PW);
  static_assert(STORES + AHEAD < 64, "what the counter holds");
  while (true) {
    fp8_f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = fp8_f32x4{0.f, 0.f, 0.f, 0.f};
    for (int kb = 0; kb < a.kblocks; ++kb) {
      asm volatile("" ::: "memory");
      // Block kb's loads have landed.  The counter counts in order: behind them are those of the RING - 2 next blocks (near
      // the end fewer: then all have to be there) and, at a tile's first block, the last tile's STORES stores.
      if (RING > 2 && kb + RING - 2 < a.kblocks) {
        if (kb == 0 && stores_behind) wait_vmcnt<STORES + AHEAD>();
        else wait_vmcnt<AHEAD>();
      } else {
        if (kb == 0 && stores_behind) wait_vmcnt<STORES>();
        else wait_vmcnt<0>();
      }
      __builtin_amdgcn_s_barrier();                       // ... for all waves, and nobody reads block kb - 1 any more
      asm volatile("" ::: "memory");
      if ((kb & 3) == 0) {
#pragma unroll
        for (int i = 0; i < FM; ++i) sx[i] = nx[i];
#pragma unroll
        for (int j = 0; j < FN; ++j) sw[j] = nw[j];
        if ((kb >> 2) + 1 < a.kquads) scales((kb >> 2) + 1);
      }
      if (kb + RING - 1 < a.kblocks) stage(kb + RING - 1);
      const char* bx = smem + kb % RING * BUF + wm * 128 + lane * 16;
      const char* bw = smem + kb % RING * BUF + XBYTES + wn * 128 + lane * 16;
      i32x8 fw[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(bw + j * 2048), hi = *reinterpret_cast<const i32x4*>(bw + j * 2048 + 1024);
        fw[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
      if (!WIDE) {
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const i32x4 lo = *reinterpret_cast<const i32x4*>(bx + i * 2048), hi = *reinterpret_cast<const i32x4*>(bx + i * 2048 + 1024);
          const i32x8 fx = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mfma_fp8(fw[j], fx, acc[i][j], sw[j], sx[i]);   // D[n][m]
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          fp8_bf16x8 ww[FN];
#pragma unroll
          for (int j = 0; j < FN; ++j) ww[j] = widen8(fw[j][2 * e], fw[j][2 * e + 1], scale_of(sw[j]));
#pragma unroll
          for (int i = 0; i < FM; ++i) {
            const i32x2 v = *reinterpret_cast<const i32x2*>(bx + i * 2048 + (e >> 1) * 1024 + (e & 1) * 8);
            const fp8_bf16x8 xx = widen8(v[0], v[1], scale_of(sx[i]));
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ww[j], xx, acc[i][j], 0, 0, 0);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < FM; ++i) sx[i] >>= 8;
#pragma unroll
      for (int j = 0; j < FN; ++j) sw[j] >>= 8;
    }

    // outputs: a lane holds n = 4 * lk .. +3 of m = lr for each 16 x 16 piece
    const long long om = m0 + wm, left_m = a.M - om;
    const int on = n0 + wn, left_n = a.N - on;
    const bool whole = left_m >= FM * 16 && left_n >= C::CN;
    int el = lane;                                        // (opaque: what the epilogue derives from it is not kept over the tiles)
    asm volatile("" : "+v"(el));
    const int er = el & 15, ek = el >> 4;
    float bias[FN][4];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[j][e] = load_bias(a, on + j * 16 + ek * 4 + e);
    lin += step;
    const bool more = lin < end;
    if (more) {
      __syncthreads();                                    // all waves have read the last block
      enter(lin);
      open();
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (WIDE) {
      float* out = reinterpret_cast<float*>(a.out) + om * a.ldo + on;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          struct __attribute__((packed, aligned(4))) Raw { float v[4]; } q;
#pragma unroll
          for (int e = 0; e < 4; ++e) q.v[e] = act_f(acc[i][j][e] + bias[j][e], a.act);
          float* o = out + (i * 16 + er) * a.ldo + j * 16 + ek * 4;
          if (whole) {
            *reinterpret_cast<Raw*>(o) = q;
          } else if (i * 16 + er < left_m) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (j * 16 + ek * 4 + e < left_n) o[e] = q.v[e];
          }
        }
    } else {
      constexpr int ROWB = C::CN * 2, CH = ROWB / 16, SWZ = CH < 8 ? CH - 1 : 7, RPI = 64 / CH;
      char* park = smem + RING * BUF + wave * C::PARK;
      __bf16* out = reinterpret_cast<__bf16*>(a.out) + om * a.ldo + on;
#pragma unroll
      for (int r0 = 0; r0 < FM * 16; r0 += C::PROWS) {
#pragma unroll
        for (int i = 0; i < C::PROWS / 16; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            typedef __attribute__((ext_vector_type(4))) __bf16 V4;
            V4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (__bf16)act_bf16(acc[r0 / 16 + i][j][e] + bias[j][e], a.act);
            const int row = i * 16 + er, at = j * 32 + ek * 8;
            *reinterpret_cast<V4*>(park + row * ROWB + (((at >> 4) ^ ((row >> 1) & SWZ)) << 4) + (at & 15)) = o;
          }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the wave's own rows: no other wave touches them
#pragma unroll
        for (int r = 0; r < C::PROWS; r += RPI) {
          const int row = r + el / CH, ch = el % CH;
          const uint4 v = *reinterpret_cast<const uint4*>(park + row * ROWB + ((ch ^ ((row >> 1) & SWZ)) << 4));
          struct __attribute__((packed, aligned(2))) Raw { __bf16 v[8]; };    // rows of odd length start at any element
          const Raw q = __builtin_bit_cast(Raw, v);
          __bf16* o = out + (r0 + row) * a.ldo + ch * 8;
          if (whole) {
            *reinterpret_cast<Raw*>(o) = q;
          } else if (r0 + row < left_m) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (ch * 8 + e < left_n) o[e] = q.v[e];
          }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // read before the next rows overwrite them
      }
    }
    if (!more) break;
    stores_behind = whole;
  }
#endif
}

// Large products: 256 x 256 tiles, eight waves of 128 x 64 (WIDE: 128 x 256 tiles, waves of 64 x 64) in two groups of four, one
// wave of each group on every SIMD, half a block apart.  While one group multiplies its block from registers, the other reads its own from LDS (the first also
// sends for the block after); then they change places (two barriers a block).  The matrix pipe of a SIMD always has a wave that needs
// nothing else.
// WIDE, the widening to bf16 is part of the reading half: two vector instructions for each matrix instruction that would otherwise
// wait for them (8192^3: 933 us with all waves in step).
template <bool WIDE> struct Fp8Pair {
  static constexpr int BM = WIDE ? 128 : 256, BN = 256, NW = 8, FM = BM / 32, FN = 4, XBYTES = BM * 128, BUF = (BM + BN) * 128;
  static constexpr int SBUF = 2048, PARK = WIDE ? 0 : 16 * 64 * 2, LDS = 2 * BUF + 2 * SBUF + NW * PARK;   // scale words: 256 rows of x, 256 of w
};
template <bool WIDE>
__global__ __launch_bounds__(512) void fp8_pair_kernel(Fp8GemmArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef Fp8Pair<WIDE> C;
  constexpr int NW = C::NW, FM = C::FM, FN = C::FN, BUF = C::BUF, XBYTES = C::XBYTES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, lk = lane >> 4;
  const int group = wave >> 2;                            // waves 0-3 and 4-7: one of each on every SIMD
  const int wm = group * (C::BM / 2), wn = (wave & 3) * 64;
  const unsigned strip = (unsigned)a.kblocks * 2048u;     // bytes of a group of 16 rows
  const int total = a.tiles_m * a.tiles_n, per = (total + 7) / 8;
  const int end = min((int)(blockIdx.x & 7) * per + per, total), step = (int)gridDim.x >> 3;
  int lin = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if (lin >= end) return;                                 // the whole workgroup

  long long m0;
  int n0, rows_m, rows_n;
  __amdgpu_buffer_rsrc_t rx, rw;
  // the first group's waves send for everything: 8 planes of either operand each, four planes apart
  const unsigned voff = (unsigned)lane * 16 + (unsigned)(wave & 1) * 1024 + (unsigned)((wave & 3) >> 1) * strip;
  auto enter = [&](int at) {
    const TileAt t = tile_at(at, a.tiles_m, a.tiles_n);
    m0 = (long long)t.m * C::BM;
    n0 = t.n * C::BN;
    rows_m = a.M - m0 < C::BM ? (int)(a.M - m0) : C::BM;
    rows_n = a.N - n0 < C::BN ? a.N - n0 : C::BN;
    rx = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x + (m0 >> 4) * strip), 0, (int)((unsigned)(rows_m + 15) / 16 * strip), 0x00020000);
    rw = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + (long long)(n0 >> 4) * strip), 0, (int)((unsigned)(rows_n + 15) / 16 * strip),
                                           0x00020000);
  };
  auto stage = [&](int kb) {
    char* base = smem + (kb & 1) * BUF + wave * 1024;
#pragma unroll
    for (int j = 0; j < C::BM / 32; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (__attribute__((address_space(3))) void*)(base + j * 4096), 16, voff + j * 2 * strip,
                                               kb * 2048, 0, 0);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (__attribute__((address_space(3))) void*)(base + XBYTES + j * 4096), 16,
                                               voff + j * 2 * strip, kb * 2048, 0, 0);
    if ((kb & 3) == 0) {                                  // the scale words of four blocks: 64 rows of either operand a wave
      const int q = kb >> 2, r0 = wave * 64;
      char* sb = smem + 2 * BUF + (q & 1) * C::SBUF + wave * 256;
      const __amdgpu_buffer_rsrc_t qx = __builtin_amdgcn_make_buffer_rsrc((void*)(a.xs + (long long)q * a.x_rows + m0), 0, rows_m * 4, 0x00020000);
      const __amdgpu_buffer_rsrc_t qw = __builtin_amdgcn_make_buffer_rsrc((void*)(a.ws + (long long)q * a.N + n0), 0, rows_n * 4, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(qx, (__attribute__((address_space(3))) void*)sb, 4, (unsigned)(r0 + lane) * 4, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(qw, (__attribute__((address_space(3))) void*)(sb + 1024), 4, (unsigned)(r0 + lane) * 4, 0, 0, 0);
    }
  };
#define PAIR_BARRIER()                     \
  do {                                     \
    asm volatile("" ::: "memory");         \
    __builtin_amdgcn_sched_barrier(0);     \
    __builtin_amdgcn_s_barrier();          \
    __builtin_amdgcn_sched_barrier(0);     \
    asm volatile("" ::: "memory");         \
  } while (0)

  enter(lin);
  if (!group) stage(0);
  bool stores_behind = false;
  constexpr int STORES = WIDE ? FM * FN : FM * 2;
  while (true) {
    fp8_f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = fp8_f32x4{0.f, 0.f, 0.f, 0.f};
    // block 0 has landed (in order behind it: the last tile's stores, which may go on)
    asm volatile("" ::: "memory");
    if (stores_behind) wait_vmcnt<STORES>();
    else wait_vmcnt<0>();
    PAIR_BARRIER();
    if (group) PAIR_BARRIER();
    for (int kb = 0; kb < a.kblocks; ++kb) {
      // reading; nobody reads block kb - 1 any more, so block kb + 1 may land in its place
      if (!group && kb + 1 < a.kblocks) stage(kb + 1);
      const char* lx = smem + (kb & 1) * BUF + wm * 128 + lane * 16;
      const char* lw = smem + (kb & 1) * BUF + XBYTES + wn * 128 + lane * 16;
      const unsigned char* sc = reinterpret_cast<const unsigned char*>(smem) + 2 * BUF + ((kb >> 2) & 1) * C::SBUF + (kb & 3);
      i32x8 fx[FM], fw[FN];
      uint32_t sx[FM], sw[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(lw + j * 2048), hi = *reinterpret_cast<const i32x4*>(lw + j * 2048 + 1024);
        fw[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        sw[j] = sc[(256 + wn + j * 16 + lr) * 4];
      }
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(lx + i * 2048), hi = *reinterpret_cast<const i32x4*>(lx + i * 2048 + 1024);
        fx[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        sx[i] = sc[(wm + i * 16 + lr) * 4];
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xc07f);                 // lgkmcnt(0): the reads are done
      fp8_bf16x8 bx[WIDE ? FM : 1][4], bw_[WIDE ? FN : 1][4];
      if constexpr (WIDE) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int j = 0; j < FN; ++j) bw_[j][e] = widen8(fw[j][2 * e], fw[j][2 * e + 1], scale_of(sw[j]));
#pragma unroll
          for (int i = 0; i < FM; ++i) bx[i][e] = widen8(fx[i][2 * e], fx[i][2 * e + 1], scale_of(sx[i]));
        }
      }
      PAIR_BARRIER();
      __builtin_amdgcn_s_setprio(1);
      if constexpr (WIDE) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bw_[j][e], bx[i][e], acc[i][j], 0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mfma_fp8(fw[j], fx[i], acc[i][j], sw[j], sx[i]);   // D[n][m]
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(0);
      asm volatile("" ::: "memory");
      wait_vmcnt<0>();                                    // block kb + 1 has landed (the first group's waves sent for it)
      PAIR_BARRIER();
    }
    if (!group) PAIR_BARRIER();

    const long long om = m0 + wm, left_m = a.M - om;
    const int on = n0 + wn, left_n = a.N - on;
    const bool whole = left_m >= FM * 16 && left_n >= 64;
    int el = lane;                                        // (opaque: what the epilogue derives from it is not kept over the tiles)
    asm volatile("" : "+v"(el));
    const int er = el & 15, ek = el >> 4;
    float bias[FN][4];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[j][e] = load_bias(a, on + j * 16 + ek * 4 + e);
    lin += step;
    const bool more = lin < end;
    if (more) {
      enter(lin);                                         // (behind the last barrier: all waves have read the last block)
      if (!group) stage(0);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (WIDE) {
      float* out = reinterpret_cast<float*>(a.out) + om * a.ldo + on;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          struct __attribute__((packed, aligned(4))) Raw { float v[4]; } q;
#pragma unroll
          for (int e = 0; e < 4; ++e) q.v[e] = act_f(acc[i][j][e] + bias[j][e], a.act);
          float* o = out + (i * 16 + er) * a.ldo + j * 16 + ek * 4;
          if (whole) {
            *reinterpret_cast<Raw*>(o) = q;
          } else if (i * 16 + er < left_m) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (j * 16 + ek * 4 + e < left_n) o[e] = q.v[e];
          }
        }
    } else {
      char* park = smem + 2 * BUF + 2 * C::SBUF + wave * C::PARK;
      __bf16* out = reinterpret_cast<__bf16*>(a.out) + om * a.ldo + on;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          typedef __attribute__((ext_vector_type(4))) __bf16 V4;
          V4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = (__bf16)act_bf16(acc[i][j][e] + bias[j][e], a.act);
          const int at = j * 32 + ek * 8;
          *reinterpret_cast<V4*>(park + er * 128 + (((at >> 4) ^ (er >> 1)) << 4) + (at & 15)) = o;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");         // the wave's own rows: no other wave touches them
#pragma unroll
        for (int r = 0; r < 16; r += 8) {
          const int row = r + (el >> 3), ch = el & 7;
          const uint4 v = *reinterpret_cast<const uint4*>(park + row * 128 + ((ch ^ (row >> 1)) << 4));
          struct __attribute__((packed, aligned(2))) Raw { __bf16 v[8]; };    // rows of odd length start at any element
          const Raw q = __builtin_bit_cast(Raw, v);
          __bf16* o = out + (i * 16 + row) * a.ldo + ch * 8;
          if (whole) {
            *reinterpret_cast<Raw*>(o) = q;
          } else if (i * 16 + row < left_m) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (ch * 8 + e < left_n) o[e] = q.v[e];
          }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");         // read before the next rows overwrite them
      }
    }
    if (!more) break;
    stores_behind = whole;
  }
#undef PAIR_BARRIER
#endif
}

// Few rows (one row at the least): a workgroup owns 16 rows and FN * 16 columns, its waves deal the blocks of 128 among
// themselves and add up through LDS at the end.  The rows of x come as they are and are laid out on the way, a block at a time,
// through 2 KB of LDS of the wave's own: one launch, and no bytes of x in memory.  What bounds it is the weights' read.  (fp32 rows into
// fp32 results with 64 columns take all 256 registers and 12 bytes of scratch a lane.)
struct Fp8DirectArgs {
  Fp8GemmArgs g;
  const void* x;             // [M][ldx] fp32 or bf16
  long long ldx;
  int K;
};

// 16 rows x 128 elements as they lie: LOADS loads, each of whole rows; LANES lanes and EACH elements a lane make a row
template <typename T> struct RawRows;
template <> struct RawRows<__bf16> {
  static constexpr int LOADS = 4, LANES = 16, EACH = 8;
  Raw8<__bf16> v[4];
  __device__ __forceinline__ void load(int j, const __bf16* p) { v[j].load(p); }
  template <bool FINITE> __device__ __forceinline__ uint32_t mag(int j) const { return v[j].template row_mag<FINITE>(); }
  static __device__ __forceinline__ uint32_t row_max(uint32_t m) { return Raw8<__bf16>::mag_bits(mag_max16<Raw8<__bf16>>(m)); }
  __device__ __forceinline__ uint2 quant(int j, float s) const { return v[j].quant(s); }
  __device__ __forceinline__ void drop(int j, int n) {                      // the first n elements become zero
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) v[j].v[i >> 1] &= i & 1 ? 0xffffu : 0xffff0000u;
  }
};
template <> struct RawRows<float> {
  static constexpr int LOADS = 8, LANES = 32, EACH = 4;
  struct __attribute__((packed, aligned(4))) F4 { float v[4]; };
  F4 v[8];
  __device__ __forceinline__ void load(int j, const float* p) { v[j] = *reinterpret_cast<const F4*>(p); }
  template <bool FINITE> __device__ __forceinline__ uint32_t mag(int j) const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = __float_as_uint(v[j].v[i]) & 0x7fffffffu;
      m = umax(m, FINITE && b >= 0x7f800000u ? 0u : b);
    }
    return m;
  }
  static __device__ __forceinline__ uint32_t row_max(uint32_t m) {
    m = mag_max16<Raw8<float>>(m);
    return umax(m, (uint32_t)__shfl_xor((int)m, 16));
  }
  __device__ __forceinline__ uint2 quant(int j, float s) const {
    ffn_s16x2 a = {0, 0};
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[j].v[0], v[j].v[1], s, false);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[j].v[2], v[j].v[3], s, true);
    return make_uint2(__builtin_bit_cast(uint32_t, a), 0);
  }
  __device__ __forceinline__ void drop(int j, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) v[j].v[i] = 0.f;
  }
};

struct Fp8Laid {};         // x is an operand already
template <> struct RawRows<Fp8Laid> {
  static constexpr int LOADS = 2, LANES = 16, EACH = 8;
  i32x4 v[2];
  uint32_t scale;
};

template <typename T, int FN, int NW, int DEPTH, bool WIDE>
__global__ __launch_bounds__(NW * 64) void fp8_direct_kernel(Fp8DirectArgs d) {
  typedef RawRows<T> R;
  constexpr bool LAID = std::is_same<T, Fp8Laid>::value;
  constexpr int OWN = 2048 + 16;                          // a wave's part of LDS: a block's bytes and its rows' scales
  const Fp8GemmArgs& a = d.g;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lk = lane >> 4;
  // Workgroups are dealt to the XCDs round robin: with eight strips of rows or more an XCD keeps to its own (x is read from
  // memory once, the smaller weights by all); with fewer it keeps to its own columns (the weights are read once).
  const int idx = (int)(blockIdx.x >> 3), xcd = (int)(blockIdx.x & 7);
  const int tm = a.tiles_m >= 8 ? idx / a.tiles_n * 8 + xcd : idx % a.tiles_m, tn = a.tiles_m >= 8 ? idx % a.tiles_n : idx / a.tiles_m * 8 + xcd;
  if (tm >= a.tiles_m || tn >= a.tiles_n) return;         // the whole workgroup
  const long long m0 = (long long)tm * 16;
  const int n0 = tn * (FN * 16);
  // lane's rows of x: row j * (64 / LANES) + lane / LANES of the strip, EACH elements from (lane % LANES) * EACH on; rows past the
  // end repeat the last one (their outputs are not stored)
  const T* px[R::LOADS];
  const unsigned char* qx = a.x + (size_t)tm * a.kblocks * 2048 + lane * 16;
  const unsigned char* qs = reinterpret_cast<const unsigned char*>(a.xs + (m0 + lr < a.M ? m0 + lr : a.M - 1));
#pragma unroll
  for (int j = 0; j < R::LOADS; ++j) {
    if (LAID) break;
    const long long m = m0 + j * (64 / R::LANES) + lane / R::LANES;
    px[j] = reinterpret_cast<const T*>(d.x) + (m < a.M ? m : a.M - 1) * d.ldx + (lane % R::LANES) * R::EACH;
  }
  const unsigned char *pw[FN], *ps[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int n = n0 + j * 16 < a.N ? n0 + j * 16 : n0, r = n + lr < a.N ? n + lr : a.N - 1;
    pw[j] = a.w + (size_t)(n >> 4) * a.kblocks * 2048 + lane * 16;
    ps[j] = reinterpret_cast<const unsigned char*>(a.ws + r);
  }
  char* own = smem + wave * OWN;
  const int k_own = (lane % R::LANES) * R::EACH;          // first element of this lane's part of a row's block
  fp8_f32x4 acc[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) acc[j] = fp8_f32x4{0.f, 0.f, 0.f, 0.f};
  // DEPTH blocks of a wave are on their way at a time.  No load stands behind a branch: the compiler's wait counts would then
  // cover the newest load, and DEPTH would be one.  So past a wave's last block the loads repeat it, and the last block of an
  // odd contraction reads x as the row's last 128 elements, moved to their places when the block is laid out.
  R x[DEPTH];
  i32x8 w[DEPTH][FN];
  uint32_t sw[DEPTH][FN];
  const int last = a.kblocks - 1, tail = d.K - 128;
  auto fetch = [&](R& nx, i32x8 (&nw)[FN], uint32_t (&ns)[FN], int kb) {
    kb = min(kb, last);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const i32x4 lo = *reinterpret_cast<const i32x4*>(pw[j] + (size_t)kb * 2048), hi = *reinterpret_cast<const i32x4*>(pw[j] + (size_t)kb * 2048 + 1024);
      nw[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      ns[j] = ps[j][(long long)(kb >> 2) * a.N * 4 + (kb & 3)];
    }
    if constexpr (LAID) {
#pragma unroll
      for (int j = 0; j < 2; ++j) nx.v[j] = *reinterpret_cast<const i32x4*>(qx + (size_t)kb * 2048 + j * 1024);
      nx.scale = qs[(long long)(kb >> 2) * a.x_rows * 4 + (kb & 3)];
    } else {
#pragma unroll
      for (int j = 0; j < R::LOADS; ++j) nx.load(j, px[j] + min(kb * 128, tail));
    }
    __builtin_amdgcn_sched_barrier(0);                    // the loads of a block stay together, in order
  };
#pragma unroll
  for (int s = 0; s < DEPTH; ++s) fetch(x[s], w[s], sw[s], wave + s * NW);
  for (int kb0 = wave; kb0 < a.kblocks; kb0 += DEPTH * NW) {
#pragma unroll
    for (int s = 0; s < DEPTH; ++s) {
      const int kb = kb0 + s * NW;
      if (kb >= a.kblocks) break;
      i32x4 lo, hi;
      uint32_t sx;
      if constexpr (LAID) {
        lo = x[s].v[0];
        hi = x[s].v[1];
        sx = x[s].scale;
      } else {
        // element e of the 128 that were read is k = e - shift of the block; those before the block are dropped
        const int shift = kb * 128 > tail ? kb * 128 - tail : 0;
        uint32_t mag[R::LOADS], any = 0;
        if (shift) {
#pragma unroll
          for (int j = 0; j < R::LOADS; ++j) x[s].drop(j, shift - k_own);
        }
#pragma unroll
        for (int j = 0; j < R::LOADS; ++j) {
          mag[j] = x[s].template mag<false>(j);
          any = Raw8<T>::mag_max(any, mag[j]);
        }
        if (Raw8<T>::mag_inf(any)) {                        // rare: leave out what is not finite
#pragma unroll
          for (int j = 0; j < R::LOADS; ++j) mag[j] = x[s].template mag<true>(j);
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int j = 0; j < R::LOADS; ++j) {
          const int sc = block_scale(R::row_max(mag[j])), row = j * (64 / R::LANES) + lane / R::LANES;
          const uint2 o = x[s].quant(j, scale_value((uint32_t)sc));
          auto place = [&](int k) { return own + ((k >> 4) & 1) * 1024 + ((k >> 5) * 16 + row) * 16 + (k & 15); };
          if (!shift) {
            if (R::EACH == 8) *reinterpret_cast<uint2*>(place(k_own)) = o;
            else *reinterpret_cast<uint32_t*>(place(k_own)) = o.x;
          } else {                                          // byte by byte; the dropped elements' zeros fill the block's end
#pragma unroll
            for (int i = 0; i < R::EACH; ++i) *place((k_own + i - shift) & 127) = (char)((i < 4 ? o.x : o.y) >> (8 * (i & 3)));
          }
          if (lane % R::LANES == 0) own[2048 + row] = (char)sc;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own part: no other wave touches it
        lo = *reinterpret_cast<const i32x4*>(own + lane * 16);
        hi = *reinterpret_cast<const i32x4*>(own + 1024 + lane * 16);
        sx = (unsigned char)own[2048 + lr];
      }
      const i32x8 q = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      if (WIDE) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const fp8_bf16x8 xx = widen8(q[2 * c], q[2 * c + 1], scale_of(sx));
#pragma unroll
          for (int j = 0; j < FN; ++j)
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(w[s][j][2 * c], w[s][j][2 * c + 1], scale_of(sw[s][j])), xx, acc[j], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[j] = mfma_fp8(w[s][j], q, acc[j], sw[s][j], sx);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next block overwrites it
      fetch(x[s], w[s], sw[s], kb + DEPTH * NW);
    }
  }
  // add the waves' sums in order; a thread then holds four outputs of a row
  __syncthreads();
  float4* part = reinterpret_cast<float4*>(smem);         // [NW][FN][64]
#pragma unroll
  for (int j = 0; j < FN; ++j) part[(wave * FN + j) * 64 + lane] = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
  __syncthreads();
  for (int p = threadIdx.x; p < FN * 64; p += NW * 64) {
    const int l = p & 63, n = n0 + (p >> 6) * 16 + (l >> 4) * 4;
    const long long m = m0 + (l & 15);
    float4 s = part[p];
#pragma unroll
    for (int q = 1; q < NW; ++q) {
      const float4 t = part[q * FN * 64 + p];
      s.x += t.x;
      s.y += t.y;
      s.z += t.z;
      s.w += t.w;
    }
    float v[4] = {s.x, s.y, s.z, s.w};
    if (a.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += load_bias(a, min(n + e, a.N - 1));
    }
    if (m < a.M) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.N) {
          if (WIDE) reinterpret_cast<float*>(a.out)[m * a.ldo + n + e] = act_f(v[e], a.act);
          else reinterpret_cast<__bf16*>(a.out)[m * a.ldo + n + e] = (__bf16)act_bf16(v[e], a.act);
        }
    }
  }
}

// ---- host ----
static int fp8_cus() {                                    // compute units of the current device
  static thread_local int device = -1, cus = 0;
  int d = 0;
  if (hipGetDevice(&d) != hipSuccess) return 256;
  if (d != device) {
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, d) != hipSuccess || cus < 8) cus = 256;
    device = d;
  }
  return cus;
}

// More than 64 KB of LDS has to be allowed for a kernel once on each device; `on`: the one that this thread allowed it on last
static int fp8_raise_lds(const void* kernel, int bytes, int* on) {
  int d = 0;
  if (bytes <= 65536) return PN_OK;
  PN_CHECK_HIP(hipGetDevice(&d));
  if (d == *on) return PN_OK;
  PN_CHECK_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  *on = d;
  return PN_OK;
}

static unsigned fp8_grid(Fp8GemmArgs& a, int bm, int bn, int resident) {
  a.tiles_m = (int)((a.M + bm - 1) / bm);
  a.tiles_n = (a.N + bn - 1) / bn;
  const long long tiles = ((long long)a.tiles_m * a.tiles_n + 7) / 8 * 8, slots = (long long)fp8_cus() / 8 * 8 * resident;
  return (unsigned)(tiles < slots ? tiles : slots);
}

template <int BM, int BN, int WM, int WN, int RING, bool WIDE> static int fp8_tile(Fp8GemmArgs a, hipStream_t s) {
  typedef Fp8Tile<BM, BN, WM, WN, RING, WIDE> C;
  static thread_local int raised_on = -1;
  const int rc = fp8_raise_lds((const void*)fp8_tile_kernel<BM, BN, WM, WN, RING, WIDE>, C::LDS, &raised_on);
  if (rc != PN_OK) return rc;
  const unsigned grid = fp8_grid(a, BM, BN, 163840 / C::LDS < 16 / C::NW ? 163840 / C::LDS : 16 / C::NW);
  hipLaunchKernelGGL((fp8_tile_kernel<BM, BN, WM, WN, RING, WIDE>), dim3(grid), dim3(C::NW * 64), C::LDS, s, a);
  PN_CHECK_LAUNCH("fp8_tile_kernel");
  return PN_OK;
}

template <bool WIDE> static int fp8_pair(Fp8GemmArgs a, hipStream_t s) {
  typedef Fp8Pair<WIDE> C;
  static thread_local int raised_on = -1;
  const int rc = fp8_raise_lds((const void*)fp8_pair_kernel<WIDE>, C::LDS, &raised_on);
  if (rc != PN_OK) return rc;
  const unsigned grid = fp8_grid(a, C::BM, C::BN, 1);
  hipLaunchKernelGGL(fp8_pair_kernel<WIDE>, dim3(grid), dim3(512), C::LDS, s, a);
  PN_CHECK_LAUNCH("fp8_pair_kernel");
  return PN_OK;
}

template <typename T, int FN, int NW, int DEPTH> static int fp8_direct(Fp8DirectArgs d, hipStream_t s) {
  constexpr int OWN = NW * 2064, PART = NW * FN * 1024, LDS = OWN > PART ? OWN : PART;
  static_assert(LDS <= 65536, "the default limit");
  d.g.tiles_m = (int)((d.g.M + 15) / 16);
  d.g.tiles_n = (d.g.N + FN * 16 - 1) / (FN * 16);
  const dim3 grid(d.g.tiles_m >= 8 ? (d.g.tiles_m + 7) / 8 * 8 * d.g.tiles_n : (d.g.tiles_n + 7) / 8 * 8 * d.g.tiles_m), wg(NW * 64);
  if (d.g.out_dtype == PN_DTYPE_F32) hipLaunchKernelGGL((fp8_direct_kernel<T, FN, NW, DEPTH, true>), grid, wg, LDS, s, d);
  else hipLaunchKernelGGL((fp8_direct_kernel<T, FN, NW, DEPTH, false>), grid, wg, LDS, s, d);
  PN_CHECK_LAUNCH("fp8_direct_kernel");
  return PN_OK;
}

// Time of a product by tiles, in us: whole rounds of the workgroups that fit on the device, each a cost per block and one per
// tile.  Measured on 256 CUs (8192^3 and 16384 x 4096 x 8192: rounds of 64 and 32 blocks; 512 x 3136 x 256: 25 blocks, a tile or
// less a CU): pairs, 256 x 256, 398 / 450 us (fp32 outputs, 128 x 256: 865 / 940); 128 x 128 523 / 562 (1000 / 998); 64 x 64
// 764 / 884 (1239 / 1327).
struct Fp8Cost { int bm, bn, resident; float round_block, round_tile, lone_block, lone_tile; };
static const Fp8Cost FP8_PAIR[2] = {{256, 256, 1, 1.35f, 13.f, 1.35f, 13.f}, {128, 256, 1, 1.6f, 14.f, 1.6f, 14.f}};  // bf16, fp32 outputs
static const Fp8Cost FP8_128[2] = {{128, 128, 2, 0.95f, 4.8f, 0.78f, 3.f}, {128, 128, 2, 1.85f, 6.f, 1.25f, 7.f}};
static const Fp8Cost FP8_64[2] = {{64, 64, 4, 0.63f, 5.f, 0.35f, 2.6f}, {64, 64, 4, 1.12f, 5.6f, 0.52f, 2.6f}};
static float fp8_cost(const Fp8Cost& c, long long m, int n, int kblocks, int cus) {
  const long long tiles = (m + c.bm - 1) / c.bm * ((n + c.bn - 1) / c.bn);
  if (tiles <= cus) return c.lone_block * kblocks + c.lone_tile;
  return (float)((tiles + cus * c.resident - 1) / (cus * c.resident)) * (c.round_block * kblocks + c.round_tile);
}

// Few tiles and a long contraction: a CU takes 64 x 64 x 128 in 0.35 us however few of them there are (what it loads), so the
// work is spread over more CUs by 16 rows x 32 or 64 columns, the blocks dealt to a workgroup's waves (512 x 3136 x 256: 6 us
// against 11).
static bool fp8_spread(long long m, int n, int k) { return k >= 1024 && (m + 15) / 16 * ((n + 63) / 64) <= 256; }
static int fp8_direct_kind(long long m, int n) { return (m + 15) / 16 * ((n + 31) / 32) <= 256 ? PN_FP8_DIRECT_32 : PN_FP8_DIRECT_64; }
template <typename T> static int fp8_direct_by_kind(int kind, const Fp8DirectArgs& d, hipStream_t s) {
  return kind == PN_FP8_DIRECT_32 ? fp8_direct<T, 2, 8, 2>(d, s) : fp8_direct<T, 4, 8, 2>(d, s);
}

// The kernel of a product's first `rows` rows, and that of the rows behind them (0: there are none)
struct Fp8Plan { int kind, rest; long long rows; };
static int fp8_small_kind(long long m, int n, int kb, int cus, bool wide) {
  if (fp8_spread(m, n, kb * 128)) return fp8_direct_kind(m, n);
  return fp8_cost(FP8_64[wide], m, n, kb, cus) <= fp8_cost(FP8_128[wide], m, n, kb, cus) ? PN_FP8_TILE_64 : PN_FP8_TILE_128;
}
static Fp8Plan fp8_plan(long long m, int n, int kb, bool wide) {
  const int cus = fp8_cus(), bm = FP8_PAIR[wide].bm;
  auto small = [&](long long rows) {
    const float c64 = fp8_cost(FP8_64[wide], rows, n, kb, cus), c128 = fp8_cost(FP8_128[wide], rows, n, kb, cus);
    return c64 < c128 ? c64 : c128;
  };
  const float by_small = small(m), by_pair = fp8_cost(FP8_PAIR[wide], m, n, kb, cus);
  // Rows that fill whole tiles of the pair kernel, and the few behind them in a launch of their own: 8200 x 2048 x 4096 takes
  // 94 us as three rounds of 256 x 256, 90 us in 128 x 128, 72 us as two rounds and 8 for a strip of 8 rows
  const long long whole = m / bm * bm;
  const float by_split = whole && whole < m ? fp8_cost(FP8_PAIR[wide], whole, n, kb, cus) + small(m - whole) : 1e30f;
  if (by_small <= by_pair && by_small <= by_split) return Fp8Plan{fp8_small_kind(m, n, kb, cus, wide), 0, m};
  if (by_pair <= by_split) return Fp8Plan{PN_FP8_PAIR, 0, m};
  return Fp8Plan{PN_FP8_PAIR, fp8_small_kind(m - whole, n, kb, cus, wide), whole};
}

template <bool WIDE> static int fp8_gemm_by_kind(int kind, const Fp8GemmArgs& a, hipStream_t s) {
  switch (kind) {
    case PN_FP8_TILE_64: return fp8_tile<64, 64, 2, 2, 2, WIDE>(a, s);
    case PN_FP8_TILE_128: return fp8_tile<128, 128, 2, 2, 2, WIDE>(a, s);
    case PN_FP8_PAIR: return fp8_pair<WIDE>(a, s);
    default: return fp8_direct_by_kind<Fp8Laid>(kind, Fp8DirectArgs{a, nullptr, 0, a.kblocks * 128}, s);
  }
}
template <bool WIDE> static int fp8_gemm_by_size(Fp8GemmArgs a, hipStream_t s) {
  const Fp8Plan plan = fp8_plan(a.M, a.N, a.kblocks, WIDE);
  Fp8GemmArgs t = a;
  a.M = plan.rows;
  const int rc = fp8_gemm_by_kind<WIDE>(plan.kind, a, s);
  if (rc != PN_OK || !plan.rest) return rc;
  t.M -= plan.rows;
  t.x += (size_t)(plan.rows / 16) * a.kblocks * 2048;
  t.xs += plan.rows;
  t.out = (char*)t.out + plan.rows * t.ldo * (WIDE ? 4 : 2);
  return fp8_gemm_by_kind<WIDE>(plan.rest, t, s);
}

int fp8_gemm_launch(const Fp8Gemm& g, hipStream_t s) {
  const Fp8GemmArgs a = {g.x.q, g.w.q, g.x.scale, g.w.scale, g.M, g.M, g.N, (g.K + 127) / 128, (g.K + 511) / 512, 0, 0,
                         g.bias, g.bias_dtype, g.act, g.out_dtype, g.out, g.ldo};
  return g.out_dtype == PN_DTYPE_F32 ? fp8_gemm_by_size<true>(a, s) : fp8_gemm_by_size<false>(a, s);
}

static int fp8_check(const void* w, long long m, int n, int k, const void* bias, int bias_dtype, int act, int out_dtype, void* out, long long ldo) {
  PN_CHECK_ARG(m >= 0 && n >= 1 && k >= 1, "fp8 product: %lld x %d x %d", m, n, k);
  PN_CHECK_ARG(act >= PN_ACT_NONE && act <= PN_ACT_GELU, "fp8 product: activation %d", act);
  PN_CHECK_ARG((out_dtype == PN_DTYPE_F32 || out_dtype == PN_DTYPE_BF16) && (!bias || bias_dtype == PN_DTYPE_F32 || bias_dtype == PN_DTYPE_BF16),
               "fp8 product: output type %d, bias type %d (fp32 or bf16)", out_dtype, bias_dtype);
  PN_CHECK_ARG(k <= 1 << 22, "fp8 product: contraction of %d", k);           // 16 groups of a tile stay within 31-bit offsets
  if (m == 0) return PN_OK;
  PN_CHECK_ARG(w && out && ((uintptr_t)w & 255) == 0, "fp8 product: weight or output missing, or an operand off its 256-byte alignment");
  PN_CHECK_ARG(ldo >= n, "fp8 product: output row stride %lld below %d", ldo, n);
  PN_CHECK_ARG((m + 15) / 16 * (((long long)n + 15) / 16) < (1ll << 31) - 64, "fp8 product: %lld x %d outputs are more than one launch takes", m, n);
  return PN_OK;
}

extern "C" int pn_fp8_gemm(const void* x, long long m, const void* w, int n, int k, const void* bias, int bias_dtype, int act, int out_dtype,
                           void* out, long long ldo, void* stream) {
  const int rc = fp8_check(w, m, n, k, bias, bias_dtype, act, out_dtype, out, ldo);
  if (rc != PN_OK || m == 0) return rc;
  PN_CHECK_ARG(x && ((uintptr_t)x & 255) == 0, "pn_fp8_gemm: x missing or off its 256-byte alignment");
  return fp8_gemm_launch(Fp8Gemm{fp8_operand(x, m, k), fp8_operand(w, n, k), m, n, k, bias, bias_dtype, act, out_dtype, out, ldo},
                         (hipStream_t)stream);
}

// Up to a workgroup of 16 x 64 a CU the rows are laid out on the way: 500 x 3136 x 256 bf16 takes 7.7 us against 4.9 + 10.7 in two
// launches (fp32 10.6 against 6.7 + 15.5), 64 x 4096 x 4096 10.3 against 3.1 + 12.2; 2000 x 1024 x 1024 (eight a CU) 43 against 12.7.
// With half as many, 16 x 32: 500 x 3136 x 256 7.7 us against 9.0, 1000 x 3136 x 256 13.5 against 9.2.
static bool fp8_is_direct(long long m, int n, int k) { return k >= 128 && (m + 15) / 16 * ((n + 63) / 64) <= 256; }

extern "C" int pn_fp8_kernels(long long m, int n, int k, int out_dtype, int laid_out) {
  PN_CHECK_ARG(m >= 1 && n >= 1 && k >= 1 && (out_dtype == PN_DTYPE_F32 || out_dtype == PN_DTYPE_BF16), "pn_fp8_kernels: %lld x %d x %d, type %d", m, n, k,
               out_dtype);
  if (!laid_out && fp8_is_direct(m, n, k)) return fp8_direct_kind(m, n);
  const Fp8Plan plan = fp8_plan(m, n, (k + 127) / 128, out_dtype == PN_DTYPE_F32);
  return plan.kind | plan.rest << 4;
}

extern "C" size_t pn_fp8_linear_workspace_bytes(long long m, int n, int k) {
  return m < 1 || n < 1 || k < 1 || fp8_is_direct(m, n, k) ? 0 : fp8_bytes(m, k);
}

extern "C" int pn_fp8_linear(int dtype, const void* x, long long m, long long ldx, const void* w, int n, int k, const void* bias, int bias_dtype,
                             int act, int out_dtype, void* out, long long ldo, void* ws, size_t ws_bytes, void* stream) {
  PN_CHECK_ARG(dtype == PN_DTYPE_F32 || dtype == PN_DTYPE_BF16, "pn_fp8_linear: element type %d (fp32 or bf16)", dtype);
  int rc = fp8_check(w, m, n, k, bias, bias_dtype, act, out_dtype, out, ldo);
  if (rc != PN_OK || m == 0) return rc;
  PN_CHECK_ARG(x && (m == 1 || ldx >= k), "pn_fp8_linear: x missing or its row stride below the row length");
  hipStream_t s = (hipStream_t)stream;
  if (fp8_is_direct(m, n, k)) {
    Fp8DirectArgs d = {{nullptr, (const unsigned char*)w, nullptr, fp8_operand(w, n, k).scale, m, m, n, (k + 127) / 128, (k + 511) / 512, 0, 0,
                        bias, bias_dtype, act, out_dtype, out, ldo}, x, m == 1 ? 0 : ldx, k};
    const int kind = fp8_direct_kind(m, n);
    return dtype == PN_DTYPE_F32 ? fp8_direct_by_kind<float>(kind, d, s) : fp8_direct_by_kind<__bf16>(kind, d, s);
  }
  if (ws_bytes < fp8_bytes(m, k) || !ws) {
    pn_set_error("pn_fp8_linear: workspace of %zu bytes is too small", ws_bytes);
    return PN_ENOSPC;
  }
  PN_CHECK_ARG(((uintptr_t)ws & 255) == 0, "pn_fp8_linear: the workspace must be 256-byte aligned");
  rc = fp8_quantize_launch(Fp8QuantJob{x, dtype, 1, m, ldx, k, ws, nullptr, nullptr}, s);
  if (rc != PN_OK) return rc;
  return fp8_gemm_launch(Fp8Gemm{fp8_operand(ws, m, k), fp8_operand(w, n, k), m, n, k, bias, bias_dtype, act, out_dtype, out, ldo}, s);
}

// ---- training: y = x w^T + bias, its gradients ----
struct Fp8TrainLayout { size_t xt, wt, saved, x, w, ws_fwd, g, gt, colsum, ws_bwd; };
static Fp8TrainLayout fp8_train_layout(long long m, int n, int k) {
  Fp8TrainLayout l;
  l.xt = fp8_bytes(k, m);
  l.wt = fp8_bytes(k, n);
  l.saved = l.xt + l.wt;
  l.x = fp8_bytes(m, k);
  l.w = fp8_bytes(n, k);
  l.ws_fwd = l.x + l.w;
  l.g = fp8_bytes(m, n);
  l.gt = fp8_bytes(n, m);
  l.colsum = pn_align_up((size_t)((m + 127) / 128) * n * 4, 256);
  l.ws_bwd = l.g + l.gt + l.colsum;
  return l;
}
static int fp8_train_check(int dtype, int w_dtype, long long m, int n, int k, const void* p, const void* saved, const void* ws) {
  PN_CHECK_ARG((dtype == PN_DTYPE_F32 || dtype == PN_DTYPE_BF16) && (w_dtype == PN_DTYPE_F32 || w_dtype == PN_DTYPE_BF16),
               "fp8_linear_train: element types %d, %d (fp32 or bf16)", dtype, w_dtype);
  PN_CHECK_ARG(m >= 1 && n >= 1 && k >= 1 && m <= 1 << 22 && n <= 1 << 22 && k <= 1 << 22, "fp8_linear_train: %lld x %d x %d", m, n, k);
  PN_CHECK_ARG(p && saved && ws && (((uintptr_t)saved | (uintptr_t)ws) & 255) == 0,
               "fp8_linear_train: null pointer, or saved operands / workspace off their 256-byte alignment");
  return PN_OK;
}
extern "C" size_t pn_fp8_train_saved_bytes(long long m, int n, int k) { return m < 1 || n < 1 || k < 1 ? 0 : fp8_train_layout(m, n, k).saved; }
extern "C" size_t pn_fp8_train_workspace_bytes(long long m, int n, int k, int backward) {
  if (m < 1 || n < 1 || k < 1) return 0;
  return backward ? fp8_train_layout(m, n, k).ws_bwd : fp8_train_layout(m, n, k).ws_fwd;
}

extern "C" int pn_fp8_train_forward(int dtype, const void* x, long long m, long long ldx, int w_dtype, const void* w, int n, int k, long long ldw,
                                    const void* bias, int bias_dtype, void* y, int save_x, int save_w, void* saved, void* ws, void* stream) {
  int rc = fp8_train_check(dtype, w_dtype, m, n, k, x, saved, ws);
  if (rc == PN_OK) rc = fp8_check(ws, m, n, k, bias, bias_dtype, PN_ACT_NONE, dtype, y, n);
  if (rc != PN_OK) return rc;
  PN_CHECK_ARG(w && (m == 1 || ldx >= k) && (n == 1 || ldw >= k), "pn_fp8_train_forward: weight missing or a row stride below the row length");
  const Fp8TrainLayout l = fp8_train_layout(m, n, k);
  char *sv = (char*)saved, *wk = (char*)ws;
  hipStream_t s = (hipStream_t)stream;
  rc = fp8_quantize_launch(Fp8QuantJob{x, dtype, 1, m, ldx, k, wk, save_x ? sv : nullptr, nullptr}, s);
  if (rc == PN_OK) rc = fp8_quantize_launch(Fp8QuantJob{w, w_dtype, 128, n, ldw, k, wk + l.x, save_w ? sv + l.xt : nullptr, nullptr}, s);
  if (rc == PN_OK)
    rc = fp8_gemm_launch(Fp8Gemm{fp8_operand(wk, m, k), fp8_operand(wk + l.x, n, k), m, n, k, bias, bias_dtype, PN_ACT_NONE, dtype, y, n}, s);
  return rc;
}

int fp8_colsum_launch(const float* partial, long long rows, int cols, int out_dtype, void* out, hipStream_t s);

extern "C" int pn_fp8_train_backward(int dtype, const void* g, long long m, long long ldg, int w_dtype, int n, int k, const void* saved, void* dx,
                                     void* dw, void* db, int db_dtype, void* ws, void* stream) {
  int rc = fp8_train_check(dtype, w_dtype, m, n, k, g, saved, ws);
  if (rc != PN_OK) return rc;
  PN_CHECK_ARG(m == 1 || ldg >= n, "pn_fp8_train_backward: row stride below the row length");
  PN_CHECK_ARG(!db || db_dtype == PN_DTYPE_F32 || db_dtype == PN_DTYPE_BF16, "pn_fp8_train_backward: bias type %d (fp32 or bf16)", db_dtype);
  if (!dx && !dw && !db) return PN_OK;
  const Fp8TrainLayout l = fp8_train_layout(m, n, k);
  const char* sv = (const char*)saved;
  char *gq = (char*)ws, *gt = gq + l.g;
  float* cs = (float*)(gt + l.gt);
  hipStream_t s = (hipStream_t)stream;
  rc = fp8_quantize_launch(Fp8QuantJob{g, dtype, 1, m, ldg, n, dx ? gq : nullptr, dw ? gt : nullptr, db ? cs : nullptr}, s);
  if (rc == PN_OK && dx)
    rc = fp8_gemm_launch(Fp8Gemm{fp8_operand(gq, m, n), fp8_operand(sv + l.xt, k, n), m, k, n, nullptr, 0, PN_ACT_NONE, dtype, dx, k}, s);
  if (rc == PN_OK && dw)
    rc = fp8_gemm_launch(Fp8Gemm{fp8_operand(gt, n, m), fp8_operand(sv, k, m), n, k, (int)m, nullptr, 0, PN_ACT_NONE, w_dtype, dw, k}, s);
  if (rc == PN_OK && db) rc = fp8_colsum_launch(cs, m, n, db_dtype, db, s);
  return rc;
}
