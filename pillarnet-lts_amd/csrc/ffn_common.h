// Shared by the operators of the feed-forward block (ffn_dropout.hip, ffn_norm.hip, fp8_quant.hip, fp8_gemm.hip):
// eight-element pieces of a row in registers, the counter-based generator and the activations.
#pragma once
#include "common.h"

// Eight consecutive elements as fp32.  Global memory takes 16-byte accesses at any element alignment, so odd row strides
// use the same instructions; `n` < 8 (the last piece of a row) goes element by element and fills with zeros.
template <typename T> struct Piece8;
template <> struct Piece8<float> {
  struct __attribute__((packed, aligned(4))) Raw { float v[4]; };
  static __device__ __forceinline__ void load(const float* p, float (&o)[8]) {
    const Raw a = *reinterpret_cast<const Raw*>(p), b = *reinterpret_cast<const Raw*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { o[i] = a.v[i]; o[4 + i] = b.v[i]; }
  }
  static __device__ __forceinline__ void store(float* p, const float (&o)[8]) {
    Raw a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) { a.v[i] = o[i]; b.v[i] = o[4 + i]; }
    *reinterpret_cast<Raw*>(p) = a;
    *reinterpret_cast<Raw*>(p + 4) = b;
  }
};
template <> struct Piece8<__bf16> {
  struct __attribute__((packed, aligned(2))) Raw { __bf16 v[8]; };
  static __device__ __forceinline__ void load(const __bf16* p, float (&o)[8]) {
    const Raw a = *reinterpret_cast<const Raw*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)a.v[i];
  }
  static __device__ __forceinline__ void store(__bf16* p, const float (&o)[8]) {
    Raw a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a.v[i] = (__bf16)o[i];      // round to nearest even
    *reinterpret_cast<Raw*>(p) = a;
  }
};
template <typename T> __device__ __forceinline__ void load8(const T* p, int n, float (&o)[8]) {
  if (n >= 8) {
    Piece8<T>::load(p, o);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = i < n ? (float)p[i] : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, int n, const float (&o)[8]) {
  if (n >= 8) {
    Piece8<T>::store(p, o);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (T)o[i];
  }
}

// Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): a keyed
// bijection of a 128-bit counter.  One counter serves the eight elements of group j = (row * cols + col) / 8, 16 bits
// each: a keep decision needs no more, and 32 bits each would double the integer work that bounds the kernel.
// counter = (j low, (j high & 0xffff) | call << 16, offset low, offset high), key = seed.
struct PhiloxKey {
  uint32_t k0, k1, o0, o1, call;
};
__device__ __forceinline__ PhiloxKey philox_key(const unsigned long long* rng, uint32_t call) {
  const unsigned long long seed = rng[0], off = rng[1];
  return PhiloxKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)off, (uint32_t)(off >> 32), call << 16};
}
__device__ __forceinline__ void philox(const PhiloxKey& k, unsigned long long group, uint32_t (&c)[4]) {
  c[0] = (uint32_t)group;
  c[1] = ((uint32_t)(group >> 32) & 0xffffu) | k.call;
  c[2] = k.o0;
  c[3] = k.o1;
  uint32_t k0 = k.k0, k1 = k.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)c[0] * 0xD2511F53u, b = (unsigned long long)c[2] * 0xCD9E8D57u;
    c[0] = (uint32_t)(b >> 32) ^ c[1] ^ k0;
    c[1] = (uint32_t)b;
    c[2] = (uint32_t)(a >> 32) ^ c[3] ^ k1;
    c[3] = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// Keep decisions of eight elements: element i is kept if its 16 bits are >= threshold, compared in the upper half of a word, so
// that every second one needs no shift.  `past` = (threshold - 1) << 16 | 0xffff: > past means the half is >= threshold.
struct Keep8 {
  uint32_t c[4], past;
  __device__ __forceinline__ bool operator()(int i) const { return (i & 1 ? c[i >> 1] : c[i >> 1] << 16) > past; }
};
// threshold 1 .. 65536; without dropping (0) the caller takes the others' branch: everything is kept
__device__ __forceinline__ uint32_t keep_past(uint32_t threshold) { return (threshold - 1) << 16 | 0xffffu; }
__device__ __forceinline__ Keep8 keep_all() { return Keep8{{~0u, ~0u, ~0u, ~0u}, 0x80000000u}; }
__device__ __forceinline__ Keep8 keep8_group(const PhiloxKey& k, unsigned long long group, uint32_t threshold) {
  Keep8 o;
  o.past = keep_past(threshold);
  philox(k, group, o.c);
  return o;
}
// ... that start at linear index e, a group's first element or not: bits of two groups, spread to whole halves (0xffff is kept)
__device__ __forceinline__ Keep8 keep8_at(const PhiloxKey& k, unsigned long long e, uint32_t threshold) {
  Keep8 o = keep8_group(k, e >> 3, threshold);
  const int sh = (int)(e & 7);
  if (sh) {
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) bits |= o(i) ? 1u << i : 0u;
    philox(k, (e >> 3) + 1, o.c);
#pragma unroll
    for (int i = 0; i < 8; ++i) bits |= o(i) ? 256u << i : 0u;
    bits >>= sh;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.c[i] = (bits >> (2 * i) & 1) * 0xffffu | (bits >> (2 * i + 1) & 1) * 0xffff0000u;
  }
  return o;
}

// GELU from the normal distribution's tail: with z = |x| / sqrt(2), q = Phi(-|x|) = exp(-z^2) * erfcx(z) / 2, and
// gelu(x) = max(x, 0) - |x| q, which cancels nowhere.  erfcx(z) / 2 = t P(t), t = 1 / (1 + z / 2): P is a weighted least
// squares fit of degree 9 made for this file (2.9e-8 relative over z in [0, 10]; beyond, exp(-z^2) underflows).  About 90
// cycles a wave against about 200 for erff's two branches; the epilogue of a large product waits for it.
__device__ __forceinline__ void gelu_parts(float x, float& ax, float& q, float& e) {
  ax = fminf(fabsf(x), 30.f);                                  // (q is zero long before; an infinity must not meet it)
  const float z = ax * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(fmaf(0.5f, z, 1.f));
  e = __builtin_amdgcn_exp2f(z * z * -1.4426950408889634f);
  float p = 0.006141550373286009f;
  p = fmaf(p, t, -0.06162668392062187f);
  p = fmaf(p, t, 0.2144658863544464f);
  p = fmaf(p, t, -0.33501750230789185f);
  p = fmaf(p, t, 0.2106454223394394f);
  p = fmaf(p, t, -0.049164727330207825f);
  p = fmaf(p, t, 0.11277339607477188f);
  p = fmaf(p, t, 0.11932181566953659f);
  p = fmaf(p, t, 0.14142858982086182f);
  p = fmaf(p, t, 0.14103224873542786f);
  q = t * p * e;
}
__device__ __forceinline__ float gelu_f(float x) {
  float ax, q, e;
  gelu_parts(x, ax, q, e);
  return (x <= 0.f ? 0.f : x) - ax * q;                        // (x <= 0 is false for NaN, which passes)
}
__device__ __forceinline__ float gelu_grad_f(float x) {        // Phi(x) + x phi(x)
  float ax, q, e;
  gelu_parts(x, ax, q, e);
  const float phi = x <= 0.f ? q : 1.f - q, d = ax * e * 0.39894228040143268f;
  return x <= 0.f ? phi - d : x > 0.f ? phi + d : x;
}
__device__ __forceinline__ float act_f(float x, int act) {
  if (act == PN_ACT_RELU) return x <= 0.f ? 0.f : x;         // NaN stays NaN, as torch.relu
  if (act == PN_ACT_GELU) return gelu_f(x);
  return x;
}

// The same for a result that is about to be rounded to bf16 (half a step: 2^-8): q = 2^P(|x|) with P a fit of degree 5 to
// log2 Phi(-a), 2.6e-4 = 2^-11.9 relative over a in [0, 5.5] (beyond, q < 2e-8, P falls on), and no reciprocal: half the cycles.
__device__ __forceinline__ float act_bf16(float x, int act) {
  const float r = x <= 0.f ? 0.f : x;
  if (act == PN_ACT_RELU) return r;
  if (act != PN_ACT_GELU) return x;
  const float a = fminf(fabsf(x), 30.f);
  float p = -0.00023323729692492634f;
  p = fmaf(p, a, 0.004869362805038691f);
  p = fmaf(p, a, -0.04459570348262787f);
  p = fmaf(p, a, -0.4696913957595825f);
  p = fmaf(p, a, -1.1462488174438477f);
  p = fmaf(p, a, -1.000362753868103f);
  return fmaf(-a, __builtin_amdgcn_exp2f(p), r);
}

// ---- e4m3 with a power-of-two scale a block ----
// Magnitudes are compared as integers (they order like their bit patterns); a block's scale byte e + 127 belongs to the
// smallest e >= -126 with the largest finite magnitude <= 448 * 2^e = 1.75 * 2^(e + 8).
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ int block_scale(uint32_t bits) {
  const int b = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b < 1 ? 1 : b;
}
__device__ __forceinline__ float scale_value(uint32_t byte) { return __uint_as_float(byte << 23); }      // 2^(byte - 127)

typedef __attribute__((ext_vector_type(2))) unsigned short ffn_u16x2;
typedef __attribute__((ext_vector_type(2))) short ffn_s16x2;
typedef __attribute__((ext_vector_type(2))) __bf16 ffn_bf16x2;

// Eight elements as they are stored; Mag: their running largest magnitudes (bf16: two at a time).  The instruction that rounds
// to e4m3 divides by the scale on the way (exact for powers of two), rounds to nearest even and turns what is not finite into NaN.
template <typename T> struct Raw8;
template <> struct Raw8<float> {
  static constexpr int MAGS = 8;                        // column magnitudes of a piece
  float v[8];
  __device__ __forceinline__ void load(const float* p) { Piece8<float>::load(p, v); }
  __device__ __forceinline__ void load_part(const float* p, int n) {      // elements from n on are zero (n >= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[i < n ? i : n - 1];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= n) v[i] = 0.f;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
  __device__ __forceinline__ void fill(float f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f;
  }
  __device__ __forceinline__ uint4 words(int j) const {
    return make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
  }
  __device__ __forceinline__ void set_words(int j, uint4 w) {
    v[4 * j] = __uint_as_float(w.x);
    v[4 * j + 1] = __uint_as_float(w.y);
    v[4 * j + 2] = __uint_as_float(w.z);
    v[4 * j + 3] = __uint_as_float(w.w);
  }
  __device__ __forceinline__ float get(int i) const { return v[i]; }
  template <bool FINITE> __device__ __forceinline__ uint32_t mag(int i) const {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    return FINITE && b >= 0x7f800000u ? 0u : b;
  }
  static __device__ __forceinline__ uint32_t mag_max(uint32_t a, uint32_t b) { return umax(a, b); }
  template <bool FINITE> __device__ __forceinline__ uint32_t row_mag() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = umax(m, mag<FINITE>(i));
    return m;
  }
  static __device__ __forceinline__ uint32_t mag_bits(uint32_t m) { return m; }               // as fp32 bits
  static __device__ __forceinline__ uint32_t col_bits(const uint32_t* m, int j) { return m[j]; }
  static __device__ __forceinline__ bool mag_inf(uint32_t m) { return m >= 0x7f800000u; }
  __device__ __forceinline__ uint2 quant(float s) const {
    ffn_s16x2 a = {0, 0}, b = {0, 0};
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[0], v[1], s, false);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[2], v[3], s, true);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[4], v[5], s, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[6], v[7], s, true);
    return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
  }
  static __device__ __forceinline__ uint2 quant_col(const Raw8 (&r)[8], int j, float s) {      // column j of eight rows
    ffn_s16x2 a = {0, 0}, b = {0, 0};
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, r[0].v[j], r[1].v[j], s, false);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, r[2].v[j], r[3].v[j], s, true);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, r[4].v[j], r[5].v[j], s, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, r[6].v[j], r[7].v[j], s, true);
    return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
  }
};
template <> struct Raw8<__bf16> {
  static constexpr int MAGS = 4;
  uint32_t v[4];
  struct __attribute__((packed, aligned(2))) Mem { uint32_t v[4]; };
  __device__ __forceinline__ void load(const __bf16* p) {
    const Mem m = *reinterpret_cast<const Mem*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = m.v[i];
  }
  __device__ __forceinline__ void load_part(const __bf16* p, int n) {
    const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
    uint32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = q[i < n ? i : n - 1];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (2 * i < n ? e[2 * i] : 0u) | (2 * i + 1 < n ? e[2 * i + 1] << 16 : 0u);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 0u;
  }
  __device__ __forceinline__ void fill(float f) {          // f: a bf16 value
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (__float_as_uint(f) >> 16) * 0x10001u;
  }
  __device__ __forceinline__ uint4 words(int) const { return make_uint4(v[0], v[1], v[2], v[3]); }
  __device__ __forceinline__ void set_words(int, uint4 w) {
    v[0] = w.x;
    v[1] = w.y;
    v[2] = w.z;
    v[3] = w.w;
  }
  __device__ __forceinline__ float get(int i) const { return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16); }
  template <bool FINITE> __device__ __forceinline__ uint32_t mag(int i) const {
    uint32_t b = v[i] & 0x7fff7fffu;
    if (FINITE) {
      if ((b & 0xffffu) >= 0x7f80u) b &= 0xffff0000u;
      if (b >= 0x7f800000u) b &= 0xffffu;
    }
    return b;
  }
  static __device__ __forceinline__ uint32_t mag_max(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ffn_u16x2, a), __builtin_bit_cast(ffn_u16x2, b)));
  }
  template <bool FINITE> __device__ __forceinline__ uint32_t row_mag() const {
    return mag_max(mag_max(mag<FINITE>(0), mag<FINITE>(1)), mag_max(mag<FINITE>(2), mag<FINITE>(3)));
  }
  static __device__ __forceinline__ uint32_t mag_bits(uint32_t m) { return umax(m & 0xffff0000u, m << 16); }
  static __device__ __forceinline__ uint32_t col_bits(const uint32_t* m, int j) { return j & 1 ? m[j >> 1] & 0xffff0000u : m[j >> 1] << 16; }
  static __device__ __forceinline__ bool mag_inf(uint32_t m) { return m >= 0x7f800000u || (m & 0xffffu) >= 0x7f80u; }
  static __device__ __forceinline__ uint32_t cvt4(uint32_t lo, uint32_t hi, float s) {
    ffn_s16x2 a = {0, 0};
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, __builtin_bit_cast(ffn_bf16x2, lo), s, false);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, __builtin_bit_cast(ffn_bf16x2, hi), s, true);
    return __builtin_bit_cast(uint32_t, a);
  }
  __device__ __forceinline__ uint2 quant(float s) const { return make_uint2(cvt4(v[0], v[1], s), cvt4(v[2], v[3], s)); }
  static __device__ __forceinline__ uint2 quant_col(const Raw8 (&r)[8], int j, float s) {
    const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;                 // halves of two rows side by side
    const int d = j >> 1;
    return make_uint2(cvt4(__builtin_amdgcn_perm(r[1].v[d], r[0].v[d], sel), __builtin_amdgcn_perm(r[3].v[d], r[2].v[d], sel), s),
                      cvt4(__builtin_amdgcn_perm(r[5].v[d], r[4].v[d], sel), __builtin_amdgcn_perm(r[7].v[d], r[6].v[d], sel), s));
  }
};
// over the 16 lanes of a row group: lane i ^ 1, i ^ 2, then the mirrored half and the mirrored row
template <typename R> __device__ __forceinline__ uint32_t mag_max16(uint32_t m) {
  m = R::mag_max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, true));
  m = R::mag_max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, true));
  m = R::mag_max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xf, 0xf, true));
  return R::mag_max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xf, 0xf, true));
}

// An operand of a product in fp8, [rows, cols] with the contraction along cols, in one allocation:
//   bytes   [ceil(rows / 16)][ceil(cols / 128)] tiles of 2 KB, a tile being what a wave multiplies: 16 rows x one block of 128, as
//           two planes of 64 x 16 bytes; entry l of plane h holds row l & 15, k = (l >> 4) * 32 + h * 16 .. + 15, so a fragment is
//           two 16-byte reads at lane * 16 from memory (one run of 2 KB) or from LDS (all banks once).  In rows, neighbouring
//           lanes would read different rows: 64 lines an instruction (measured: a block of 16 rows then took a CU 540 cycles);
//   scales  (256-byte aligned behind them) words [ceil(blocks / 4)][rows], byte b & 3 of word (b >> 2, row) = e + 127 of block b.
struct Fp8Operand {
  const unsigned char* q;
  const uint32_t* scale;
};
static inline __host__ __device__ size_t fp8_q_bytes(long long rows, long long cols) {
  return (size_t)((rows + 15) / 16) * (size_t)((cols + 127) / 128) * 2048;
}
static inline size_t fp8_bytes(long long rows, long long cols) {
  return pn_align_up(fp8_q_bytes(rows, cols) + (size_t)((cols + 511) / 512) * (size_t)rows * 4, 256);
}
static inline Fp8Operand fp8_operand(const void* p, long long rows, long long cols) {
  const unsigned char* q = (const unsigned char*)p;
  return Fp8Operand{q, (const uint32_t*)(q ? q + fp8_q_bytes(rows, cols) : nullptr)};
}

// fp8_quant.hip, fp8_gemm.hip: launches without argument checks
struct Fp8QuantJob {
  const void* x;
  int dtype, block_rows;
  long long rows, ldx;
  int cols;
  void *q, *qt;             // operands to write: x, its transpose (either may be NULL)
  float* colsum;            // [ceil(rows / 128)][cols] or NULL
};
int fp8_quantize_launch(const Fp8QuantJob& j, hipStream_t s);
struct Fp8Gemm {
  Fp8Operand x, w;
  long long M;
  int N, K;
  const void* bias;
  int bias_dtype, act, out_dtype;
  void* out;
  long long ldo;
};
int fp8_gemm_launch(const Fp8Gemm& g, hipStream_t s);
