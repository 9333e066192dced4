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
__device__ __forceinline__ uint32_t philox_u16(const uint32_t (&c)[4], int i) { return (c[i >> 1] >> (16 * (i & 1))) & 0xffffu; }

// keep decisions of the eight elements that start at linear index e (a group boundary or not): bit i set = kept
__device__ __forceinline__ uint32_t keep_bits8(const PhiloxKey& k, unsigned long long e, uint32_t threshold) {
  uint32_t c[4], bits = 0;
  philox(k, e >> 3, c);
#pragma unroll
  for (int i = 0; i < 8; ++i) bits |= (philox_u16(c, i) >= threshold ? 1u : 0u) << i;
  const int sh = (int)(e & 7);
  if (sh) {
    uint32_t hi = 0;
    philox(k, (e >> 3) + 1, c);
#pragma unroll
    for (int i = 0; i < 8; ++i) hi |= (philox_u16(c, i) >= threshold ? 1u : 0u) << i;
    bits = ((bits | hi << 8) >> sh) & 0xffu;
  }
  return bits;
}

__device__ __forceinline__ float gelu_f(float x) { return 0.5f * x * (1.f + erff(x * 0.70710678118654752f)); }
__device__ __forceinline__ float gelu_grad_f(float x) {
  return fmaf(x * 0.39894228040143268f, expf(-0.5f * x * x), 0.5f * (1.f + erff(x * 0.70710678118654752f)));
}
__device__ __forceinline__ float act_f(float x, int act) {
  if (act == PN_ACT_RELU) return x <= 0.f ? 0.f : x;         // NaN stays NaN, as torch.relu
  if (act == PN_ACT_GELU) return gelu_f(x);
  return x;
}
