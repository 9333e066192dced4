// Residual join with the norms on its two sides, gate, scale and dropout:
//   u = post(f)   v = dropout(u)   h = round(x + scale * gate * v)   y = act(norm(h))
// post / norm: layer (mean and variance over the row), rms, affine (weight and bias only), none.  One launch per direction
// instead of up to a dozen; every row is read once and kept in registers between its two norms.
//
// Statistics are two-pass (mean, then the mean of squared distances) in fp32 over the registers.  The norm reads h as it is
// stored, so the backward pass, which reads the stored h again, differentiates exactly what was computed.
//
// Bound by memory, with the next row on its way while one is worked on: 32768 x 4096 bf16, layer scale and LayerNorm, 199 us
// (5.4 TB/s); 65536 x 256 fp32, LayerNorm, 42 us (6.4 TB/s).  With both norms, gate and dropout (16 x 1031 x 2048 bf16: forward
// 57 us, 4.8 TB/s; backward 91 us, 4.4 TB/s, and 7 for the column sums) the generator and two sums across each row leave too
// few waves to hide all of it.  Slower than that: rows whose length is no multiple of eight (16 x 1031 x 2047: 78 and 124 us), and rows
// a little over a power of two (4096 x 4200 bf16, both norms: forward 65 us, 2.1 TB/s: one workgroup of twelve waves on a CU, nine of
// them with columns).
//
// Small launches (512 x 49 x 64 fp32, LayerNorm: 9 us forward and 10 backward for 26 MB each, 3 TB/s) are one pass of 784 workgroups: the
// launch, one trip to memory there and one back, and nothing to hide them behind.
//
// Where registers do not suffice (bytes of scratch a lane as the compiler reports them):
//   backward with a branch, 4097 - 8192 columns: 32 - 36 for bf16 rows with fp32 parameters, 100 - 116 for fp32 rows, none for bf16 with
//     bf16 parameters (4096 x 8192, both norms: 131, 244 and 115 us; the rows are 403 MB in bf16);
//   forward over 8192 columns, where 1024 threads have 128 registers for 16 columns each: 172 - 324 with post norm or dropout (2048 x
//     16384, both norms: bf16 131 us, fp32 257), up to 100 without (LayerNorm: 59 and 153);
//   backward over 8192 columns: 780 - 1108 with a branch that is read (bf16 761 us, fp32 1166: 0.5 - 0.7 TB/s), 276 - 408 otherwise (164, 302).
// The backward kernel that reads the branch keeps five column sums whatever is asked for: with dropout or a gate alone it is hardly faster.
#include "ffn_common.h"

struct NormArgs {
  pnResidualNorm p;
  const void *gh, *gy;
  void *h, *y, *dx, *df;
  void* dgate_rows;        // backward with a gate for each row: its gradient needs no sum over rows
  float* stats;            // [rows][4]: mean and factor of the norm, mean and factor of the post norm
  float* partial;          // backward: [chunks][sums][cols]
  int chunk_rows;          // rows of one chunk (a multiple of the workgroup's row slots), chunks never span two gates
  int chunks_per_group;
  long long group_rows;
  float keep_scale;
};

// a + its neighbour's: lanes 1, 2, 4, 8 apart by DPP (past the first two as mirrored half and whole rows of 16, whose quads agree by
// then), rows 16 and 32 apart by the swap of two registers' rows.  No trip through LDS, where a shuffle takes some 100 cycles.
template <int O> __device__ __forceinline__ float add_across(float v) {
  const int i = __float_as_int(v);
  if constexpr (O <= 8) {
    constexpr int CTRL = O == 1 ? 0xB1 : O == 2 ? 0x4E : O == 4 ? 0x141 : 0x140;
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, i, CTRL, 0xf, 0xf, true));
  } else if constexpr (O == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(i, i, false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
  }
}
template <int W> __device__ __forceinline__ float lanes_sum(float v) {
  if (W > 1) v = add_across<1>(v);
  if (W > 2) v = add_across<2>(v);
  if (W > 4) v = add_across<4>(v);
  if (W > 8) v = add_across<8>(v);
  if (W > 16) v = add_across<16>(v);
  if (W > 32) v = add_across<32>(v);
  return v;
}

// Sums over the L threads that share a row (L <= 64: across the lanes; more, or L = 0 for the whole workgroup: one LDS exchange,
// two buffers so that one barrier is enough).  The order of the additions depends on L (or the workgroup's size) alone.
template <int L, int NT> struct RowSum {
  static constexpr int SLOTS = 16;
  float2* lds;             // [2][SLOTS]
  int turn = 0;
  __device__ __forceinline__ explicit RowSum(float2* buf) : lds(buf) {
    if (L == 0) {          // the places of the waves that there are not
      if (threadIdx.x < 2 * SLOTS) lds[threadIdx.x] = make_float2(0.f, 0.f);
      __syncthreads();
    }
  }
  template <bool TWO> __device__ __forceinline__ float2 sums(float a, float b) {
    constexpr int W = L >= 1 && L < 64 ? L : 64, WAVES = L == 0 ? SLOTS : L > 64 ? L / 64 : 1;
    a = lanes_sum<W>(a);
    if (TWO) b = lanes_sum<W>(b);
    if (WAVES > 1) {
      float2* buf = lds + turn * SLOTS;
      turn ^= 1;
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) buf[wave] = make_float2(a, b);
      __syncthreads();
      const float2 v = buf[(L == 0 ? 0 : wave & ~(WAVES - 1)) + (threadIdx.x & (WAVES - 1))];
      a = lanes_sum<WAVES>(v.x);
      if (TWO) b = lanes_sum<WAVES>(v.y);
    }
    return make_float2(a, b);
  }
  __device__ __forceinline__ float2 operator()(float a, float b) { return sums<true>(a, b); }
  __device__ __forceinline__ float operator()(float a) { return sums<false>(a, 0.f).x; }
};

// Columns of a thread: K pieces of eight, l threads a row.  EXACT: the row is l * 8 * K wide, every thread owns all of its pieces.  RAGGED (at
// least 8 wide): a piece that would reach past the row's end is moved back onto its last eight columns; the columns that it then
// shares with its neighbour are computed twice and counted once.  So every load is whole and unconditional: a load behind a branch
// of its own waits for the one before it.  TINY: fewer than eight columns, all of them the first thread's.
enum { EXACT, RAGGED, TINY };
template <int K, int MODE> struct Cols {
  int c[K], dup[K];          // first column, columns that another thread owns
  int n;
  __device__ __forceinline__ Cols(int t, int l, int C) : n(C) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int at = (k * l + t) * 8;
      c[k] = MODE == EXACT ? at : MODE == RAGGED ? min(at, C - 8) : 0;
      dup[k] = MODE == EXACT ? 0 : MODE == RAGGED ? at - c[k] : t == 0 ? 0 : 8;
    }
  }
  __device__ __forceinline__ bool mine(int k, int i) const {
    return MODE == EXACT ? true : MODE == RAGGED ? i >= dup[k] : dup[k] == 0 && i < n;
  }
  __device__ __forceinline__ bool any(int k) const { return MODE == EXACT ? true : dup[k] < 8; }
  template <typename T> __device__ __forceinline__ void raw(const T* row, int k, Raw8<T>& o) const {
    if (MODE == TINY) o.load_part(row, n);
    else o.load(row + c[k]);
  }
  template <typename T> __device__ __forceinline__ void store(T* row, int k, const float (&v)[8]) const {
    if (MODE != TINY) Piece8<T>::store(row + c[k], v);
    else store8(row, n, v);
  }
  template <typename P> __device__ __forceinline__ void param(const void* p, int k, Raw8<P>& o, float fill) const {
    o.fill(fill);
    if (p) raw(reinterpret_cast<const P*>(p), k, o);
  }
};

// The gate's row of a row that advances by `step` rows at a time: no division in the loop.
struct GateRow {
  long long row, rest, by, by_rest, per;
  __device__ __forceinline__ GateRow(long long first, long long step, long long rows_per_gate) : per(rows_per_gate) {
    row = first / per;
    rest = first - row * per;
    by = step / per;
    by_rest = step - by * per;
  }
  __device__ __forceinline__ void next() {
    row += by;
    rest += by_rest;
    if (rest >= per) {
      rest -= per;
      ++row;
    }
  }
};

// mean and 1 / sqrt(var + eps) of the row held as v[K][8]
template <int K, typename Own, typename Sum>
__device__ __forceinline__ float2 row_stats(const float (&v)[K][8], int kind, float eps, const Own& own, Sum& sum) {
  if (kind != PN_NORM_LAYER && kind != PN_NORM_RMS) return make_float2(0.f, 1.f);
  float mean = 0.f, s = 0.f;
  if (kind == PN_NORM_LAYER) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += own.mine(k, i) ? v[k][i] : 0.f;
    mean = sum(s) / (float)own.n;
  }
  s = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = v[k][i] - mean;
      s = own.mine(k, i) ? fmaf(d, d, s) : s;
    }
  const float var = sum(s) / (float)own.n;
  return make_float2(mean, 1.f / sqrtf(var + eps));
}

// L threads a row, NT a workgroup; L = 0: the workgroup, of up to NT threads, has one row.
// FULL: the branch passes a post norm or dropout (with the registers that takes); otherwise gate and scale only.
template <typename T, typename P, int L, int K, int NT, int MODE, bool FULL>
__global__ __launch_bounds__(NT) void residual_norm_fwd_kernel(NormArgs a) {
  constexpr int SLOTS = L ? NT / L : 1;
  __shared__ float2 lds[2 * RowSum<L, NT>::SLOTS];
  RowSum<L, NT> sum(lds);
  const pnResidualNorm& p = a.p;
  const int slot = L ? threadIdx.x / L : 0, t = L ? threadIdx.x % L : threadIdx.x, C = p.cols;
  const Cols<K, MODE> own(t, L ? L : blockDim.x, C);
  const T* X = reinterpret_cast<const T*>(p.x);
  const T* F = reinterpret_cast<const T*>(p.branch);
  const P* G = reinterpret_cast<const P*>(p.gate);
  T* H = reinterpret_cast<T*>(a.h);
  T* Y = reinterpret_cast<T*>(a.y);
  PhiloxKey key{};
  if (FULL && p.threshold) key = philox_key(reinterpret_cast<const unsigned long long*>(p.rng), p.call);
  auto draw = [&](long long row, int c) {                 // rows of whole pieces start at a group of the generator
    const unsigned long long e = (unsigned long long)row * C + c;
    return MODE == EXACT || (C & 7) == 0 ? keep8_group(key, e >> 3, p.threshold) : keep8_at(key, e, p.threshold);
  };
  Raw8<P> nw[K], nb[K], pw[FULL ? K : 1], pb[FULL ? K : 1];     // as they are stored: bf16 takes half the registers
#pragma unroll
  for (int k = 0; k < K; ++k) {
    own.param(p.norm_weight, k, nw[k], 1.f);
    own.param(p.norm_bias, k, nb[k], 0.f);
    if (FULL) {
      own.param(p.post_weight, k, pw[k], 1.f);
      own.param(p.post_bias, k, pb[k], 0.f);
    }
  }
  // The next row (and its gate) is on its way while this one is worked on; nothing is loaded in between, as waiting for a
  // later load would wait for these too.  Past the last row the loads repeat it.
  const long long step = (long long)gridDim.x * SLOTS, first = (long long)blockIdx.x * SLOTS + slot;
  GateRow gate(first, step, p.rows_per_gate);
  Raw8<T> nx[K], nf[K];
  Raw8<P> ng[K];
  auto fetch = [&](long long row) {
    const bool in = row < p.rows;
    row = in ? row : p.rows - 1;
#pragma unroll
    for (int k = 0; k < K; ++k) own.raw(X + row * p.ldx, k, nx[k]);
    if (F) {
#pragma unroll
      for (int k = 0; k < K; ++k) own.raw(F + row * p.ldb, k, nf[k]);
    }
    if (G) {
#pragma unroll
      for (int k = 0; k < K; ++k) own.raw(G + (in ? gate.row * C : 0), k, ng[k]);
    }
  };
  fetch(first);
  for (long long base = (long long)blockIdx.x * SLOTS; base < p.rows; base += step) {
    const bool live = base + slot < p.rows;
    const long long row = live ? base + slot : p.rows - 1;
    float h[K][8], f[K][8], g[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[k][i] = nx[k].get(i);
        f[k][i] = F ? nf[k].get(i) : 0.f;
        g[k][i] = G ? p.scale * ng[k].get(i) : p.scale;
      }
    gate.next();
    if (base + step < p.rows) fetch(base + step + slot);
    float2 fs = make_float2(0.f, 1.f);
    if (F) {
      if (FULL) fs = row_stats<K>(f, p.post_kind, p.post_eps, own, sum);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        Keep8 keep = keep_all();
        if (FULL && p.threshold) keep = draw(row, own.c[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float u = f[k][i];
          if (FULL) {
            if (p.post_kind != PN_NORM_NONE) u = fmaf((u - fs.x) * fs.y, pw[k].get(i), pb[k].get(i));
            u = keep(i) ? u * a.keep_scale : 0.f;
          }
          h[k][i] = (float)(T)fmaf(g[k][i], u, h[k][i]);
        }
        if (live && own.any(k)) own.store(H + row * C, k, h[k]);
      }
    }
    float2 hs = make_float2(0.f, 1.f);
    if (Y) {
      hs = row_stats<K>(h, p.norm_kind, p.norm_eps, own, sum);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = act_f(fmaf((h[k][i] - hs.x) * hs.y, nw[k].get(i), nb[k].get(i)), p.act);
        if (live && own.any(k)) own.store(Y + row * C, k, o);
      }
    }
    if (a.stats && live && t == 0)
      *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(hs.x, hs.y, fs.x, fs.y);
  }
}

// Backward.  A workgroup owns a chunk of consecutive rows and keeps the column sums (gradients of weights, biases and gate)
// in registers over the whole chunk; its partial sums go to memory once, and residual_norm_sum_kernel adds the chunks in
// order: no atomics, the same bits on every run.
//
// Rows over 4096 wide with a branch, 16 columns a thread (at eight, 1024 threads leave 128 registers each: the sums alone are 40,
// and spilled ones wait for the next row's loads): the parameters wait in LDS, and no row is fetched ahead.  Up to 8192 columns that
// leaves little or no scratch; past them 1024 threads have 128 registers again.
static constexpr __host__ __device__ bool bwd_parks(int L, int K, int NT, bool branch) { return branch && L == 0 && K == 2 && NT == 512; }
static constexpr int NSUM_NORM = 2, NSUM_ALL = 5;      // weight, bias | post weight, post bias, gate

template <typename T, typename P, int L, int K, int NT, int MODE, bool BRANCH>
__global__ __launch_bounds__(NT) void residual_norm_bwd_kernel(NormArgs a) {
  constexpr int SLOTS = L ? NT / L : 1, NS = BRANCH ? NSUM_ALL : NSUM_NORM;
  constexpr bool PARK = bwd_parks(L, K, NT, BRANCH), AHEAD = !PARK;
  __shared__ float2 lds[2 * RowSum<L, NT>::SLOTS];
  __shared__ float cols_lds[SLOTS > 1 ? NT * 8 : 1];
  extern __shared__ __attribute__((aligned(16))) char parked[];
  RowSum<L, NT> sum(lds);
  const pnResidualNorm& p = a.p;
  const int threads = L ? L : blockDim.x, slot = L ? threadIdx.x / L : 0, t = L ? threadIdx.x % L : threadIdx.x, C = p.cols;
  const Cols<K, MODE> own(t, threads, C);
  const int group = blockIdx.x / a.chunks_per_group, chunk = blockIdx.x % a.chunks_per_group;
  const long long g_begin = (long long)group * a.group_rows, g_end = min(g_begin + a.group_rows, (long long)p.rows);
  const long long r_begin = g_begin + (long long)chunk * a.chunk_rows, r_end = min(r_begin + a.chunk_rows, g_end);
  const T* H = reinterpret_cast<const T*>(p.branch ? a.h : p.x);
  const long long ldh = p.branch ? C : p.ldx;
  const T* F = reinterpret_cast<const T*>(p.branch);
  const T* GH = reinterpret_cast<const T*>(a.gh);
  const T* GY = reinterpret_cast<const T*>(a.gy);
  PhiloxKey key{};
  if (BRANCH && p.threshold) key = philox_key(reinterpret_cast<const unsigned long long*>(p.rng), p.call);
  auto draw = [&](long long row, int c) {                 // rows of whole pieces start at a group of the generator
    const unsigned long long e = (unsigned long long)row * C + c;
    return MODE == EXACT || (C & 7) == 0 ? keep8_group(key, e >> 3, p.threshold) : keep8_at(key, e, p.threshold);
  };
  const float inv_c = 1.f / (float)C;
  const bool relu = p.act == PN_ACT_RELU;
  const P* G = reinterpret_cast<const P*>(p.gate);
  float acc[NS][K][8];
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[s][k][i] = 0.f;
  constexpr int VECS = BRANCH ? 4 : 2, WORDS = sizeof(Raw8<P>) / 16;
  Raw8<P> held[PARK ? 1 : VECS][K];
  uint4* park = reinterpret_cast<uint4*>(parked) + t;     // [VECS][K][WORDS][threads]: a thread's own places
#pragma unroll
  for (int v = 0; v < VECS; ++v)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      Raw8<P> r;
      own.param(v == 0 ? p.norm_weight : v == 1 ? (relu ? p.norm_bias : nullptr) : v == 2 ? p.post_weight : p.post_bias, k, r, v & 1 ? 0.f : 1.f);
      if (PARK) {
#pragma unroll
        for (int j = 0; j < WORDS; ++j) park[((v * K + k) * WORDS + j) * threads] = r.words(j);
      } else {
        held[PARK ? 0 : v][k] = r;
      }
    }
  auto param = [&](int v, int k) {
    if (!PARK) return held[PARK ? 0 : v][k];
    Raw8<P> r;
#pragma unroll
    for (int j = 0; j < WORDS; ++j) r.set_words(j, park[((v * K + k) * WORDS + j) * threads]);
    return r;
  };

  Raw8<T> ngh[K], ngy[K], nh[K], nf[K];
  Raw8<P> ng[K];
  float4 nst = make_float4(0.f, 1.f, 0.f, 1.f);
  GateRow gate(min(r_begin + slot, r_end - 1), SLOTS, p.rows_per_gate);
  auto fetch = [&](long long row) {                      // as in the forward pass, a row ahead
    const bool in = row < r_end;
    row = in ? row : r_end - 1;
    if (BRANCH && G) {
#pragma unroll
      for (int k = 0; k < K; ++k) own.raw(G + (in ? gate.row * C : 0), k, ng[k]);
    }
    if (GY) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        own.raw(GY + row * C, k, ngy[k]);
        own.raw(H + row * ldh, k, nh[k]);
      }
    }
    if (GH) {
#pragma unroll
      for (int k = 0; k < K; ++k) own.raw(GH + row * C, k, ngh[k]);
    }
    if (BRANCH) {
#pragma unroll
      for (int k = 0; k < K; ++k) own.raw(F + row * p.ldb, k, nf[k]);
    }
    if (a.stats) nst = *reinterpret_cast<const float4*>(a.stats + row * 4);
  };
  if (AHEAD && r_begin < r_end) fetch(r_begin + slot);
  for (long long base = r_begin; base < r_end; base += SLOTS) {
    if (!AHEAD) fetch(base + slot);
    const bool live = base + slot < r_end;
    const long long row = live ? base + slot : r_end - 1;
    Raw8<T> rgh[K], rgy[K], rh[K], rf[K];
    Raw8<P> rg[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rgh[k] = ngh[k];
      rgy[k] = ngy[k];
      rh[k] = nh[k];
      rf[k] = nf[k];
      rg[k] = ng[k];
    }
    const float4 st = nst;
    gate.next();
    if (AHEAD && base + SLOTS < r_end) fetch(base + SLOTS + slot);
    float dh[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) dh[k][i] = GH ? rgh[k].get(i) : 0.f;
    if (GY) {
      float tw[K][8], hh[K][8], s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const Raw8<P> nw = param(0, k);
        Raw8<P> nb;
        if (relu) nb = param(1, k);
        else nb.fill(0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          hh[k][i] = (rh[k].get(i) - st.x) * st.y;
          float g = rgy[k].get(i);
          if (relu && fmaf(hh[k][i], nw.get(i), nb.get(i)) <= 0.f) g = 0.f;
          tw[k][i] = g * nw.get(i);
          if (live && own.mine(k, i)) {
            acc[0][k][i] = fmaf(g, hh[k][i], acc[0][k][i]);
            acc[1][k][i] += g;
          }
          if (own.mine(k, i)) {
            s1 += tw[k][i];
            s2 = fmaf(tw[k][i], hh[k][i], s2);
          }
        }
      }
      if (p.norm_kind == PN_NORM_LAYER || p.norm_kind == PN_NORM_RMS) {
        const float2 m = sum(s1, s2);
        const float m1 = p.norm_kind == PN_NORM_LAYER ? m.x * inv_c : 0.f, m2 = m.y * inv_c;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) dh[k][i] = fmaf(st.y, (tw[k][i] - m1) - hh[k][i] * m2, dh[k][i]);
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) dh[k][i] += tw[k][i];
      }
    }
    if (a.dx) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (live && own.any(k)) own.store(reinterpret_cast<T*>(a.dx) + row * C, k, dh[k]);
    }
    if (!BRANCH && a.df) {                                // a branch that is only scaled: its values are not needed
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) dh[k][i] *= p.scale;
        if (live && own.any(k)) own.store(reinterpret_cast<T*>(a.df) + row * C, k, dh[k]);
      }
    }
    if constexpr (BRANCH) {
      float fh[K][8], s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float dg[8];
        Keep8 keep = keep_all();
        if (p.threshold) keep = draw(row, own.c[k]);
        const Raw8<P> pw = param(2, k), pb = param(3, k);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          fh[k][i] = (rf[k].get(i) - st.z) * st.w;
          const float u = p.post_kind != PN_NORM_NONE ? fmaf(fh[k][i], pw.get(i), pb.get(i)) : fh[k][i];
          const bool kept = keep(i);
          const float sd = p.scale * dh[k][i], v = kept ? u * a.keep_scale : 0.f;
          const float du = kept ? (G ? rg[k].get(i) : 1.f) * sd * a.keep_scale : 0.f;
          dg[i] = sd * v;
          if (live && own.mine(k, i)) {
            acc[NS - 1][k][i] += dg[i];
            acc[NS - 3][k][i] = fmaf(du, fh[k][i], acc[NS - 3][k][i]);
            acc[NS - 2][k][i] += du;
          }
          dh[k][i] = p.post_kind != PN_NORM_NONE ? du * pw.get(i) : du;
          if (own.mine(k, i)) {
            s1 += dh[k][i];
            s2 = fmaf(dh[k][i], fh[k][i], s2);
          }
        }
        if (a.dgate_rows && live && own.any(k)) {
          own.store(reinterpret_cast<P*>(a.dgate_rows) + row * C, k, dg);
        }
      }
      if (p.post_kind == PN_NORM_LAYER || p.post_kind == PN_NORM_RMS) {
        const float2 m = sum(s1, s2);
        const float m1 = p.post_kind == PN_NORM_LAYER ? m.x * inv_c : 0.f, m2 = m.y * inv_c;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) dh[k][i] = st.w * ((dh[k][i] - m1) - fh[k][i] * m2);
      }
      if (a.df) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (live && own.any(k)) own.store(reinterpret_cast<T*>(a.df) + row * C, k, dh[k]);
      }
    }
  }

  // the chunk's sums: add the workgroup's row slots, in order, every thread a share of the columns
  float* out = a.partial + (size_t)blockIdx.x * NS * C;
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (SLOTS > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) cols_lds[(slot * 8 + i) * threads + t] = own.mine(k, i) ? acc[s][k][i] : 0.f;
        __syncthreads();
        // L * 8 columns, in the order (i, t) in which they lie; the columns that two threads share are the last one's to count
        for (int q = threadIdx.x; q < threads * 8; q += NT) {
          const int i = q / threads, tt = q % threads;
          const Cols<K, MODE> theirs(tt, threads, C);
          float v = 0.f;
#pragma unroll 8
          for (int z = 0; z < SLOTS; ++z) v += cols_lds[z * threads * 8 + q];
          if (theirs.mine(k, i)) out[s * C + theirs.c[k] + i] = v;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (own.mine(k, i)) out[s * C + own.c[k] + i] = acc[s][k][i];
      }
    }
}

// out[v][c] = sum over the chunks of vector v: blockIdx.x picks the vector (weight, bias, post weight, post bias, then
// one gate row each), blockIdx.y its 64 columns; 16 chunk lanes.  A launch holds less than 2^32 threads along x, 2^22 workgroups of this
// kernel: past SUM_GRID vectors a workgroup goes on to another.
// PARTS: blockIdx.z picks a part of SUM_PART chunks and the sums stay fp32 chunk sums, [part][sums][cols] at out[0]: with a chunk for
// each of many gates a single pass over them would be a few workgroups' (100000 gates of two rows, 256 columns: 10 ms).
static constexpr int SUM_PART = 256, SUM_GRID = 1 << 21;
struct SumArgs {
  const float *partial, *gate_partial;      // chunk sums; those of the gates' rows
  void* out[NSUM_ALL];
  int cols, sums, chunks, chunks_per_group, out_bf16, vecs;
};
template <bool PARTS> __global__ __launch_bounds__(1024) void residual_norm_sum_kernel(SumArgs a) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.y * 64 + lane;
  for (int v = blockIdx.x; v < a.vecs; v += gridDim.x) {
    const int s = v < NSUM_ALL - 1 ? v : NSUM_ALL - 1, group = PARTS ? blockIdx.z : v - s;
    void* out = a.out[PARTS ? 0 : s];
    if (!out) continue;                                                    // the same for the whole workgroup
    const bool gate = s == NSUM_ALL - 1;
    const int first = PARTS ? group * SUM_PART : gate ? group * a.chunks_per_group : 0;
    const int count = PARTS ? min(SUM_PART, a.chunks - first) : gate ? a.chunks_per_group : a.chunks;
    float acc = 0.f;
    if (c < a.cols) {
      const float* p = (gate ? a.gate_partial : a.partial) + ((size_t)first * a.sums + s) * a.cols + c;
#pragma unroll 8
      for (int i = w; i < count; i += 16) acc += p[(size_t)i * a.sums * a.cols];
    }
    lds[w][lane] = acc;
    __syncthreads();
    if (w == 0 && c < a.cols) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) t += lds[i][lane];
      const size_t at = PARTS ? ((size_t)group * a.sums + s) * a.cols + c : (size_t)group * a.cols + c;
      if (!PARTS && a.out_bf16) reinterpret_cast<__bf16*>(out)[at] = (__bf16)t;
      else reinterpret_cast<float*>(out)[at] = t;
    }
    __syncthreads();                                                       // read before the next vector's sums overwrite them
  }
}
// parts that the chunks are added in before the last sum (0: one pass)
static long long sum_parts(long long chunks) { return chunks > 4 * SUM_PART ? (chunks + SUM_PART - 1) / SUM_PART : 0; }

static int norm_check(const pnResidualNorm* p) {
  PN_CHECK_ARG(p, "residual_norm: null pointer");
  PN_CHECK_ARG(p->dtype == PN_DTYPE_F32 || p->dtype == PN_DTYPE_BF16, "residual_norm: element type %d (fp32 or bf16)", p->dtype);
  PN_CHECK_ARG(p->param_dtype == PN_DTYPE_F32 || p->param_dtype == PN_DTYPE_BF16, "residual_norm: parameter type %d (fp32 or bf16)",
               p->param_dtype);
  PN_CHECK_ARG(p->dtype == PN_DTYPE_BF16 || p->param_dtype == PN_DTYPE_F32, "residual_norm: fp32 rows take fp32 parameters");
  PN_CHECK_ARG(p->cols >= 1 && p->cols <= PN_NORM_MAX_COLS, "residual_norm: %d columns (1..%d)", p->cols, PN_NORM_MAX_COLS);
  PN_CHECK_ARG(p->rows >= 0 && p->rows < (1ll << 40) / p->cols, "residual_norm: %lld rows", (long long)p->rows);
  PN_CHECK_ARG(p->post_kind >= PN_NORM_NONE && p->post_kind <= PN_NORM_RMS, "residual_norm: post norm %d (none, layer, rms)",
               p->post_kind);
  PN_CHECK_ARG(p->norm_kind >= PN_NORM_NONE && p->norm_kind <= PN_NORM_AFFINE, "residual_norm: norm %d", p->norm_kind);
  PN_CHECK_ARG(p->act == PN_ACT_NONE || p->act == PN_ACT_RELU, "residual_norm: activation %d (none or relu)", p->act);
  PN_CHECK_ARG(p->branch || (!p->gate && p->post_kind == PN_NORM_NONE && !p->threshold),
               "residual_norm: gate, post norm and dropout act on a branch");
  PN_CHECK_ARG(p->branch || p->norm_kind != PN_NORM_NONE, "residual_norm: neither a branch nor a norm");
  PN_CHECK_ARG(p->threshold <= 65536u && p->call < 65536u && (p->rng || !p->threshold), "residual_norm: dropout threshold %u, call %u",
               p->threshold, p->call);
  PN_CHECK_ARG(p->rows == 0 || (p->x && (p->rows == 1 || (p->ldx >= p->cols && (!p->branch || p->ldb >= p->cols)))),
               "residual_norm: x missing or a row stride below the row length");
  PN_CHECK_ARG(!p->gate || (p->rows_per_gate >= 1 && p->rows % p->rows_per_gate == 0),
               "residual_norm: %lld rows do not divide into gates of %lld rows", (long long)p->rows, (long long)p->rows_per_gate);
  PN_CHECK_ARG(!p->gate || p->rows_per_gate == 1 || p->rows / p->rows_per_gate <= 1 << 23, "residual_norm: more than 2^23 gates of several rows");
  return PN_OK;
}

static NormArgs norm_args(const pnResidualNorm* p) {
  NormArgs a = {};
  a.p = *p;
  a.keep_scale = !p->threshold ? 1.f : p->threshold < 65536u ? 65536.f / (65536.f - (float)p->threshold) : 0.f;
  if (!p->gate) a.p.rows_per_gate = p->rows > 0 ? p->rows : 1;
  return a;
}

// Waves of the forward pass: 32 a CU, which then go from row to row with the next row on its way.  Without post norm and dropout rows
// up to 4096 gain from four times as many (their own turnover overlaps better: 16499 x 2048 bf16 52 -> 47 us, 32768 x 4096 204 -> 199);
// wider ones and the others lose (4096 x 8192 with both: 68 -> 79 us).
static constexpr int FWD_WAVES = 8192, FWD_WAVES_PLAIN = 32768;

// Threads per row: the fewest that hold the row at eight elements each (K pieces of eight over 8192 columns, and in the backward
// pass with a branch over 4096), so that a narrow row does not idle a wave; over 1024 columns the workgroup is as large as its row,
// in whole waves (granule 64) or in a wave for each SIMD (256).  Where registers leave room for 8 or 16 waves a CU, odd numbers of
// them leave SIMDs idle: backward with a branch 16496 x 2104 bf16 184 us against 229, 8192 x 3000 104 against 153; forward with post
// norm or dropout over 2048 columns 59 against 70 (8192 x 3000), below it whole waves are as good or better (16496 x 1304: 51 against
// 56).  Without them whole waves win up to 2560 columns forward (16496 x 2104: 59 against 68; 4096 x 7000: 57 against 47) and at all
// widths backward.
#define NORM_BY_COLS(C, WIDE, GO)                                                \
  (C) <= 64 ? GO(8, 1, 256) : (C) <= 128 ? GO(16, 1, 256) : (C) <= 256 ? GO(32, 1, 256) : (C) <= 512 ? GO(64, 1, 256) \
  : (C) <= 1024 ? GO(128, 1, 256) : (C) <= 4096 ? GO(0, 1, 512) : (C) <= 8192 ? WIDE : GO(0, 2, 1024)
static int norm_threads(int C, int L, int K, int NT, int granule) {
  return L ? NT : ((C + 8 * K - 1) / (8 * K) + granule - 1) / granule * granule;
}
static int fwd_granule(int C, bool full) { return C <= (full ? 2048 : 2560) ? 64 : 256; }
static int bwd_granule(bool branch) { return branch ? 256 : 64; }

template <typename T, typename P, int L, int K, int NT> static int norm_fwd(const NormArgs& a, hipStream_t s) {
  const bool full = a.p.post_kind != PN_NORM_NONE || a.p.threshold;
  const int granule = fwd_granule(a.p.cols, full);
#define FWD(MODE, L_, K_, NT_)                                                                                                \
  do {                                                                                                                       \
    const int threads = norm_threads(a.p.cols, L_, K_, NT_, granule), slots = L_ ? NT_ / (L_ ? L_ : 1) : 1;                                \
    const long long need = (a.p.rows + slots - 1) / slots, most = (full || NT_ > 512 ? FWD_WAVES : FWD_WAVES_PLAIN) / (threads / 64);                            \
    const dim3 grid((unsigned)(need < most ? need : most)), wg(threads);                                                         \
    if (full) hipLaunchKernelGGL((residual_norm_fwd_kernel<T, P, L_, K_, NT_, MODE, true>), grid, wg, 0, s, a);              \
    else hipLaunchKernelGGL((residual_norm_fwd_kernel<T, P, L_, K_, NT_, MODE, false>), grid, wg, 0, s, a);                  \
  } while (0)
  if (a.p.cols == (L ? L : norm_threads(a.p.cols, L, K, NT, granule)) * K * 8) FWD(EXACT, L, K, NT);
  else if (a.p.cols >= 8) FWD(RAGGED, L, K, NT);
  else FWD(TINY, 8, 1, 256);
#undef FWD
  PN_CHECK_LAUNCH("residual_norm_fwd_kernel");
  return PN_OK;
}

template <typename T, typename P> static int norm_fwd_by_cols(const NormArgs& a, hipStream_t s) {
#define GO(L, K, NT) norm_fwd<T, P, L, K, NT>(a, s)
  return NORM_BY_COLS(a.p.cols, GO(0, 1, 1024), GO);
#undef GO
}

extern "C" int pn_residual_norm_forward(const pnResidualNorm* p, void* h, void* y, float* stats, void* stream) {
  const int rc = norm_check(p);
  if (rc != PN_OK) return rc;
  if (p->rows == 0) return PN_OK;
  PN_CHECK_ARG(((uintptr_t)stats & 15) == 0, "residual_norm: the statistics must be 16-byte aligned");
  PN_CHECK_ARG((h || !p->branch) && (y || p->norm_kind == PN_NORM_NONE), "residual_norm: output missing");
  NormArgs a = norm_args(p);
  a.h = h;
  a.y = p->norm_kind == PN_NORM_NONE ? nullptr : y;
  a.stats = stats;
  hipStream_t s = (hipStream_t)stream;
  // fp32 rows go with fp32 parameters, bf16 rows with either
  if (p->dtype == PN_DTYPE_F32) return norm_fwd_by_cols<float, float>(a, s);
  return p->param_dtype == PN_DTYPE_F32 ? norm_fwd_by_cols<__bf16, float>(a, s) : norm_fwd_by_cols<__bf16, __bf16>(a, s);
}

// Chunks of the backward pass: about BWD_WAVES waves in all (8 a CU: what the kernel with a branch keeps resident; a workgroup a CU at the least), whole passes
// over the row slots, none across two gates.  Half as many again leave a part-filled round: 8192 x 4096 bf16 with a branch 95 -> 118 us.
static constexpr int BWD_WAVES = 2048;
struct NormChunks { long long groups, group_rows; int per_group, rows, sums; };
static NormChunks norm_chunks(const pnResidualNorm* p, bool branch) {
  NormChunks c;
  c.groups = p->gate && p->rows_per_gate > 1 ? p->rows / p->rows_per_gate : 1;
  if (c.groups < 1) c.groups = 1;
  c.group_rows = c.groups > 1 ? p->rows_per_gate : p->rows;
#define SLOTS_OF(L, K, NT) (L ? NT / (L ? L : 1) : 1)
#define WAVES_OF(L, K, NT) (norm_threads(p->cols, L, K, NT, bwd_granule(branch)) / 64)
  const int slots = NORM_BY_COLS(p->cols, 1, SLOTS_OF), waves = NORM_BY_COLS(p->cols, (branch ? WAVES_OF(0, 2, 512) : WAVES_OF(0, 1, 1024)), WAVES_OF);
#undef SLOTS_OF
#undef WAVES_OF
  const long long passes = (c.group_rows + slots - 1) / slots;
  const int wgs = waves > 8 ? 256 : BWD_WAVES / waves;
  long long want = (wgs + c.groups - 1) / c.groups;
  if (want > passes) want = passes;
  if (want < 1) want = 1;
  const long long per = (passes + want - 1) / want;
  c.rows = (int)(per * slots);
  c.per_group = (int)((passes + per - 1) / per);
  c.sums = branch ? NSUM_ALL : NSUM_NORM;
  return c;
}
static bool norm_reads_branch(const pnResidualNorm* p) { return p->branch && (p->gate || p->post_kind != PN_NORM_NONE || p->threshold); }

extern "C" size_t pn_residual_norm_workspace_bytes(const pnResidualNorm* p) {
  if (norm_check(p) != PN_OK) return 0;
  const NormChunks c = norm_chunks(p, norm_reads_branch(p));
  const long long chunks = c.groups * c.per_group;
  return (size_t)(chunks + sum_parts(chunks)) * c.sums * p->cols * sizeof(float);
}

template <typename T, typename P, int L, int K, int NT, int MODE, bool BRANCH> static int norm_bwd(const NormArgs& a, unsigned grid, hipStream_t s) {
  const int threads = norm_threads(a.p.cols, L, K, NT, bwd_granule(BRANCH));
  PN_CHECK_ARG((unsigned long long)grid * threads < 1ull << 32, "residual_norm: %u chunks of %d threads are more than one launch takes", grid, threads);
  size_t lds = 0;
  if (bwd_parks(L, K, NT, BRANCH)) {
    lds = (size_t)4 * K * 8 * sizeof(P) * threads;
    static thread_local int raised_on = -1;                // the device that this thread allowed more than 64 KB on last
    int d = 0;
    PN_CHECK_HIP(hipGetDevice(&d));
    if (d != raised_on) {
      PN_CHECK_HIP(hipFuncSetAttribute((const void*)residual_norm_bwd_kernel<T, P, L, K, NT, MODE, BRANCH>,
                                       hipFuncAttributeMaxDynamicSharedMemorySize, 4 * K * 8 * (int)sizeof(P) * NT));
      raised_on = d;
    }
  }
  hipLaunchKernelGGL((residual_norm_bwd_kernel<T, P, L, K, NT, MODE, BRANCH>), dim3(grid), dim3(threads), lds, s, a);
  PN_CHECK_LAUNCH("residual_norm_bwd_kernel");
  return PN_OK;
}
template <typename T, typename P, int L, int K, int NT, bool BRANCH> static int norm_bwd_by_mode(const NormArgs& a, unsigned grid, hipStream_t s) {
  if (a.p.cols == (L ? L : norm_threads(a.p.cols, L, K, NT, bwd_granule(BRANCH))) * K * 8) return norm_bwd<T, P, L, K, NT, EXACT, BRANCH>(a, grid, s);
  return a.p.cols >= 8 ? norm_bwd<T, P, L, K, NT, RAGGED, BRANCH>(a, grid, s) : norm_bwd<T, P, 8, 1, 256, TINY, BRANCH>(a, grid, s);
}
template <typename T, typename P, bool BRANCH> static int norm_bwd_by_cols(const NormArgs& a, unsigned grid, hipStream_t s) {
#define GO(L, K, NT) norm_bwd_by_mode<T, P, L, K, NT, BRANCH>(a, grid, s)
  return NORM_BY_COLS(a.p.cols, GO(0, (BRANCH ? 2 : 1), (BRANCH ? 512 : 1024)), GO);
#undef GO
}
template <typename T, typename P> static int norm_bwd_by_branch(const NormArgs& a, bool branch, unsigned grid, hipStream_t s) {
  return branch ? norm_bwd_by_cols<T, P, true>(a, grid, s) : norm_bwd_by_cols<T, P, false>(a, grid, s);
}

extern "C" int pn_residual_norm_backward(const pnResidualNorm* p, const void* h, const float* stats, const void* gh,
                                         const void* gy, void* dx, void* dbranch, void* dweight, void* dbias,
                                         void* dpost_weight, void* dpost_bias, void* dgate, void* ws, size_t ws_bytes,
                                         void* stream) {
  const int rc = norm_check(p);
  if (rc != PN_OK) return rc;
  const bool branch = norm_reads_branch(p);
  PN_CHECK_ARG(gh || gy, "residual_norm: no gradient given");
  PN_CHECK_ARG(!gy || p->norm_kind != PN_NORM_NONE, "residual_norm: gradient of an output that there is not");
  PN_CHECK_ARG(p->rows == 0 || !gy || h || !p->branch, "residual_norm: the stored rows are needed");
  PN_CHECK_ARG(p->rows == 0 || stats || (p->norm_kind != PN_NORM_LAYER && p->norm_kind != PN_NORM_RMS && p->post_kind == PN_NORM_NONE),
               "residual_norm: the stored statistics are needed");
  PN_CHECK_ARG(((uintptr_t)stats & 15) == 0, "residual_norm: the statistics must be 16-byte aligned");
  PN_CHECK_ARG(!dbranch || (p->branch && (branch || p->scale != 1.f)), "residual_norm: the branch's gradient is dx itself");
  PN_CHECK_ARG(!dgate || p->gate, "residual_norm: gradient of a gate that there is not");
  const NormChunks c = norm_chunks(p, branch);
  hipStream_t s = (hipStream_t)stream;
  const long long chunks = p->rows ? c.groups * c.per_group : 0;
  if (chunks) {
    if (ws_bytes < (size_t)(chunks + sum_parts(chunks)) * c.sums * p->cols * sizeof(float) || !ws) {
      pn_set_error("residual_norm: workspace of %zu bytes is too small", ws_bytes);
      return PN_ENOSPC;
    }
    NormArgs a = norm_args(p);
    a.h = const_cast<void*>(h);
    a.stats = const_cast<float*>(stats);
    a.gh = gh;
    a.gy = gy;
    a.dx = dx;
    a.df = dbranch;
    if (p->gate && p->rows_per_gate == 1 && p->rows > 1) {
      a.dgate_rows = dgate;
      dgate = nullptr;
    }
    a.partial = (float*)ws;
    a.chunk_rows = c.rows;
    a.chunks_per_group = c.per_group;
    a.group_rows = c.group_rows;
    const unsigned grid = (unsigned)chunks;
    const int r = p->dtype == PN_DTYPE_F32 ? norm_bwd_by_branch<float, float>(a, branch, grid, s)
                  : p->param_dtype == PN_DTYPE_F32 ? norm_bwd_by_branch<__bf16, float>(a, branch, grid, s)
                                                   : norm_bwd_by_branch<__bf16, __bf16>(a, branch, grid, s);
    if (r != PN_OK) return r;
  }
  if (dweight || dbias || dpost_weight || dpost_bias || dgate) {
    const long long vecs = dgate ? NSUM_ALL - 1 + c.groups : (dpost_weight || dpost_bias) ? NSUM_ALL - 1 : NSUM_NORM;
    if (!p->rows) dgate = nullptr;                 // no rows, no gates
    SumArgs q = {(const float*)ws, (const float*)ws, {dweight, dbias, dpost_weight, dpost_bias, dgate}, p->cols, c.sums, (int)chunks,
                 chunks ? c.per_group : 0, p->param_dtype == PN_DTYPE_BF16, (int)vecs};
    const unsigned col_groups = (p->cols + 63) / 64;
    if (const long long parts = sum_parts(chunks)) {
      SumArgs in_parts = q;
      float* sums = (float*)ws + (size_t)chunks * c.sums * p->cols;
      in_parts.out[0] = sums;
      in_parts.vecs = c.sums < NSUM_ALL ? c.sums : NSUM_ALL - 1;
      hipLaunchKernelGGL(residual_norm_sum_kernel<true>, dim3(in_parts.vecs, col_groups, (unsigned)parts), dim3(1024), 0, s, in_parts);
      PN_CHECK_LAUNCH("residual_norm_sum_kernel");
      q.partial = sums;
      q.chunks = (int)parts;
    }
    hipLaunchKernelGGL(residual_norm_sum_kernel<false>, dim3((unsigned)(vecs < SUM_GRID ? vecs : SUM_GRID), col_groups), dim3(1024), 0, s, q);
    PN_CHECK_LAUNCH("residual_norm_sum_kernel");
  }
  return PN_OK;
}
