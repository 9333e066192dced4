// Activation + dropout, forward and backward:  y = keep ? act(x) / (1 - p) : 0.
//
// The mask is never stored: both passes draw it again from (seed, offset, call, element index), so the only traffic is
// the tensors themselves.  A dropped element is SELECTED to zero, not multiplied, so an infinity or NaN behind the mask
// does not reach the output or the gradient.  p is the 16-bit threshold's: T / 65536, and the scale uses that T.
// Backward of ReLU + dropout reads y instead of x: y > 0 exactly where the element was kept and positive (scaling up never
// underflows), which frees x and needs no generator.
//
// Bound by memory.  A thread takes eight elements, what one run of the generator decides and 16 bytes of bf16: 65536 x 2048 bf16
// with ReLU, p = 0.1: forward 85 us (6.3 TB/s), backward 142 us (5.7 TB/s).  In fp32 with GELU (6271 x 1023: 13 and 17 us, 4 and
// 4.5 TB/s) the generator's 40 integer multiplies and the fitted tail are about half the cycles.  Strided rows take a 64-bit division a
// piece, and in fp32 16 - 24 bytes of scratch a lane (load8_view's elements).
#include "ffn_common.h"

struct DropArgs {
  const void* x;                     // forward: x; backward: what the derivative needs (gelu: x, relu: y, none: NULL)
  const void* g;                     // backward only
  void* out;
  const unsigned long long* rng;     // {seed, offset} in device memory
  long long rows, cols, ldx, ldg;
  unsigned threshold, call;
  float scale;
};

// element pieces of a [rows, cols] view with row stride ld, by linear index
template <typename T>
__device__ __forceinline__ void load8_view(const T* p, long long ld, long long cols, unsigned long long e, int n, float (&o)[8]) {
  if (ld == cols) {
    load8(p + e, n, o);
    return;
  }
  unsigned long long row = e / (unsigned long long)cols;
  long long col = (long long)(e - row * cols);
  if (col + 8 <= cols) {
    load8(p + row * ld + col, n, o);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    o[i] = i < n ? (float)p[row * ld + col] : 0.f;
    if (++col == cols) { col = 0; ++row; }
  }
}

template <typename T, int ACT, bool BWD>
__device__ __forceinline__ void act_dropout_piece(const DropArgs& a, const PhiloxKey& key, unsigned long long e, int n, const float (&x)[8],
                                                  const float (&g)[8]) {
  Keep8 keep = keep_all();
  if (a.threshold && !(BWD && ACT == PN_ACT_RELU)) keep = keep8_group(key, e >> 3, a.threshold);
  float o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!BWD) {
      o[i] = keep(i) ? act_f(x[i], ACT) * a.scale : 0.f;
    } else if (ACT == PN_ACT_RELU) {
      o[i] = x[i] <= 0.f ? 0.f : g[i] * a.scale;
    } else {
      const float d = ACT == PN_ACT_GELU ? gelu_grad_f(x[i]) : 1.f;
      o[i] = keep(i) ? g[i] * a.scale * d : 0.f;
    }
  }
  store8(reinterpret_cast<T*>(a.out) + e, n, o);
}

// Where a workgroup's pieces are all whole and the rows lie one behind the other, no load stands behind a branch of its own.
template <typename T, int ACT, bool BWD>
__global__ __launch_bounds__(256) void act_dropout_kernel(DropArgs a) {
  const unsigned long long total = (unsigned long long)a.rows * a.cols, block = (unsigned long long)blockIdx.x * 2048, e = block + threadIdx.x * 8;
  const T *xp = reinterpret_cast<const T*>(a.x), *gp = reinterpret_cast<const T*>(a.g);
  constexpr bool X = !BWD || ACT != PN_ACT_NONE;
  PhiloxKey key{};
  if (a.threshold && !(BWD && ACT == PN_ACT_RELU)) key = philox_key(a.rng, a.call);
  float x[8], g[8];
  if (block + 2048 <= total && (!X || a.ldx == a.cols) && (!BWD || a.ldg == a.cols)) {
    Raw8<T> rx, rg;
    if (X) rx.load(xp + e);
    if (BWD) rg.load(gp + e);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = X ? rx.get(i) : 0.f;
      g[i] = BWD ? rg.get(i) : 0.f;
    }
    act_dropout_piece<T, ACT, BWD>(a, key, e, 8, x, g);
    return;
  }
  if (e >= total) return;
  const int n = total - e < 8 ? (int)(total - e) : 8;
  if (X) load8_view(xp, a.ldx, a.cols, e, n, x);
  if (BWD) load8_view(gp, a.ldg, a.cols, e, n, g);
  act_dropout_piece<T, ACT, BWD>(a, key, e, n, x, g);
}

template <typename T, bool BWD>
static int launch_act_dropout(const DropArgs& a, int act, hipStream_t s) {
  const dim3 grid((unsigned)((a.rows * a.cols + 2047) / 2048)), wg(256);
  switch (act) {
    case PN_ACT_NONE: hipLaunchKernelGGL((act_dropout_kernel<T, PN_ACT_NONE, BWD>), grid, wg, 0, s, a); break;
    case PN_ACT_RELU: hipLaunchKernelGGL((act_dropout_kernel<T, PN_ACT_RELU, BWD>), grid, wg, 0, s, a); break;
    default: hipLaunchKernelGGL((act_dropout_kernel<T, PN_ACT_GELU, BWD>), grid, wg, 0, s, a); break;
  }
  PN_CHECK_LAUNCH("act_dropout_kernel");
  return PN_OK;
}

static int act_dropout(bool bwd, int dtype, DropArgs a, int act, void* stream) {
  PN_CHECK_ARG(dtype == PN_DTYPE_F32 || dtype == PN_DTYPE_BF16, "act_dropout: element type %d (fp32 or bf16)", dtype);
  PN_CHECK_ARG(act >= PN_ACT_NONE && act <= PN_ACT_GELU, "act_dropout: activation %d", act);
  PN_CHECK_ARG(a.threshold <= 65536u && a.call < 65536u, "act_dropout: threshold %u (0..65536), call %u (0..65535)", a.threshold, a.call);
  PN_CHECK_ARG(a.rows >= 0 && a.cols >= 0, "act_dropout: negative size");
  if (a.rows == 0 || a.cols == 0) return PN_OK;
  // (workgroups of 256 threads and 2048 elements; a launch holds less than 2^32 threads)
  PN_CHECK_ARG(a.rows <= ((1ll << 35) - 2048) / a.cols, "act_dropout: %lld x %lld elements are more than one launch takes", a.rows, a.cols);
  PN_CHECK_ARG(a.out && (a.x || (bwd && act == PN_ACT_NONE)) && (a.g || !bwd), "act_dropout: null pointer");
  PN_CHECK_ARG(a.rng || !a.threshold, "act_dropout: dropping needs the generator's state");
  PN_CHECK_ARG((!a.x || a.ldx >= a.cols || a.rows == 1) && (!a.g || a.ldg >= a.cols || a.rows == 1), "act_dropout: row stride below the row length");
  if (a.rows == 1) a.ldx = a.ldg = a.cols;
  a.scale = a.threshold < 65536u ? 65536.f / (65536.f - (float)a.threshold) : 0.f;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PN_DTYPE_F32) return bwd ? launch_act_dropout<float, true>(a, act, s) : launch_act_dropout<float, false>(a, act, s);
  return bwd ? launch_act_dropout<__bf16, true>(a, act, s) : launch_act_dropout<__bf16, false>(a, act, s);
}

extern "C" int pn_act_dropout_forward(int dtype, const void* x, long long rows, long long cols, long long ldx, int act,
                                      unsigned threshold, const void* rng, unsigned call, void* y, void* stream) {
  DropArgs a = {x, nullptr, y, (const unsigned long long*)rng, rows, cols, ldx, 0, threshold, call, 1.f};
  return act_dropout(false, dtype, a, act, stream);
}

extern "C" int pn_act_dropout_backward(int dtype, const void* g, const void* saved, long long rows, long long cols,
                                       long long ldg, long long lds, int act, unsigned threshold, const void* rng,
                                       unsigned call, void* dx, void* stream) {
  DropArgs a = {saved, g, dx, (const unsigned long long*)rng, rows, cols, lds, ldg, threshold, call, 1.f};
  return act_dropout(true, dtype, a, act, stream);
}

// One thread: hand out the state a pass uses and move the stored one on, so that a replayed graph draws anew.
__global__ void dropout_draw_kernel(unsigned long long* state, unsigned long long* used) {
  used[0] = state[0];
  used[1] = state[1];
  state[1] += 1;
}
extern "C" int pn_dropout_draw(void* state, void* used, void* stream) {
  PN_CHECK_ARG(state && used, "pn_dropout_draw: null pointer");
  hipLaunchKernelGGL(dropout_draw_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, (unsigned long long*)state,
                     (unsigned long long*)used);
  PN_CHECK_LAUNCH("dropout_draw_kernel");
  return PN_OK;
}
