"""Feed-forward operators on the GPU against oracle/ffn_oracle.py (64 bits).

Tolerances are counted in half steps of the types, u = eps / 2 relative to the value a rounding acts on:
  dropout      two fp32 roundings (scale, product) and the output's; GELU adds an absolute error of |x| * 4u (its tail q <= 1/2
               from the fitted t P(t) e^(-z^2): t is within 3u, which the product's sensitivity of at most 2.26 to it takes to
               6.8u of q, 3.4u |x|, and the last product's rounding).
  norms        a sum over a row takes at most 8 K serial, 6 additions across lanes and 4 across waves (K <= 2): 26 roundings, and
               as many for the second statistic, so every normalised value is within 96u of r * (|t| + mean |t|) + |n|; the
               gradients add two more such sums.
  column sums  R rows (and chunks) are added in fp32: (R + 64)u of the sum of magnitudes, plus what the summands are off.
  fp8          bytes and scales are exact.  Products: whole numbers below 2^24 are exact; an fp32 result may be off by one step
               for each of K additions, 2K u of the sum of magnitudes.  A bf16 result comes from the fp8 matrix instruction, which
               drops from each product what lies 2^-16 below the largest of its eight (measured with single pairs of products):
               up to 7 * 2^-16 of that largest product more, so 7 * 2^-16 of the sum of magnitudes."""
import math

import numpy as np
import pytest
import torch

import fp8_product_cases as pc
from oracle import ffn_oracle as fo
from pillarnet_lts_amd import _lib, ffn_ops
from pillarnet_lts_amd._lib import PillarnetHipError

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
BOTH = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])


def d(t):
    return t.detach().double().cpu().numpy()


def within(got, want, tol, what=""):
    got = d(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300)):.3g} x tolerance"


def rng_of(seed, offset, cuda):
    return torch.tensor([seed, offset], dtype=torch.int64, device=cuda)


@pytest.fixture
def large(cuda):
    """cuda, for tests whose tensors should not count in the peaks that later tests look at."""
    yield cuda
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()


# ---- activation + dropout ----------------------------------------------------------------------------------------------
@BOTH
@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
@pytest.mark.parametrize("shape", [(1,), (1, 1), (3, 7), (5, 8), (2, 3, 64), (129, 257), (1000, 33)])
@pytest.mark.parametrize("p", [0.0, 0.3, 1.0])
def test_act_dropout(cuda, dtype, act, shape, p):
    rs = np.random.RandomState(len(shape) * 7 + shape[0])
    seed, off, call = 0x1234567890ABCDEF, (5 << 32) + 77, 11
    x = torch.from_numpy(rs.randn(*shape).astype(np.float32) * 2).to(dtype).to(cuda).requires_grad_()
    g = torch.from_numpy(rs.randn(*shape).astype(np.float32)).to(dtype).to(cuda)
    y = ffn_ops.act_dropout(x, p, rng_of(seed, off, cuda) if p else None, call, act)
    xd, gd = d(x), d(g)
    k = fo.drop_scale(p, seed, off, call, shape)
    want = fo.act(xd, act) * k
    extra = 4 * U32 * np.abs(xd) * k if act == "gelu" else 0.0
    within(y, want, (U[dtype] + 3 * U32) * np.abs(want) + extra, "y")
    if y is x:
        assert act == "none" and p == 0
        return
    dx, = torch.autograd.grad(y, x, g)
    want = gd * k * fo.act_grad(xd, act)
    # gelu': Phi within 4u, x phi(x) <= 0.25 within 8u (exp 2 ulp = 4u, its argument's rounding times |x^2 / 2| phi: 1u, products)
    extra = 8 * U32 * np.abs(gd) * k * (1 + np.abs(xd)) if act == "gelu" else 0.0
    within(dx, want, (U[dtype] + 4 * U32) * np.abs(want) + extra, "dx")
    assert (d(dx)[k == 0] == 0).all() and (d(y)[k == 0] == 0).all()


@BOTH
def test_act_dropout_strides_and_masked_places(cuda, dtype):
    """the mask goes by the element's index, whatever the strides; nothing behind a dropped element gets out."""
    rs = np.random.RandomState(3)
    wide = torch.from_numpy(rs.randn(37, 90).astype(np.float32)).to(dtype).to(cuda)
    rng = rng_of(99, 1, cuda)
    base = ffn_ops.act_dropout(wide[:, 3:72].contiguous(), 0.4, rng)
    assert torch.equal(ffn_ops.act_dropout(wide[:, 3:72], 0.4, rng), base)                       # odd offset, odd stride
    assert torch.equal(ffn_ops.act_dropout(wide[:, 3:72].t().contiguous().t(), 0.4, rng), base)  # column-major
    even = wide[:, 8:72]
    assert torch.equal(ffn_ops.act_dropout(even, 0.4, rng), ffn_ops.act_dropout(even.contiguous(), 0.4, rng))
    x = wide[:, 3:72].clone()
    kept = torch.from_numpy(fo.drop_scale(0.4, 99, 1, 0, (37, 69)) > 0).to(cuda)
    x[~kept] = torch.tensor([math.nan, math.inf, -math.inf], device=cuda, dtype=dtype).repeat((~kept).sum() // 3 + 1)[: (~kept).sum()]
    for act in ("none", "relu", "gelu"):
        xl = x.clone().requires_grad_()
        y = ffn_ops.act_dropout(xl, 0.4, rng, 0, act)
        assert torch.isfinite(y).all() and (y[~kept] == 0).all()
        gr = torch.where(kept, 1.0, math.nan).to(dtype)
        dx, = torch.autograd.grad(y, xl, gr)
        assert (dx[~kept] == 0).all() if act != "relu" else not torch.isnan(dx[~kept]).any()
        assert torch.isfinite(dx).all()
        e, = torch.autograd.grad(ffn_ops.act_dropout(xl, 0.4, rng, 0, act).sum(), xl)            # expanded gradient
        f, = torch.autograd.grad(ffn_ops.act_dropout(xl, 0.4, rng, 0, act), xl, torch.ones_like(xl))
        assert torch.equal(e, f)


def test_act_dropout_gradient_against_differences(cuda):
    x = torch.randn(64, 40, generator=torch.Generator().manual_seed(0)).to(cuda)
    rng, g = rng_of(5, 6, cuda), torch.randn(64, 40, generator=torch.Generator().manual_seed(1)).to(cuda)
    for act in ("none", "relu", "gelu"):
        xl = x.clone().requires_grad_()
        dx, = torch.autograd.grad(ffn_ops.act_dropout(xl, 0.25, rng, 2, act), xl, g)
        h = 2.0 ** -7                  # truncation h^2/6 max |gelu'''| (< 1.3) * scale 4/3 * |g|; rounding u |y| / h; a ReLU's kink within h
        step = (ffn_ops.act_dropout(x + h, 0.25, rng, 2, act) - ffn_ops.act_dropout(x - h, 0.25, rng, 2, act)) / (2 * h) * g
        ok = x.abs() > 2 * h if act == "relu" else torch.ones_like(x, dtype=torch.bool)
        tol = g.abs() * (h * h / 6 * 1.3 * 4 / 3 + 16 * U32 * (x.abs() + 1) * 4 / 3 / h) + 1e-7
        assert ((step - dx).abs() <= tol)[ok].all(), act


def test_dropout_state_moves_on_and_replays(cuda):
    st = ffn_ops.DropoutState((1 << 64) - 3, cuda)
    a, b = st.draw(), st.draw()
    assert a.tolist() == [-3, 0] and b.tolist() == [-3, 1] and st.state.tolist() == [-3, 2]
    x = torch.randn(70, 130, device=cuda, dtype=torch.bfloat16)
    k = fo.drop_scale(0.5, (1 << 64) - 3, 1, 0, (70, 130)) > 0
    assert np.array_equal(d(ffn_ops.act_dropout(x, 0.5, b)) != 0, k & (d(x) != 0))
    out = torch.empty_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ffn_ops.act_dropout(x, 0.5, st.draw())
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out.copy_(ffn_ops.act_dropout(x, 0.5, st.draw()))
    for i in range(3, 6):
        graph.replay()
        want = ffn_ops.act_dropout(x, 0.5, rng_of(-3, i, cuda))
        assert torch.equal(out, want), i


def test_act_dropout_beyond_32_bit_offsets(large, cuda):
    """4.3e9 elements: the last groups have element indices past 2^32."""
    cols, rows = 1 << 20, 4099
    x = torch.ones((rows, cols), dtype=torch.bfloat16, device=cuda)
    y = ffn_ops.act_dropout(x, 0.5, rng_of(7, 8, cuda), 3)
    for row in (0, 4095, 4096, 4098):
        k = fo.drop_scale(0.5, 7, 8, 3, (64,), start=row * cols + cols - 64)
        assert np.array_equal(d(y[row, -64:]), k)


def test_act_dropout_refusals(cuda):
    x, rng = torch.zeros(4, 8, device=cuda), rng_of(1, 2, cuda)
    for call in (lambda: ffn_ops.act_dropout(x.half(), 0.5, rng), lambda: ffn_ops.act_dropout(x, 0.5), lambda: ffn_ops.act_dropout(x, 1.5, rng),
                 lambda: ffn_ops.act_dropout(x, 0.5, rng.int()), lambda: ffn_ops.act_dropout(x, 0.5, rng.cpu()),
                 lambda: ffn_ops.act_dropout(x, 0.5, rng, 65536), lambda: ffn_ops.act_dropout(x, 0.5, rng, act="silu"),
                 lambda: ffn_ops.act_dropout(torch.zeros((), device=cuda), 0.5, rng)):
        with pytest.raises(PillarnetHipError):
            call()
    for shape in ((0, 8), (4, 0), (0,)):
        e = torch.zeros(shape, device=cuda, requires_grad=True)
        y = ffn_ops.act_dropout(e, 0.5, rng, act="gelu")
        assert y.shape == shape and torch.autograd.grad(y.sum(), e)[0].shape == shape


# ---- residual join and norms -------------------------------------------------------------------------------------------
def _join_case(cuda, dtype, pdtype, B, T, C, post, norm, gate, p, branch, act, scale, seed=0, strided=False):
    rs = np.random.RandomState(seed + B * 31 + T * 7 + C)
    n = lambda *s, m=0.0, sd=1.0: torch.from_numpy((rs.randn(*s) * sd + m).astype(np.float32))

    def data(*s, **kw):
        t = n(*s, **kw).to(dtype).to(cuda)
        if strided:                             # the same values at an odd offset inside wider rows
            w = torch.zeros(*s[:-1], s[-1] + 5, dtype=dtype, device=cuda)
            w[..., 3:3 + s[-1]] = t
            t = w[..., 3:3 + s[-1]]
        return t

    par = lambda *s, **kw: n(*s, **kw).to(pdtype).to(cuda).requires_grad_()
    t = dict(x=data(B, T, C, sd=2.0, m=0.3).requires_grad_())
    if branch:
        t["f"] = data(B, T, C, m=0.2).requires_grad_()
        if gate:
            t["gate"] = par(*{"channel": (C,), "sample": (B, C), "row": (B, T, C)}[gate], m=0.5)
        if post:
            t["pw"], t["pb"] = par(C, m=1.0, sd=0.2), par(C, sd=0.2)
    if norm:
        t["w"], t["b"] = par(C, m=1.0, sd=0.2), par(C, sd=0.2)
    args = dict(scale=scale if branch else 1.0, gate=t.get("gate"), act=act,
                post_norm=ffn_ops.Norm(post, t["pw"], t["pb"], 1e-5) if post and branch else None,
                norm=ffn_ops.Norm(norm, t["w"], t["b"], 1e-3) if norm else None,
                dropout=(p, rng_of(21, 4, cuda), 9) if branch and p else None)
    return t, args, (lambda: ffn_ops.residual_norm(t["x"], t.get("f"), **args))


def _join_check(t, args, out, grads, gh, gy, dtype, pdtype, p, post, norm, gate, act):
    """h, y and every gradient against the formulas, each from the values the kernels stored."""
    v = {k: d(q) for k, q in t.items()}
    shape = v["x"].shape
    R = shape[0] * shape[1]
    u = U[dtype]
    branch = "f" in t
    y = h = None
    if branch and norm:
        h, y = out
    elif branch:
        h = out
    else:
        y = out
    s = args["scale"]
    k = fo.drop_scale(p if branch else 0, 21, 4, 9, shape)
    if branch:
        fn, fm, fr = fo.normalise(v["f"], post, 1e-5)
        fu = fn * v["pw"] + v["pb"] if post else fn
        ga = v["gate"] if gate else np.ones(1)
        ga = ga[:, None, :] if gate == "sample" else ga
        fe = 96 * U32 * (fr * (np.abs(v["f"]) + np.abs(v["f"]).mean(-1, keepdims=True)) + np.abs(fn)) if post else 0 * fn   # of fn
        ue = fe * np.abs(v.get("pw", 1.0)) + 2 * U32 * np.abs(fu)
        want = v["x"] + s * ga * fu * k
        within(h, want, u * np.abs(want) + 4 * U32 * (np.abs(v["x"]) + np.abs(s * ga * fu * k)) + np.abs(s * ga * k) * ue, "h")
        hv = d(h)
    else:
        hv = v["x"]
    if norm:
        hn, hm, hr = fo.normalise(hv, norm, 1e-3)
        stat = norm != "affine"
        he = 96 * U32 * (hr * (np.abs(hv) + np.abs(hv).mean(-1, keepdims=True)) + np.abs(hn)) if stat else 0 * hn
        pre = hn * v["w"] + v["b"]
        want = fo.act(pre, act)
        pe = he * np.abs(v["w"]) + 3 * U32 * (np.abs(hn * v["w"]) + np.abs(v["b"]))
        within(y, want, u * np.abs(want) + pe, "y")
    if grads is None:
        return
    zero = np.zeros(shape)
    dh, de = (d(gh).copy() if gh is not None else zero.copy()), zero.copy()
    if norm and gy is not None:
        live = (pre > 0) if act == "relu" else np.ones(shape, bool)
        sure = (np.abs(pre) > pe) if act == "relu" else np.ones(shape, bool)
        assert sure.mean() > 0.99
        live = np.where(sure, live, d(y) > 0)        # within rounding of the kink either side is right: take the kernel's
        gp = d(gy) * live
        tw = gp * v["w"]
        n_ = fo.normalise_grad(tw, hn, hr, norm)
        A = np.abs(tw) + np.abs(tw).mean(-1, keepdims=True) + np.abs(hn) * np.abs(tw * hn).mean(-1, keepdims=True)
        if stat:
            de += hr * (160 * U32 * A + np.abs(tw * he).mean(-1, keepdims=True) * np.abs(hn) + he * np.abs((tw * hn).mean(-1, keepdims=True)))
        else:
            de += 3 * U32 * np.abs(tw)
        dh = dh + n_
        de += 2 * U32 * (np.abs(dh) + np.abs(n_))
        for name, q, qe in (("w", gp * hn, np.abs(gp) * he), ("b", gp, zero)):
            want = q.sum((0, 1))
            within(grads[name], want, U[pdtype] * np.abs(want) + (R + 64) * U32 * np.abs(q).sum((0, 1)) + qe.sum((0, 1)), "d" + name)
    within(grads["x"], dh, u * np.abs(dh) + de, "dx")
    if not branch:
        return
    du = s * ga * dh * k
    due = np.abs(s * ga * k) * (de + 4 * U32 * np.abs(dh))
    if gate:
        q, qe = s * dh * fu * k, np.abs(s * k) * (de * np.abs(fu) + np.abs(dh) * ue) + 4 * U32 * np.abs(s * dh * fu * k)
        ax = {"channel": (0, 1), "sample": 1, "row": ()}[gate]
        want = q.sum(ax)
        within(grads["gate"], want, U[pdtype] * np.abs(want) + (R + 64) * U32 * np.abs(q).sum(ax) + qe.sum(ax), "dgate")
    if post:
        for name, q, qe in (("pw", du * fn, due * np.abs(fn) + np.abs(du) * fe), ("pb", du, due)):
            want = q.sum((0, 1))
            within(grads[name], want, U[pdtype] * np.abs(want) + (R + 64) * U32 * np.abs(q).sum((0, 1)) + qe.sum((0, 1)), "d" + name)
        tp = du * v["pw"]
        want = fo.normalise_grad(tp, fn, fr, post)
        tpe = due * np.abs(v["pw"])
        A = np.abs(tp) + np.abs(tp).mean(-1, keepdims=True) + np.abs(fn) * np.abs(tp * fn).mean(-1, keepdims=True)
        e = fr * (160 * U32 * A + tpe + tpe.mean(-1, keepdims=True) + np.abs(fn) * (tpe * np.abs(fn)).mean(-1, keepdims=True)
                  + np.abs(tp * fe).mean(-1, keepdims=True) * np.abs(fn) + fe * np.abs((tp * fn).mean(-1, keepdims=True)))
        within(grads["f"], want, u * np.abs(want) + e, "df")
    else:
        within(grads["f"], du, u * np.abs(du) + due, "df")


def _join_run(cuda, dtype, pdtype, B, T, C, post, norm, gate, p, branch, act="none", scale=0.5, use=("h", "y"), strided=False):
    t, args, call = _join_case(cuda, dtype, pdtype, B, T, C, post, norm, gate, p, branch, act, scale, strided=strided)
    out = call()
    outs = list(out) if isinstance(out, tuple) else [out]
    names = [n for n, on in (("h", branch), ("y", norm)) if on]
    gen = torch.Generator().manual_seed(1)
    g = {n: torch.randn(B, T, C, generator=gen).to(dtype).to(cuda) for n in names}
    used = [n for n in names if n in use]
    grads = torch.autograd.grad([o for o, n in zip(outs, names) if n in used], list(t.values()), [g[n] for n in used], allow_unused=True)
    grads = dict(zip(t, grads))
    _join_check(t, args, out, grads, g.get("h") if "h" in used else None, g.get("y") if "y" in used else None, dtype, pdtype, p, post,
                norm, gate, act)
    with torch.no_grad():
        again = call()
    for a, b in zip(outs, again if isinstance(again, tuple) else [again]):
        assert torch.equal(a, b)                 # serving gives the training pass's bits


@BOTH
@pytest.mark.parametrize("C", [1, 7, 8, 33, 64, 65, 128, 200, 256, 500, 512, 1000, 1024, 2048, 2050, 4096, 5001, 8192, 16384])
def test_residual_norm_widths(cuda, dtype, C):
    _join_run(cuda, dtype, dtype, 2, 37, C, "rms", "layer", "channel", 0.1, True)


@BOTH
@pytest.mark.parametrize("C", [7, 64, 120, 250, 512, 1001, 1024, 2048, 2104, 3000, 4096, 4200, 8192, 9000, 16384])
def test_residual_norm_widths_without_post_norm_and_dropout(cuda, dtype, C):
    """the kernels for a gate alone, and for no branch."""
    _join_run(cuda, dtype, dtype, 2, 23, C, None, "rms", "channel", 0.0, True)
    _join_run(cuda, dtype, dtype, 1, 29, C, None, "layer", None, 0.0, False, act="relu")


@pytest.mark.parametrize("C", [1031, 1536, 4100, 5001, 8192, 9000])
def test_residual_norm_wide_rows_with_wider_parameters(cuda, C):
    """bf16 rows, fp32 parameters, workgroups of the row's size: odd and whole widths on either side of their limits."""
    _join_run(cuda, torch.bfloat16, torch.float32, 2, 19, C, "layer", "rms", "sample", 0.2, True, act="relu")
    _join_run(cuda, torch.bfloat16, torch.float32, 1, 5, C, None, "layer", None, 0.0, False, act="relu")


def test_residual_norm_beyond_32_bit_offsets(large, cuda):
    """4.3e9 elements: the last rows are those of a call of their own (a mask by element index among them)."""
    C, R = 4104, 1047000
    assert R * C > 1 << 32
    x = torch.zeros((R, C), dtype=torch.bfloat16, device=cuda)
    tail = torch.randn(8, C, device=cuda).bfloat16()
    x[-8:] = tail
    w, rng = torch.randn(C, device=cuda).bfloat16(), rng_of(3, 4, cuda)
    h, y = ffn_ops.residual_norm(x, x, scale=0.5, norm=ffn_ops.Norm("layer", w), dropout=(0.25, rng, 2))
    keep = torch.from_numpy(fo.drop_scale(0.25, 3, 4, 2, (8, C), start=(R - 8) * C)).to(cuda).float() * 0.5
    hw, yw = ffn_ops.residual_norm(tail, tail, gate=keep.bfloat16(), norm=ffn_ops.Norm("layer", w))
    within(h[-8:], d(tail) * (1 + d(keep)), 1.01 * U[torch.bfloat16] * np.abs(d(tail)) * (1 + d(keep)), "h")
    # 0.5 / 0.75 rounded to bf16 as a gate, h rounded on either side, y rounded on either side: five half steps, one for the statistics
    assert (y[-8:].float() - yw.float()).norm() <= 6 * U[torch.bfloat16] * yw.float().norm()
    assert (h[: 8] == 0).all() and (y[: 8] == 0).all()


@BOTH
@pytest.mark.parametrize("post", [None, "layer", "rms"])
@pytest.mark.parametrize("norm", [None, "layer", "rms", "affine"])
@pytest.mark.parametrize("gate", [None, "channel", "sample", "row"])
def test_residual_norm_kinds(cuda, dtype, post, norm, gate):
    _join_run(cuda, dtype, torch.float32, 3, 41, 72, post, norm, gate, 0.3 if gate != "row" else 0.0, True,
              act="relu" if norm == "layer" else "none")


@BOTH
@pytest.mark.parametrize("norm", ["layer", "rms", "affine"])
@pytest.mark.parametrize("B,T", [(1, 1), (1, 2), (5, 1), (4, 700)])
def test_residual_norm_without_a_branch(cuda, dtype, norm, B, T):
    _join_run(cuda, dtype, dtype, B, T, 48, None, norm, None, 0.0, False, act="relu")


@BOTH
@pytest.mark.parametrize("use", [("h",), ("y",)])
def test_residual_norm_with_one_output_used(cuda, dtype, use):
    _join_run(cuda, dtype, dtype, 2, 19, 96, "rms", "layer", "sample", 0.2, True, use=use)
    _join_run(cuda, dtype, dtype, 2, 19, 96, None, "layer", None, 0.0, True, scale=1.0, use=use)     # the branch's gradient is dx
    _join_run(cuda, dtype, dtype, 2, 19, 100, None, "rms", None, 0.0, True, scale=0.3, use=use)      # ... or a multiple of it


@BOTH
@pytest.mark.parametrize("B,T,C", [(1, 1, 256), (300, 1, 64), (7, 1, 5001), (1, 5000, 40), (64, 3, 520), (1100, 2, 40)])
def test_residual_norm_row_counts(cuda, dtype, B, T, C):
    _join_run(cuda, dtype, dtype, B, T, C, "layer", "rms", "sample", 0.5, True)


@BOTH
def test_residual_norm_strided_rows(cuda, dtype):
    _join_run(cuda, dtype, dtype, 2, 21, 67, "rms", "layer", "channel", 0.2, True, strided=True)
    _join_run(cuda, dtype, dtype, 2, 21, 64, None, "layer", None, 0.0, False, strided=True)


def test_residual_norm_mixed_parameter_types_and_missing_weights(cuda):
    x, f = torch.randn(2, 30, 64, device=cuda).bfloat16(), torch.randn(2, 30, 64, device=cuda).bfloat16()
    w16, g32 = torch.randn(64, device=cuda).bfloat16().requires_grad_(), torch.randn(64, device=cuda, requires_grad=True)
    h, y = ffn_ops.residual_norm(x, f, gate=g32, norm=ffn_ops.Norm("rms", w16))
    h2, y2 = ffn_ops.residual_norm(x, f, gate=g32, norm=ffn_ops.Norm("rms", w16.detach().float(), torch.zeros(64, device=cuda)))
    assert torch.equal(h, h2) and torch.equal(y, y2)
    dw, dg = torch.autograd.grad(y.float().sum(), (w16, g32))
    assert dw.dtype == torch.bfloat16 and dg.dtype == torch.float32 and dw.abs().sum() > 0
    plain = ffn_ops.residual_norm(x, norm=ffn_ops.Norm("layer"))
    n = fo.normalise(d(x), "layer", 1e-5)[0]
    within(plain, n, U[torch.bfloat16] * np.abs(n) + 1e-5, "y")


def test_residual_norm_masked_branch_and_equal_rows(cuda):
    """infinities behind dropped elements do not reach h or the gradients; a constant row has variance zero."""
    x = torch.randn(8, 64, device=cuda, requires_grad=True)
    f = torch.randn(8, 64, device=cuda)
    kept = torch.from_numpy(fo.drop_scale(0.5, 21, 4, 9, (8, 64)) > 0).to(cuda)
    f = torch.where(kept, f, math.inf).requires_grad_()
    gate = torch.randn(64, device=cuda, requires_grad=True)
    h, y = ffn_ops.residual_norm(x, f, gate=gate, norm=ffn_ops.Norm("layer"), dropout=(0.5, rng_of(21, 4, cuda), 9))
    grads = torch.autograd.grad((h, y), (x, f, gate), (torch.randn_like(h), torch.randn_like(y)))
    assert all(torch.isfinite(q).all() for q in (h, y, *grads)) and (grads[1][~kept] == 0).all()
    c = torch.full((5, 100), 3.25, device=cuda)
    assert (ffn_ops.residual_norm(c, norm=ffn_ops.Norm("layer")) == 0).all()


def test_residual_norm_gradient_against_differences(cuda):
    t, args, call = _join_case(cuda, torch.float32, torch.float32, 2, 6, 24, "rms", "layer", "sample", 0.25, True, "none", 0.5)
    gen = torch.Generator().manual_seed(2)
    gh, gy = torch.randn(2, 6, 24, generator=gen).to(cuda), torch.randn(2, 6, 24, generator=gen).to(cuda)
    grads = dict(zip(t, torch.autograd.grad(call(), list(t.values()), (gh, gy))))
    loss = lambda: sum((o.double() * g.double()).sum().item() for o, g in zip(call(), (gh, gy)))
    gen = torch.Generator().manual_seed(3)
    for name, leaf in t.items():
        v = torch.randn(leaf.shape, generator=gen).to(cuda)
        slope = (grads[name].double() * v.double()).sum().item()
        keep, step = leaf.detach().clone(), 2.0 ** -7
        with torch.no_grad():
            leaf.copy_(keep + step * v); up = loss()
            leaf.copy_(keep - step * v); down = loss()
            leaf.copy_(keep)
        got = (up - down) / (2 * step)
        # rounding: 576 outputs of size <= 8 with gradients of size 1, each within 8u, added at random: 24 * 64 * u / step; truncation:
        # step^2 / 6 times a third derivative along v, which is below the slope's own scale times 100 for rows of 24
        scale_ = grads[name].double().norm().item() * v.double().norm().item()
        assert abs(got - slope) <= 24 * 64 * U32 / step + step * step / 6 * 100 * scale_, (name, got, slope)


def test_residual_norm_repeats_its_bits(cuda):
    t, args, call = _join_case(cuda, torch.bfloat16, torch.float32, 4, 900, 256, "rms", "layer", "sample", 0.1, True, "none", 0.5)
    g = [torch.randn(4, 900, 256, device=cuda).bfloat16() for _ in range(2)]
    first = torch.autograd.grad(call(), list(t.values()), g)
    for _ in range(3):
        for a, b in zip(first, torch.autograd.grad(call(), list(t.values()), g)):
            assert torch.equal(a, b)


def test_residual_norm_most_gates_of_several_rows(large, cuda):
    """2^23 gates of two rows: more vectors of column sums than one launch has workgroups of 1024 threads.  Whole numbers: exact."""
    B = 1 << 23
    gen = torch.Generator(device="cuda").manual_seed(6)
    whole = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=gen, device=cuda).float()
    x, f, gate, gh = whole(-3, 4, B, 2, 1), whole(-3, 4, B, 2, 1), whole(-2, 3, B, 1), whole(-3, 4, B, 2, 1)
    gy, w = torch.zeros(B, 2, 1, device=cuda), whole(2, 3, 1)
    gy[::1 << 10] = 1.0                                                # 2^14 rows of 2^24: their sum with |h| <= 9 stays below 2^24
    leaves = [t.requires_grad_() for t in (x, f, gate, w)]
    h, y = ffn_ops.residual_norm(x, f, gate=gate, norm=ffn_ops.Norm("affine", w))
    dx, df, dg, dw = torch.autograd.grad((h, y), leaves, (gh, gy))
    g = gate.detach()[:, None]
    want = x + g * f
    assert torch.equal(h, want) and torch.equal(y, 2 * want)
    dh = gh + 2 * gy
    assert torch.equal(dx, dh) and torch.equal(df, g * dh) and torch.equal(dg, (dh * f).sum(1))
    assert dw.item() == (gy * want).double().sum().item()


def test_residual_norm_refusals(cuda):
    x = torch.zeros(4, 6, 8, device=cuda)
    w, N = torch.zeros(8, device=cuda), ffn_ops.Norm
    for call in (lambda: ffn_ops.residual_norm(x), lambda: ffn_ops.residual_norm(x, x.bfloat16(), norm=N("layer")),
                 lambda: ffn_ops.residual_norm(x, x[:2]), lambda: ffn_ops.residual_norm(x, gate=w, norm=N("rms")),
                 lambda: ffn_ops.residual_norm(x, x, gate=torch.zeros(3, 8, device=cuda)), lambda: ffn_ops.residual_norm(x, x, act="relu"),
                 lambda: ffn_ops.residual_norm(x, x, gate=w[:7]), lambda: ffn_ops.residual_norm(x, x, post_norm=N("affine", w)),
                 lambda: ffn_ops.residual_norm(x, norm=N("layer", w[:4])), lambda: ffn_ops.residual_norm(x, norm=N("layer", w.double())),
                 lambda: ffn_ops.residual_norm(x, norm=N("layer", w.cpu())), lambda: ffn_ops.residual_norm(x, x, dropout=(0.5, None, 0)),
                 lambda: ffn_ops.residual_norm(x, x, norm=N("rms"), act="gelu"), lambda: ffn_ops.residual_norm(x.half(), norm=N("rms")),
                 lambda: ffn_ops.residual_norm(torch.zeros(2, 16385, device=cuda), norm=N("rms"))):
        with pytest.raises(PillarnetHipError):
            call()
    e, g = torch.zeros(0, 6, 8, device=cuda, requires_grad=True), torch.ones(8, device=cuda, requires_grad=True)
    h, y = ffn_ops.residual_norm(e, e * 2, gate=g, norm=N("layer", g))
    de, dg = torch.autograd.grad(y.sum() + h.sum(), (e, g))
    assert h.shape == y.shape == de.shape == (0, 6, 8) and (dg == 0).all()


# ---- fp8 ---------------------------------------------------------------------------------------------------------------
def _values(rs, R, C, dtype):
    x = rs.randn(R, C) * np.exp(rs.randn(R, 1) * 3) * np.exp(rs.randn(1, C))
    x[rs.rand(R, C) < 0.05] = 0
    return torch.from_numpy(x.astype(np.float32)).to(dtype)


@BOTH
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 128), (3, 129), (127, 64), (128, 128), (129, 300), (700, 515), (260, 1024)])
def test_fp8_quantize_is_exact(cuda, dtype, block_rows, R, C):
    x = _values(np.random.RandomState(R + C), R, C, dtype)
    q, qt = ffn_ops.fp8_quantize(x.to(cuda), block_rows, True, True)
    want = fo.quantise(d(x), block_rows)
    wt = fo.quantise(d(x).T, 1) if block_rows == 1 else want.T
    np.testing.assert_array_equal(d(q.values()), want)
    np.testing.assert_array_equal(d(qt.values()), wt)
    for o, exps in ((q, fo.block_exponents(d(x), block_rows)), (qt, fo.block_exponents(d(x).T, block_rows))):
        bytes_, e = o.bytes_and_exponents()
        assert (bytes_[:, o.cols:] == 0).all()                                 # padding that products run over
        np.testing.assert_array_equal(e.cpu().numpy(), exps.repeat(block_rows, 0)[: o.rows])
    same = lambda a, b: torch.equal(a.values(), b.values())
    assert same(ffn_ops.fp8_quantize(x.to(cuda), block_rows)[0], q) and same(ffn_ops.fp8_quantize(x.to(cuda), block_rows, False, True)[1], qt)
    wide = torch.zeros(R, C + 7, dtype=dtype, device=cuda)
    wide[:, 3:3 + C] = x.to(cuda)
    q3 = ffn_ops.fp8_quantize(wide[:, 3:3 + C], block_rows, True, True)
    assert same(q3[0], q) and same(q3[1], qt)


@BOTH
def test_fp8_quantize_extremes(cuda, dtype):
    x = torch.zeros(6, 256)
    x[0, 5], x[1, 7], x[2, 9] = math.inf, -math.inf, math.nan
    x[0, :4], x[2, 128:] = 100.0, 3.0
    x[3, 0], x[3, 1] = 2.0 ** -130, 3e38                                       # fp32 subnormal next to the largest values
    x[4, :2] = torch.tensor([2.0 ** -133, 2.0 ** -149])
    x = x.to(dtype)
    got = d(ffn_ops.fp8_quantize(x.to(cuda))[0].values())
    want = fo.quantise(d(x))
    np.testing.assert_array_equal(got, want)
    # 100 = 400 / 4 in its block; 400 lies halfway between 384 and 416, and 384 (mantissa 100) is the even one: 96
    assert np.isnan(got[0, 5]) and np.isnan(got[1, 7]) and np.isnan(got[2, 9]) and got[0, 0] == 96 and got[2, 200] == 3


SHAPES = [(1, 1, 1), (1, 128, 16), (1, 515, 33), (2, 1000, 129), (7, 256, 7), (16, 384, 256), (17, 130, 64), (33, 640, 100), (64, 512, 200),
          (65, 127, 257), (128, 128, 128), (129, 1152, 130), (300, 257, 1), (500, 3136, 256), (513, 300, 515), (1030, 96, 1025)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@BOTH
def test_fp8_matmul_exact_on_whole_numbers(cuda, dtype, M, K, N):
    """whole numbers times block scales: every partial sum is a whole number below 2^24 times one power of two, so the result has
    to be exact, whatever the order of the sums."""
    rs = np.random.RandomState(M + K + N)
    x, w = rs.randint(-8, 9, (M, K)).astype(np.float64), rs.randint(-8, 9, (N, K)).astype(np.float64)
    sx, sw = 2.0 ** rs.randint(-2, 3, (M, 1)), 2.0 ** rs.randint(-2, 3, (1, 1))
    kb = np.arange(K) // 128                                                    # blocks differ in scale; products stay whole / 256
    x, w = x * 2.0 ** (kb % 3) * sx, w * 2.0 ** -(kb % 3) * sw
    b = rs.randint(-4, 5, N).astype(np.float32)
    xt, wt = torch.from_numpy(x).float().to(dtype).to(cuda), torch.from_numpy(w).float().to(cuda)
    assert np.array_equal(d(xt), x)
    want = x @ w.T + b
    y = ffn_ops.fp8_linear(xt, ffn_ops.Fp8Weight(wt, torch.from_numpy(b).to(cuda)), out_dtype=torch.float32)
    np.testing.assert_array_equal(d(y), want)
    r = ffn_ops.fp8_linear(xt.view(1, M, K), ffn_ops.Fp8Weight(wt), act="relu", out_dtype=torch.bfloat16)
    want = torch.from_numpy(np.maximum(x @ w.T, 0)).to(torch.bfloat16).double().numpy()[None]
    np.testing.assert_array_equal(d(r), want)


def _product_tol(a, b, dtype, out):
    return (2 * a.shape[1] * U32 + (7 * 2.0 ** -16 if dtype == torch.bfloat16 else 0)) * (np.abs(a) @ np.abs(b).T) + U[dtype] * np.abs(out) + 4 * U32 * np.abs(out)


@pytest.mark.parametrize("M,K,N", SHAPES)
@BOTH
def test_fp8_linear_against_64_bits(cuda, dtype, M, K, N):
    rs = np.random.RandomState(M * 3 + K + N)
    x, w = _values(rs, M, K, dtype), torch.from_numpy((rs.randn(N, K) / K ** 0.5).astype(np.float32))
    b = torch.from_numpy(rs.randn(N).astype(np.float32))
    xq, wq = fo.quantise(d(x)), fo.quantise(d(w), 128)
    plan = ffn_ops.Fp8Weight(w.to(cuda), b.to(cuda))
    pre = xq @ wq.T + d(b)
    for act in ("none", "relu", "gelu"):
        want = fo.act(pre, act)
        tol = 1.13 * (_product_tol(xq, wq, dtype, 0 * pre) + 8 * U32 * np.abs(pre) + U32 * np.abs(d(b))) + 4 * U32 * np.abs(pre) + U[dtype] * np.abs(want)   # |gelu'| <= 1.13
        if act == "gelu" and dtype == torch.bfloat16:       # the tail Phi(-|x|) of a bf16 result is a fit to 2.6e-4 relative
            tol = tol + 2.6e-4 * np.abs(pre) * (0.5 - 0.5 * fo._erf(np.abs(pre) / math.sqrt(2)))
        got = ffn_ops.fp8_linear(x.to(cuda), plan, act)
        assert got.dtype == dtype
        within(got, want, tol, act)
    if K * N >= 4096 and M >= 16:               # at random, K roundings of 2u add up to about 2u sqrt(K) of the result
        got = d(ffn_ops.fp8_linear(x.to(cuda), plan, out_dtype=torch.float32))
        assert np.linalg.norm(got - pre) <= 4 * U32 * math.sqrt(K) * np.linalg.norm(pre)


def test_fp8_weight_from_blocks_and_infinities(cuda):
    rs = np.random.RandomState(0)
    w = torch.from_numpy(rs.randn(200, 300).astype(np.float32)).to(cuda)
    a = ffn_ops.Fp8Weight(w)
    e = torch.from_numpy(fo.block_exponents(d(w), 128)).to(cuda)
    v = (w * torch.exp2(-e.float()).repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :300]).to(torch.float8_e4m3fn)
    b = ffn_ops.Fp8Weight.from_blocks(v, e)
    assert all(torch.equal(p, q) for p, q in zip(a.data.bytes_and_exponents(), b.data.bytes_and_exponents()))
    x = torch.randn(5, 300, device=cuda)
    x[2, 17] = math.inf
    y = ffn_ops.fp8_linear(x, b)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4]]).all()     # an infinity marks its own row only
    z = ffn_ops.fp8_linear(torch.zeros(3, 300, device=cuda), b)
    assert (z == 0).all()


@pytest.mark.parametrize("etype", [torch.int8, torch.uint8, torch.int16, torch.int64])
def test_fp8_weight_exponents_of_any_integer_type(cuda, etype):
    """exponents in a narrow type stand for what they say, and those past -126 .. 127 for the nearer end."""
    v = torch.ones(3, 200, device=cuda).to(torch.float8_e4m3fn)
    for a, b in ((5, 3), (torch.iinfo(etype).max, 0), (max(torch.iinfo(etype).min, -200), 1)):
        e = torch.tensor([[a, b]], dtype=etype, device=cuda)
        got = ffn_ops.Fp8Weight.from_blocks(v, e).data.bytes_and_exponents()[1]
        assert got.tolist() == [[max(-126, min(127, a)), b]] * 3


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16], ids=["w32", "w16"])
@BOTH
@pytest.mark.parametrize("M,K,N,bias", [(1, 8, 8, True), (5, 130, 260, False), (130, 257, 96, True), (512, 640, 256, True), (700, 129, 515, False)])
def test_fp8_linear_train(cuda, dtype, wdtype, M, K, N, bias):
    rs = np.random.RandomState(M + K)
    x = _values(rs, M, K, dtype).to(cuda).requires_grad_()
    w = torch.from_numpy((rs.randn(N, K) / K ** 0.5).astype(np.float32)).to(wdtype).to(cuda).requires_grad_()
    b = torch.from_numpy(rs.randn(N).astype(np.float32)).to(cuda).requires_grad_() if bias else None
    g = _values(rs, M, N, dtype).to(cuda)
    y = ffn_ops.fp8_linear_train(x.view(1, M, K), w, b)[0]
    leaves = [x, w] + ([b] if bias else [])
    dx, dw, *db = torch.autograd.grad(y, leaves, g)
    xq, wq = fo.quantise(d(x)), fo.quantise(d(w), 128)
    want = xq @ wq.T + (d(b) if bias else 0)
    within(y, want, _product_tol(xq, wq, dtype, want) + (U32 * np.abs(d(b)) if bias else 0), "y")
    gq, gt, xt = fo.quantise(d(g)), fo.quantise(d(g).T), fo.quantise(d(x).T)
    want = gq @ wq
    within(dx, want, _product_tol(gq, wq.T, dtype, want), "dx")
    want = gt @ xt.T
    assert dw.dtype == wdtype
    within(dw, want, _product_tol(gt, xt, wdtype, want), "dw")
    if bias:
        want = d(g).sum(0)
        within(db[0], want, U32 * np.abs(want) + (M + 8) * U32 * np.abs(d(g)).sum(0), "db")


def _whole(gen, R, C, step, cuda):
    """[R, C] of whole numbers up to 8 times a power of two for each row and, by 2^(+-block % 3), each block of 128 columns: e4m3 holds
    them exactly, and products of two such operands with opposite steps are whole numbers times their rows' powers."""
    v = torch.randint(-8, 9, (R, C), generator=gen, device=cuda).float()
    return v * torch.exp2(step * (torch.arange(C, device=cuda) // 128 % 3).float())


@pytest.mark.parametrize("case", pc.CASES, ids=lambda c: "x".join(map(str, c[0])) + ("-fp32" if c[1] == pc.F32 else "-bf16") + ("-laid" if c[2] else ""))
def test_fp8_products_of_every_kernel_are_exact(large, cuda, case):
    """Whole numbers: partial sums stay below 5129 * 64 * 2^3 * 2^2 < 2^24 steps of the smallest power, so fp32 results are exact in any
    order of the sums, and bf16 ones are rounded once (all products of an instruction lie within its 16 bits)."""
    (M, K, N), out, laid, kind, rest = case
    got = _lib.lib().pn_fp8_kernels(M, N, K, out, laid)
    assert (got & 15, got >> 4) == (kind, rest)
    dtype = torch.float32 if out == pc.F32 else torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(M + N)
    x = _whole(gen, M, K, 1, cuda) * torch.exp2(torch.randint(-2, 3, (M, 1), generator=gen, device=cuda).float())
    w = _whole(gen, N, K, -1, cuda) * torch.exp2((torch.arange(N, device=cuda) // 128 % 2).float())[:, None]
    b = torch.randint(-4, 5, (N,), generator=gen, device=cuda).float()
    want = x.double() @ w.double().t() + b.double()
    x = x.to(dtype)
    if laid:
        y = ffn_ops.fp8_matmul(ffn_ops.fp8_quantize(x)[0], ffn_ops.fp8_quantize(w, 128)[0], b, out_dtype=dtype)
    else:
        y = ffn_ops.fp8_linear(x, ffn_ops.Fp8Weight(w, b))
    assert y.dtype == dtype and torch.equal(y, want.to(torch.float32).to(dtype))
    plan = ffn_ops.Fp8Weight(w)                                                  # the public entry, ReLU in the epilogue, no bias
    assert torch.equal(ffn_ops.fp8_linear(x, plan, "relu"), (want - b.double()).relu().to(torch.float32).to(dtype))


@pytest.mark.parametrize("case", pc.TRAIN, ids=lambda c: "x".join(map(str, c[0])) + ("-fp32" if c[1] == pc.F32 else "-bf16"))
def test_fp8_training_products_of_every_kernel_are_exact(large, cuda, case):
    (M, K, N), out, kinds = case
    assert tuple(_lib.lib().pn_fp8_kernels(*q, 1) for q in pc.products(M, K, N, out)) == kinds
    dtype = torch.float32 if out == pc.F32 else torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(M)
    whole = lambda *s: torch.randint(-8, 9, s, generator=gen, device=cuda).float()
    x, w, g = whole(M, K).to(dtype).requires_grad_(), whole(N, K).requires_grad_(), whole(M, N).to(dtype)
    b = whole(N).requires_grad_()
    y = ffn_ops.fp8_linear_train(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    X, W, G = (t.detach().double() for t in (x, w, g))
    assert torch.equal(y, (X @ W.t() + b.double()).float().to(dtype))           # sums below 6314 * 64 < 2^19
    assert torch.equal(dx, (G @ W).float().to(dtype))
    assert torch.equal(dw, (G.t() @ X).float()) and torch.equal(db, G.sum(0).float())


@pytest.mark.parametrize("M,K,N", [(8, 384, 64), (300, 90, 300), (2104, 1160, 69), (2312, 1160, 2312)])
@pytest.mark.parametrize("k", [100, 124, 126, 130, 135])
def test_fp8_products_of_tiny_rows(cuda, M, K, N, k):
    """rows down to fp32's smallest normal numbers, on every kind of kernel: a bf16 result is what it is at any scale, an fp32 result is off by
    half of bf16's smallest step, 2^-134, for each value of x beyond its sums' rounding."""
    gen = torch.Generator(device="cuda").manual_seed(K)
    x, w = _whole(gen, M, K, 0, cuda), _whole(gen, N, K, 0, cuda)
    x[:, ::5] *= 2.0 ** -9
    x[:, ::7] *= 56
    x = (x.double() * 2.0 ** -k).float()
    xq, W = ffn_ops.fp8_quantize(x)[0].values().double(), w.double()
    want, mags = xq @ W.t(), xq.abs() @ W.abs().t()
    plan = ffn_ops.Fp8Weight(w)
    y = ffn_ops.fp8_linear(x, plan)
    assert ((y.double() - want).abs() <= 2 * K * U32 * mags + 2.0 ** -134 * W.abs().sum(1) + 2.0 ** -149).all()
    y = ffn_ops.fp8_linear(x, plan, out_dtype=torch.bfloat16)
    assert ((y.double() - want).abs() <= (2 * K * U32 + 7 * 2.0 ** -16) * mags + U[torch.bfloat16] * want.abs() + 2.0 ** -134).all()


def test_fp8_matmul_refusals(cuda):
    x, w = (ffn_ops.fp8_quantize(torch.randn(*s, device=cuda))[0] for s in ((6, 64), (32, 64)))
    assert ffn_ops.fp8_matmul(x, w).shape == (6, 32)
    assert ffn_ops.fp8_matmul(ffn_ops.fp8_quantize(torch.zeros(0, 64, device=cuda))[0], w).shape == (0, 32)
    b = torch.zeros(32, device=cuda)
    for call in (lambda: ffn_ops.fp8_matmul(torch.zeros(6, 64, device=cuda), w), lambda: ffn_ops.fp8_matmul(x, ffn_ops.fp8_quantize(torch.zeros(32, 65, device=cuda))[0]),
                 lambda: ffn_ops.fp8_matmul(x, w, b[:5]), lambda: ffn_ops.fp8_matmul(x, w, b.cpu()), lambda: ffn_ops.fp8_matmul(x, w, act="silu"),
                 lambda: ffn_ops.fp8_matmul(x, w, out_dtype=torch.float16)):
        with pytest.raises(PillarnetHipError):
            call()


def test_fp8_linear_train_gradient_against_differences(cuda):
    """where the rounding is exact (small whole numbers) the product is linear, and differences are exact."""
    rs = np.random.RandomState(4)
    x = torch.from_numpy(rs.randint(-7, 8, (6, 140)).astype(np.float32)).to(cuda).requires_grad_()
    w = torch.from_numpy(rs.randint(-7, 8, (10, 140)).astype(np.float32)).to(cuda).requires_grad_()
    b = torch.from_numpy(rs.randint(-7, 8, 10).astype(np.float32)).to(cuda).requires_grad_()
    g = torch.from_numpy(rs.randint(-3, 4, (6, 10)).astype(np.float32)).to(cuda)
    grads = torch.autograd.grad(ffn_ops.fp8_linear_train(x, w, b), (x, w, b), g)
    for leaf, gr in zip((x, w, b), grads):
        for at in [(0,) * leaf.dim(), tuple(s - 1 for s in leaf.shape)]:
            keep = leaf.detach()[at].item()
            vals = []
            for s in (1.0, -1.0):
                with torch.no_grad():
                    leaf[at] = keep + s
                    vals.append((ffn_ops.fp8_linear_train(x, w, b) * g).double().sum().item())
                    leaf[at] = keep
            assert (vals[0] - vals[1]) / 2 == gr[at].item()


def test_fp8_partial_gradients_and_refusals(cuda):
    x, w = torch.randn(20, 64, device=cuda), torch.randn(32, 64, device=cuda)
    b = torch.randn(32, device=cuda, requires_grad=True)
    full = [t.clone().requires_grad_() for t in (x, w)]
    ref = torch.autograd.grad(ffn_ops.fp8_linear_train(*full, b).sum(), full + [b])
    for i in range(2):
        leaves = [t.clone().requires_grad_(k == i) for k, t in enumerate((x, w))]
        assert torch.equal(torch.autograd.grad(ffn_ops.fp8_linear_train(*leaves, b.detach()).sum(), leaves[i])[0], ref[i])
    assert torch.equal(torch.autograd.grad(ffn_ops.fp8_linear_train(x, w, b).sum(), b)[0], ref[2])
    e = torch.zeros(0, 64, device=cuda, requires_grad=True)
    wl = w.clone().requires_grad_()
    de, dw, db = torch.autograd.grad(ffn_ops.fp8_linear_train(e, wl, b).sum(), (e, wl, b))
    assert de.shape == (0, 64) and (dw == 0).all() and (db == 0).all()
    plan = ffn_ops.Fp8Weight(w)
    assert ffn_ops.fp8_linear(e.detach(), plan).shape == (0, 32)
    for call in (lambda: ffn_ops.fp8_linear(x[:, :60], plan), lambda: ffn_ops.fp8_linear(x, w), lambda: ffn_ops.fp8_linear(x.half(), plan),
                 lambda: ffn_ops.fp8_linear(x.clone().requires_grad_(), plan), lambda: ffn_ops.fp8_linear(x, plan, act="silu"),
                 lambda: ffn_ops.fp8_linear(x, plan, out_dtype=torch.float16), lambda: ffn_ops.Fp8Weight(w, b[:5]),
                 lambda: ffn_ops.fp8_linear_train(x, w.t()), lambda: ffn_ops.fp8_linear_train(x, w, b[:3]),
                 lambda: ffn_ops.fp8_quantize(x, 64), lambda: ffn_ops.fp8_quantize(x, rows=False),
                 lambda: ffn_ops.Fp8Weight.from_blocks(w.to(torch.float8_e4m3fn), torch.zeros(2, 1, device=cuda, dtype=torch.int32)),
                 lambda: ffn_ops.Fp8Weight.from_blocks(w, torch.zeros(1, 1, device=cuda, dtype=torch.int32))):
        with pytest.raises(PillarnetHipError):
            call()


def test_fp8_beyond_32_bit_offsets(large, cuda):
    """x and out of 4.3e9 elements each: the last rows are those of a call of their own (the same sums, other kernels: whole numbers)."""
    M, K, N = (1 << 21) + 5, 2056, 24
    x = torch.zeros((M, K), dtype=torch.bfloat16, device=cuda)
    x[-300:] = torch.randint(-3, 4, (300, K), device=cuda).bfloat16()
    w = torch.randint(-3, 4, (N, K), device=cuda).float()
    y = ffn_ops.fp8_linear(x, ffn_ops.Fp8Weight(w), out_dtype=torch.float32)
    assert torch.equal(y[-300:], x[-300:].float() @ w.t()) and (y[: 300] == 0).all()
    q, s = ffn_ops.fp8_quantize(x, rows=False, transposed=True)[1]._parts()
    B = q.shape[1]                                                           # (the last three blocks of the transpose, by hand)
    vals = q[:, -3:].permute(0, 4, 1, 3, 2, 5).reshape(-1, 3 * 128)[:K].view(torch.float8_e4m3fn).float()
    scale = torch.stack([s[b // 4, :, b % 4] for b in range(B - 3, B)], 1).int() << 23
    got = (vals * scale.view(torch.float32).repeat_interleave(128, 1))[:, : M - (B - 3) * 128]
    assert torch.equal(got[:, -200:], x[-200:].float().t())
    del x, q, s, y
    K, N = 128, 2056
    x = torch.zeros((M, K), dtype=torch.bfloat16, device=cuda)
    x[-300:] = torch.randint(-3, 4, (300, K), device=cuda).bfloat16()
    w = torch.randint(-3, 4, (N, K), device=cuda).float()
    y = ffn_ops.fp8_linear(x, ffn_ops.Fp8Weight(w))
    assert torch.equal(y[-300:], (x[-300:].float() @ w.t()).bfloat16()) and (y[: 300] == 0).all()


def test_second_derivatives_are_refused(cuda):
    """create_graph gives the first gradient; asking for the gradient of it raises instead of giving zeros."""
    x = torch.randn(6, 64, device=cuda, requires_grad=True)
    w = torch.randn(32, 64, device=cuda, requires_grad=True)
    for call in (lambda: ffn_ops.act_dropout(x, 0.0, act="gelu"), lambda: ffn_ops.residual_norm(x, norm=ffn_ops.Norm("rms")),
                 lambda: ffn_ops.fp8_linear_train(x, w)):
        (g,) = torch.autograd.grad(call().square().sum(), x, create_graph=True)
        (want,) = torch.autograd.grad(call().square().sum(), x)
        assert torch.equal(g, want)
        with pytest.raises(RuntimeError):                       # torch finds no way from g to x
            torch.autograd.grad(g.sum(), x, retain_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_forward_mode_tangents_are_refused(cuda):
    from pillarnet_lts_amd import second_stage
    fw = torch.autograd.forward_ad
    x, w = torch.randn(6, 64, device=cuda), torch.randn(32, 64, device=cuda)
    plan = ffn_ops.Fp8Weight(w)
    head = second_stage.RoIHeadTemplate(1, {}).to(cuda)
    head.fp8 = True
    fc = torch.nn.Linear(64, 32).to(cuda).requires_grad_(False)
    with fw.dual_level():
        t = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: ffn_ops.act_dropout(t, 0.0, act="gelu"), lambda: ffn_ops.residual_norm(t, norm=ffn_ops.Norm("rms")),
                     lambda: ffn_ops.residual_norm(x, t), lambda: ffn_ops.fp8_linear_train(t, w), lambda: ffn_ops.fp8_linear(t, plan),
                     lambda: head.fused_linear(fc, t)):
            with pytest.raises(PillarnetHipError, match="no forward-mode derivative"):
                call()
        assert head.fused_linear(fc, x).shape == (6, 32)


# ---- together ----------------------------------------------------------------------------------------------------------
def test_feed_forward_block_captured_and_on_another_stream(cuda):
    """one block as the heads use it -- norm, fp8 product, activation + dropout, fp8 product, residual join -- forward and backward,
    eagerly, on a side stream, and captured with a draw inside: every replay gives the eager pass's bits for its draw."""
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen).to(cuda)
    x0, g = r(3, 50, 96), r(3, 50, 96)
    P = dict(w1=r(192, 96) / 10, b1=r(192), w2=r(96, 192) / 14, b2=r(96), nw=r(96), nb=r(96), gate=r(3, 96), pw=r(96), pb=r(96))
    st = ffn_ops.DropoutState(42, cuda)

    def step(rng):
        x, p = x0.clone().requires_grad_(), {k: v.clone().requires_grad_() for k, v in P.items()}
        n = ffn_ops.residual_norm(x, norm=ffn_ops.Norm("layer", p["nw"], p["nb"]))
        a = ffn_ops.act_dropout(ffn_ops.fp8_linear_train(n, p["w1"], p["b1"]), 0.2, rng, 0, "gelu")
        f = ffn_ops.fp8_linear_train(a, p["w2"], p["b2"])
        h, y = ffn_ops.residual_norm(x, f, gate=p["gate"], scale=0.7, post_norm=ffn_ops.Norm("rms", p["pw"], p["pb"]),
                                     norm=ffn_ops.Norm("layer", p["nw"], p["nb"]), dropout=(0.1, rng, 1))
        return [h, y, *torch.autograd.grad((h, y), [x, *p.values()], (g, g))]

    want = [[t.detach().clone() for t in step(rng_of(42, i, cuda))] for i in range(4)]
    assert any(not torch.equal(a, b) for a, b in zip(want[0], want[1]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(st.draw())
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want[0]):
        assert torch.equal(a, b)
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [t.detach() for t in step(st.draw())]
    for i in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(out, want[i])):
            assert torch.equal(a, b), (i, k)
        (x0 @ P["w1"].t()).relu().sum().item()                                   # eager work between replays


def test_operators_under_torchs_other_modes(cuda):
    """inference mode, activation checkpointing (the second forward pass draws the same masks) and saved tensors kept on the host give
    the bits of the plain pass."""
    from torch.utils.checkpoint import checkpoint
    gen = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen).to(cuda).requires_grad_()
    x, w1, b1, w2, nw, gate, rng = r(40, 72), r(136, 72), r(136), r(72, 136), r(72), r(72), rng_of(8, 1, cuda)
    leaves, g = [x, w1, b1, w2, nw, gate], torch.randn(40, 72, generator=gen).to(cuda)

    def block(x):
        a = ffn_ops.act_dropout(ffn_ops.fp8_linear_train(x, w1, b1), 0.3, rng, 0, "gelu")
        return ffn_ops.residual_norm(x, ffn_ops.fp8_linear_train(a, w2), gate=gate, norm=ffn_ops.Norm("rms", nw), dropout=(0.3, rng, 1))[1]

    y = block(x)
    want = torch.autograd.grad(y, leaves, g)
    with torch.inference_mode():
        assert torch.equal(block(x.detach()), y)
    z = checkpoint(block, x, use_reentrant=False)
    assert torch.equal(z, y)
    for a, b in zip(torch.autograd.grad(z, leaves, g), want):
        assert torch.equal(a, b)
    with torch.autograd.graph.save_on_cpu():
        z = block(x)
    for a, b in zip(torch.autograd.grad(z, leaves, g), want):
        assert torch.equal(a, b)
    y = block(x)
    with torch.no_grad():
        nw.mul_(2)                                                 # a parameter that the backward pass reads
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves, g)


def test_an_entrys_refusal_is_the_frameworks_error(cuda):
    B = (1 << 23) + 1
    x = torch.zeros(B, 2, 1, device=cuda)
    with pytest.raises(PillarnetHipError, match="gates of several rows"):
        ffn_ops.residual_norm(x, x, gate=torch.zeros(B, 1, device=cuda))
    x.requires_grad_()
    with pytest.raises(PillarnetHipError, match="gates of several rows"):
        ffn_ops.residual_norm(x, x, gate=torch.zeros(B, 1, device=cuda))


def test_a_refusal_in_a_backward_pass_is_the_frameworks_error(cuda):
    """an entry that refuses its arguments on the engine's thread; the hooks hand the nodes saved tensors that the host's checks refuse."""
    x, w, rng = torch.randn(6, 64, device=cuda, requires_grad=True), torch.randn(32, 64, device=cuda), rng_of(1, 2, cuda)
    off = lambda t, step: torch.empty(t.numel() + step, dtype=t.dtype, device=cuda)[step:].view(t.shape)
    cases = [(lambda: ffn_ops.residual_norm(x, norm=ffn_ops.Norm("rms")), lambda t: off(t, 1) if t.shape == (6, 4) else t, "16-byte aligned"),
             (lambda: ffn_ops.act_dropout(x, 0.5, rng), lambda t: t[:0].clone() if t.dtype == torch.int64 else t, "generator's state"),
             (lambda: ffn_ops.fp8_linear_train(x, w), lambda t: off(t, 1), "256-byte alignment")]
    for call, unpack, says in cases:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y, z = call(), call()
        with pytest.raises(PillarnetHipError, match=says):
            y.sum().backward()
        with pytest.raises(PillarnetHipError, match=says):
            torch.autograd.grad(z.sum(), x)
    assert torch.isfinite(torch.autograd.grad(ffn_ops.fp8_linear_train(x, w).sum(), x)[0]).all()


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_draw_inside_a_recomputed_pass_is_refused(cuda, reentrant):
    """it would drop other elements than the pass whose gradient is asked for; drawn outside, checkpointing gives the plain gradient."""
    from torch.utils.checkpoint import checkpoint
    st, x = ffn_ops.DropoutState(3, cuda), torch.randn(8, 64, device=cuda, requires_grad=True)
    y = checkpoint(lambda x: ffn_ops.act_dropout(x, 0.5, st.draw(), act="gelu").square(), x, use_reentrant=reentrant)
    with pytest.raises(PillarnetHipError, match="inside a backward pass"):
        y.sum().backward()
    rng = st.draw()
    block = lambda x: ffn_ops.act_dropout(x, 0.5, rng, act="gelu").square()
    x.grad = None
    checkpoint(block, x, use_reentrant=reentrant).sum().backward()
    assert torch.equal(x.grad, torch.autograd.grad(block(x).sum(), x)[0])
