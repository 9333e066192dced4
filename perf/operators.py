"""What is measured of the operators of a feed-forward block: activation + dropout from a counter-based generator, residual
join + norms + gate, and the product in 8-bit floating point with one scale for each block of 128.

`listed()` / `draw()` give cases, `prepare()` the inputs, `run()` one pass (plain torch operations, or with `own` the
framework's operators), `work()` what a pass cannot do without, `exact()` the same outputs from the definitions in 64 bits."""
import functools
import math

import torch

own = False


# ---- cases -------------------------------------------------------------------------------------------------------------
def _dropout(rows, cols, dtype, act, p, **kw):
    return dict(op="dropout", rows=rows, cols=cols, dtype=dtype, act=act, p=p, **kw)


def _norm(samples, rows, cols, dtype, post, norm, gate, p, train, **kw):
    return dict(op="norm", samples=samples, rows=rows, cols=cols, dtype=dtype, post=post, norm=norm, gate=gate, p=p,
                train=train, **kw)


def _product(m, k, n, dtype, act, train, **kw):
    return dict(op="fp8", m=m, k=k, n=n, dtype=dtype, act=act, train=train, **kw)


def listed():
    return [
        # ReLU + dropout behind a 256-wide RoI layer: four images of 128 sampled RoIs, forward and backward
        _dropout(512, 256, "float32", "relu", 0.3, name="dropout_roi_fc"),
        # GELU + dropout at an odd width and row count, forward and backward
        _dropout(6271, 1023, "float32", "gelu", 0.1, name="dropout_gelu_odd"),
        # ReLU + dropout on the widened rows of a feed-forward block, a large training batch, forward and backward
        _dropout(65536, 2048, "bfloat16", "relu", 0.1, name="dropout_ffn_wide"),
        # the RoI feed-forward head while serving: 500 RoIs of one frame, residual + LayerNorm
        _norm(1, 500, 256, "float32", "none", "layer", "none", 0.0, False, name="norm_roi_serve"),
        # the mixer's channel norm while training: 512 RoIs x 49 grid points x 64 channels
        _norm(512, 49, 64, "float32", "none", "layer", "none", 0.0, True, name="norm_mixer_train"),
        # a block with norms on both sides, a gate for each sample and dropout, ragged row count, training
        _norm(16, 1031, 2048, "bfloat16", "rms", "rms", "sample", 0.1, True, name="norm_sandwich_train"),
        # wide rows while serving: layer scale on the branch, LayerNorm for the next block
        _norm(1, 32768, 4096, "bfloat16", "none", "layer", "channel", 0.0, False, name="norm_wide_serve"),
        # one row through a wide layer: the weights' read is what counts
        _product(1, 8192, 8192, "bfloat16", "none", False, name="fp8_one_row"),
        # the first shared layer of the RoI head while serving: 500 RoIs x (49 x 64) -> 256, bias + ReLU
        _product(500, 3136, 256, "float32", "relu", False, name="fp8_roi_fc_serve"),
        # the same layer while training on 512 sampled RoIs: output, input, weight and bias gradients
        _product(512, 3136, 256, "float32", "none", True, name="fp8_roi_fc_train"),
        # a feed-forward layer while training on many rows, row count ragged
        _product(8200, 2048, 4096, "bfloat16", "none", True, name="fp8_ffn_train"),
        # a wide feed-forward layer over many rows while serving, bias + GELU
        _product(16384, 4096, 8192, "bfloat16", "gelu", False, name="fp8_ffn_wide"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["dropout", "norm", "fp8"])
    dtype = rng.choice(["float32", "bfloat16"])
    if op == "dropout":
        cols = _log(rng, 16, 4100)
        rows = min(_log(rng, 1, 65536), (1 << 26) // cols)
        return _dropout(rows, cols, dtype, rng.choice(["none", "relu", "gelu"]), rng.choice([0.1, 0.3, 0.5]))
    if op == "norm":
        cols = _log(rng, 16, 8192)
        samples = rng.randint(1, 32)
        rows = max(1, min(_log(rng, 1, 2048), (1 << 24) // (cols * samples)))
        return _norm(samples, rows, cols, dtype, rng.choice(["none", "layer", "rms"]), rng.choice(["layer", "rms", "affine"]),
                     rng.choice(["none", "channel", "sample"]), rng.choice([0.0, 0.1]), rng.choice([True, False]))
    train = rng.choice([True, False])
    k, n = _log(rng, 64, 8192), _log(rng, 8, 8192)
    m = max(1, min(_log(rng, 1, 16384), (1 << (36 if train else 38)) // (k * n)))
    return _product(m, k, n, dtype, "none" if train else rng.choice(["none", "relu", "gelu"]), train)


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _dtype(case):
    return getattr(torch, case["dtype"])


def prepare(case, seed):
    """Inputs on the GPU from the seed alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = _dtype(case)

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(mean, std, generator=gen).to(dtype)

    s = dict(case=dict(case), rng=torch.randint(0, 1 << 62, (2,), generator=gen, device="cuda", dtype=torch.int64))
    if case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        s.update(x=normal(*shape).requires_grad_(), g=normal(*shape))
    elif case["op"] == "norm":
        B, T, C = case["samples"], case["rows"], case["cols"]
        s.update(x=normal(B, T, C, std=2.0, mean=0.1), f=normal(B, T, C, std=0.5, mean=0.05), gh=normal(B, T, C),
                 gy=normal(B, T, C), w=normal(C, std=0.1, mean=1.0), b=normal(C, std=0.1),
                 pw=normal(C, std=0.1, mean=1.0), pb=normal(C, std=0.1),
                 gate=normal(C, std=0.2, mean=0.5) if case["gate"] == "channel" else normal(B, C, std=0.2, mean=0.5))
        if case["train"]:
            for k in ("x", "f", "w", "b", "pw", "pb", "gate"):
                s[k].requires_grad_()
    else:
        M, K, N = case["m"], case["k"], case["n"]
        # rows of a feature map after a ReLU-like layer differ in size from row to row
        x = normal(M, K, dtype=torch.float32) * normal(M, 1, std=0.7, dtype=torch.float32).exp()
        w, b = normal(N, K, std=K ** -0.5, dtype=torch.float32), normal(N, std=0.1, dtype=torch.float32)
        s.update(x=x.to(dt))
        if case["train"]:           # master weights in 32 bits
            s.update(w=w.requires_grad_(), b=b.requires_grad_(), g=normal(M, N))
            s["x"].requires_grad_()
        else:                       # a serving program keeps the weights as the bytes and exponents they were laid out in
            q, e = _quantise(w, 128)
            s.update(wq=q, we=e, b=b)
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------
def _pow2(e):
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantise(x, rows):
    """[R, C] in 32 bits -> e4m3 values of `x / 2^e`, and e for each block of `rows` x 128: the smallest exponent from
    -126 up with which the block's largest magnitude stays within 448 = 1.75 * 2^8."""
    R, C = x.shape
    r, c = -(-R // rows), -(-C // 128)
    v = torch.nn.functional.pad(x, (0, c * 128 - C, 0, r * rows - R)).view(r, rows, c, 128)
    bits = v.abs().amax((1, 3)).view(torch.int32)
    e = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000)).clamp(min=1) - 127
    q = (v * _pow2(-e)[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(r * rows, c * 128)[:R, :C].contiguous(), e


def _values(q, e, rows):
    """What the bytes of `_quantise` stand for."""
    R, C = q.shape
    s = _pow2(e).repeat_interleave(rows, 0)[:R].repeat_interleave(128, 1)[:, :C]
    return q.float() * s


def _rounded(x, rows):
    return _values(*_quantise(x, rows), rows)


def _mul(a, k):
    """high and low word of the product of 32-bit words held in 64-bit integers."""
    p = a * k
    return (p >> 32) & 0xFFFFFFFF, p & 0xFFFFFFFF


def _round(s, key):
    h0, l0 = _mul(s[0], 0xD2511F53)
    h1, l1 = _mul(s[2], 0xCD9E8D57)
    return h1 ^ s[1] ^ key[0], l1, h0 ^ s[3] ^ key[1], l0


def _keep(rng, count, p, call):
    """[count] truth values: 16-bit word i of the Philox4x32-10 stream reaches the threshold."""
    seed, off = rng[0], rng[1]
    lo, hi = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    j = torch.arange(-(-count // 8), device=rng.device)
    start = (j & 0xFFFFFFFF, ((j >> 32) & 0xFFFF) | (call << 16), (off & 0xFFFFFFFF).expand_as(j),
             ((off >> 32) & 0xFFFFFFFF).expand_as(j))
    words = functools.reduce(_round, [((lo + i * 0x9E3779B9) & 0xFFFFFFFF, (hi + i * 0xBB67AE85) & 0xFFFFFFFF)
                                      for i in range(10)], start)
    w = torch.stack(words, 1)
    return torch.stack((w & 0xFFFF, w >> 16), 2).view(-1)[:count] >= _threshold(p)


def _threshold(p):
    return min(65535, max(1, round(p * 65536)))


def _act(x, act):
    if act == "relu":
        return x.clamp(min=0)
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    return x


def _act_grad(x, act):
    if act == "relu":
        return (x > 0).to(x.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(x)


def _plain_dropout(s):
    c, x, g = s["case"], s["x"].float(), s["g"].float()
    k = _keep(s["rng"], x.numel(), c["p"], 0).view_as(x) * (65536 / (65536 - _threshold(c["p"])))
    dt = _dtype(c)
    return {"y": (_act(x, c["act"]) * k).to(dt), "dx": (g * k * _act_grad(x, c["act"])).to(dt)}


def _normalise(t, kind):
    """the normalised rows and the factor in front of them."""
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    if kind in ("layer", "rms"):
        r = torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-5)
        return t * r, r
    return t, torch.ones_like(t[..., :1])


def _normalise_grad(t, n, r, kind):
    """gradient of `_normalise` for a gradient t of its rows n."""
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    if kind in ("layer", "rms"):
        t = t - n * (t * n).mean(-1, keepdim=True)
    return t * r


def _plain_norm(s):
    c = s["case"]
    dt, B, T, C = _dtype(c), c["samples"], c["rows"], c["cols"]
    x, f, w, b, pw, pb = (s[k].float() for k in ("x", "f", "w", "b", "pw", "pb"))
    gate = {"none": 1.0, "channel": s["gate"].float(), "sample": s["gate"].float()[..., None, :]}[c["gate"]]
    k = 1.0
    if c["p"] > 0:
        k = _keep(s["rng"], f.numel(), c["p"], 1).view_as(f) * (65536 / (65536 - _threshold(c["p"])))
    fn, fr = _normalise(f, c["post"])
    v = (fn * pw + pb if c["post"] != "none" else fn) * k
    h = (x + 0.5 * gate * v).to(dt)                     # the norm reads what is stored
    hn, hr = _normalise(h.float(), c["norm"])
    out = {"h": h, "y": (hn * w + b).to(dt)}
    if not c["train"]:
        return out
    gh, gy = s["gh"].float(), s["gy"].float()
    dh = gh + _normalise_grad(gy * w, hn, hr, c["norm"])
    du = 0.5 * gate * dh * k
    out.update(dx=dh.to(dt), dw=(gy * hn).sum((0, 1)).to(dt), db=gy.sum((0, 1)).to(dt),
               df=(_normalise_grad(du * pw, fn, fr, c["post"]) if c["post"] != "none" else du).to(dt))
    if c["gate"] != "none":
        out["dgate"] = (0.5 * dh * v).sum(1 if c["gate"] == "sample" else (0, 1)).to(dt)
    if c["post"] != "none":
        out.update(dpw=(du * fn).sum((0, 1)).to(dt), dpb=du.sum((0, 1)).to(dt))
    return out


def _plain_fp8(s):
    c, x = s["case"], s["x"].float()
    dt = _dtype(c)
    if not c["train"]:
        return {"y": _act(_rounded(x, 1) @ _values(s["wq"], s["we"], 128).t() + s["b"], c["act"]).to(dt)}
    g, w = s["g"].float(), _rounded(s["w"], 128)
    return {"y": (_rounded(x, 1) @ w.t() + s["b"]).to(dt), "dx": (_rounded(g, 1) @ w).to(dt),
            "dw": _rounded(g.t(), 1) @ _rounded(x.t(), 1).t(), "db": g.sum(0)}


# ---- the framework's operators -----------------------------------------------------------------------------------------
def _own_dropout(s):
    from pillarnet_lts_amd import ffn_ops
    c = s["case"]
    y = ffn_ops.act_dropout(s["x"], c["p"], s["rng"], act=c["act"])
    return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["g"])[0]}


def _own_norm(s):
    from pillarnet_lts_amd import ffn_ops
    c = s["case"]
    gate = s["gate"] if c["gate"] != "none" else None
    post = ffn_ops.Norm(c["post"], s["pw"], s["pb"]) if c["post"] != "none" else None
    h, y = ffn_ops.residual_norm(s["x"], s["f"], gate=gate, scale=0.5, post_norm=post, norm=ffn_ops.Norm(c["norm"], s["w"], s["b"]),
                                 dropout=(c["p"], s["rng"], 1) if c["p"] > 0 else None)
    if not c["train"]:
        return {"h": h, "y": y}
    names = ["x", "f", "w", "b"] + (["gate"] if gate is not None else []) + (["pw", "pb"] if post is not None else [])
    grads = torch.autograd.grad((h, y), [s[k] for k in names], (s["gh"], s["gy"]))
    return {"h": h, "y": y, **{"d" + k: g for k, g in zip(names, grads)}}


def _own_fp8(s):
    from pillarnet_lts_amd import ffn_ops
    c = s["case"]
    if not c["train"]:
        if "plan" not in s:         # laid out once, as a program that serves does when it loads its weights
            s["plan"] = ffn_ops.Fp8Weight.from_blocks(s["wq"], s["we"], bias=s["b"])
        return {"y": ffn_ops.fp8_linear(s["x"], s["plan"], act=c["act"])}
    y = ffn_ops.fp8_linear_train(s["x"], s["w"], s["b"])
    dx, dw, db = torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["g"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"dropout": _own_dropout, "norm": _own_norm, "fp8": _own_fp8}[op](state)
    with torch.no_grad():
        return {"dropout": _plain_dropout, "norm": _plain_norm, "fp8": _plain_fp8}[op](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "dropout":     # x, g in; y, dx out
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * size * n, "flops": 4 * n}
    if case["op"] == "norm":        # x, branch in; h, y out; training: two gradients in, two out
        n = case["samples"] * case["rows"] * case["cols"]
        return {"bytes": (8 if case["train"] else 4) * size * n, "flops": (40 if case["train"] else 12) * n}
    m, k, n = case["m"], case["k"], case["n"]
    if not case["train"]:           # x, the weights' bytes and bias in; y out
        return {"bytes": size * m * (k + n) + n * k + 4 * n, "flops": 2 * m * n * k}
    return {"bytes": 2 * size * m * (k + n) + 8 * n * k + 8 * n, "flops": 6 * m * n * k}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _exact_keep(rng, shape, p, call):
    """the same stream, with the 64-bit product put together from 16-bit halves."""
    seed, off = (int(v) & (1 << 64) - 1 for v in rng.tolist())
    mask, n = 0xFFFFFFFF, math.prod(shape)
    i = torch.arange(-(-n // 8) * 8, device="cuda").view(-1, 8)[:, 0] // 8
    c = [i % (1 << 32), i // (1 << 32) % (1 << 16) + call * 65536, torch.full_like(i, off & mask), torch.full_like(i, off >> 32)]
    key = [seed & mask, seed >> 32]

    def wide(a, m):
        mid = a * (m % 65536)
        top = a * (m // 65536) + mid // 65536
        return top // 65536, top % 65536 * 65536 + mid % 65536

    for _ in range(10):
        (ah, al), (bh, bl) = wide(c[0], 0xD2511F53), wide(c[2], 0xCD9E8D57)
        c = [bh ^ c[1] ^ key[0], bl, ah ^ c[3] ^ key[1], al]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    u = torch.empty((i.numel(), 8), dtype=torch.int32, device="cuda")
    for k in range(4):
        u[:, 2 * k], u[:, 2 * k + 1] = c[k] % 65536, c[k] // 65536
    t = min(65535, max(1, round(p * 65536)))
    return torch.where(u.view(-1)[:n].view(shape) < t, 0.0, 65536 / (65536 - t)).double()


def _exact_act(x, act):
    """value and derivative."""
    if act == "relu":
        return torch.where(x > 0, x, 0.0), torch.where(x > 0, 1.0, 0.0).double()
    if act == "gelu":
        phi = torch.special.ndtr(x)
        return x * phi, phi + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    return x, torch.ones_like(x)


def _exact_e4m3(x, rows):
    """[R, C] doubles -> the nearest values (ties to even) of 4 significant bits with the block's exponent, no finer than
    its 2^-9 steps."""
    R, C = x.shape
    out = torch.empty_like(x)
    full = torch.zeros((-(-R // rows) * rows, -(-C // 128) * 128), dtype=torch.float64, device=x.device)
    full[:R, :C] = x
    v = full.view(-1, rows, full.shape[1] // 128, 128)
    m, e = torch.frexp(v.abs().amax((1, 3), keepdim=True) / 448)
    e = torch.where(m > 0.5, e, e - 1).clamp(min=-126)                # smallest e with amax / 448 <= 2^e
    scale = torch.exp2(e.double())
    t = v / scale
    step = torch.exp2(torch.frexp(t)[1].clamp(min=-5).double() - 4)   # 3 bits behind the first; subnormals from 2^-6 down
    out.copy_((torch.round(t / step) * step * scale).view(full.shape)[:R, :C])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and v.dtype in (torch.float32, torch.bfloat16)}
    if case["op"] == "dropout":
        k = _exact_keep(s["rng"], d["x"].shape, case["p"], 0)
        a, da = _exact_act(d["x"], case["act"])
        return {"y": a * k, "dx": d["g"] * k * da}
    if case["op"] == "fp8":
        if not case["train"]:
            w = s["wq"].double().clone()
            w *= torch.exp2(s["we"].double()).repeat_interleave(128, 0)[: w.shape[0]].repeat_interleave(128, 1)[:, : w.shape[1]]
            return {"y": _exact_act(_exact_e4m3(d["x"], 1) @ w.t() + d["b"], case["act"])[0]}
        w = _exact_e4m3(d["w"], 128)
        return {"y": _exact_e4m3(d["x"], 1) @ w.t() + d["b"], "dx": _exact_e4m3(d["g"], 1) @ w,
                "dw": _exact_e4m3(d["g"].t().contiguous(), 1) @ _exact_e4m3(d["x"].t().contiguous(), 1).t(), "db": d["g"].sum(0)}
    # the joined rows, differentiated by autograd in 64 bits; the norm reads the rows that were stored
    leaves = {k: d[k].requires_grad_() for k in ("x", "f", "w", "b", "pw", "pb", "gate")}
    x, f = leaves["x"], leaves["f"]

    def norm(t, kind, w, b):
        if kind == "layer":
            var, mean = torch.var_mean(t, -1, keepdim=True, correction=0)
            t = (t - mean) / torch.sqrt(var + 1e-5)
        elif kind == "rms":
            t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-5)
        return t * w + b

    v = norm(f, case["post"], leaves["pw"], leaves["pb"]) if case["post"] != "none" else f
    if case["p"] > 0:
        v = v * _exact_keep(s["rng"], f.shape, case["p"], 1)
    if case["gate"] != "none":
        v = v * (leaves["gate"] if case["gate"] == "channel" else leaves["gate"].unsqueeze(1))
    h = x + v / 2
    stored = h + (h.detach().to(_dtype(case)).double() - h.detach())
    y = norm(stored, case["norm"], leaves["w"], leaves["b"])
    out = {"h": h.detach(), "y": y.detach()}
    if case["train"]:
        names = ["x", "f", "w", "b"] + (["gate"] if case["gate"] != "none" else []) + (["pw", "pb"] if case["post"] != "none" else [])
        grads = torch.autograd.grad((stored, y), [leaves[k] for k in names], (d["gh"], d["gy"]))
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out
