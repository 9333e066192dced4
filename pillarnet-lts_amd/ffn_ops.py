"""Operators of the RoI heads' feed-forward blocks (det3d/models/roi_heads/roi_ffn_head.py:34-39,101-102, the FC stacks
with Dropout of roi_head_template.py:23-39, the mixers of mlp_layers.py:24-117) on hand-written kernels:

  act_dropout       activation + dropout; the mask is drawn again in the backward pass and never stored
  residual_norm     residual + scale * gate * dropout(post_norm(branch)), then the next block's norm
  fp8_linear        product in 8-bit floating point (e4m3) with a power-of-two scale for each block of 128
  fp8_linear_train  the same while training, with both gradients in fp8

All take fp32 or bf16 tensors on the GPU, run on the current stream of the tensors' device, allocate through torch's
caching allocator only and wait for nothing, so they can be captured into a HIP graph.  A graph that holds a backward pass
is captured while no eager autograd graph over the same leaves is alive (torch's own rule for captured backward passes).
Derivatives are reverse-mode and of first order: tensors with a forward-mode tangent are refused."""
from collections import namedtuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import PillarnetHipError

_DTYPES = {torch.float32: _lib.PN_DTYPE_F32, torch.bfloat16: _lib.PN_DTYPE_BF16}


def _require(cond, message):
    if not cond:
        raise PillarnetHipError(message)


def _check(what, *tensors):
    """GPU tensors of one device, fp32 or bf16."""
    dev = tensors[0].device
    for t in tensors:
        if t.device.type != "cuda":
            raise PillarnetHipError(f"{what}: tensors must live on the GPU (no CPU fallback)")
        if t.device != dev:
            raise PillarnetHipError(f"{what}: tensors on {dev} and {t.device}")
        if t.dtype not in _DTYPES:
            raise PillarnetHipError(f"{what}: {t.dtype} (fp32 or bf16)")


_FN = {}
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _call(name, device, *args):
    """One C entry on `device`'s current stream, with `device` current during the launch."""
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(_lib.lib(), name)
    i = device.index
    if i == _current_device():
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _raw_stream(i))
    if rc:
        _lib.check(rc, name)


_EXT = None


def _nodes():
    """The autograd nodes (csrc/ffn_autograd.cpp)."""
    global _EXT
    if _EXT is None:
        _EXT = _lib.autograd()
    return _EXT


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(x):
    """x as [rows, cols] with unit column stride and a row stride >= cols; a copy only where no view has them."""
    C = x.shape[-1]
    if x.is_contiguous():
        return x if x.dim() == 2 else x.view(-1, C) if C else x.reshape(0, 0)
    try:
        v = x.view(-1, C)
        if v.stride(1) == 1 and (v.shape[0] <= 1 or v.stride(0) >= C):
            return v
    except RuntimeError:
        pass
    return x.contiguous().view(-1, C)


def _strided(x):
    """(x or a copy of it, its row stride) as _rows, without a view where x is contiguous."""
    if x.is_contiguous():
        return x, x.shape[-1]
    x = _rows(x)
    return x, x.stride(0)


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_tangent(what, x):
    """Where a kernel is called outside of the autograd nodes: a tangent would be dropped without a word."""
    if forward_ad._current_level >= 0:
        _require(forward_ad.unpack_dual(x).tangent is None, f"{what}: no forward-mode derivative")


# ---- activation + dropout ----------------------------------------------------------------------------------------------
def dropout_threshold(p):
    """The 16-bit threshold of a drop probability: p is taken to the nearest 1 / 65536, at least one step for p > 0 and
    at most 65535 for p < 1; the kept elements are scaled by 65536 / (65536 - threshold), so the mean is kept exactly."""
    _require(0.0 <= p <= 1.0, f"dropout probability {p} (0 to 1)")
    if p == 0.0 or p == 1.0:
        return int(p) * 65536
    return min(65535, max(1, round(p * 65536)))


class DropoutState:
    """(seed, offset) of the generator in device memory.  `draw()` hands out the pair a pass uses -- an int64 tensor [2]
    that its forward and backward share -- and moves the offset on, on the device: a captured and replayed graph draws new
    masks on every replay."""

    def __init__(self, seed, device="cuda"):
        seed = int(seed) & (1 << 64) - 1
        self.state = torch.tensor([seed - (1 << 64) if seed >> 63 else seed, 0], dtype=torch.int64, device=device)
        _require(self.state.device.type == "cuda", "DropoutState: the state must live on the GPU (no CPU fallback)")

    def draw(self):
        _require(torch._C._current_graph_task_id() == -1, "DropoutState: no draw inside a backward pass (draw outside of what is checkpointed)")
        used = torch.empty_like(self.state)
        _call("pn_dropout_draw", self.state.device, self.state.data_ptr(), used.data_ptr())
        return used


def _check_rng(what, rng, device, call):
    _require(isinstance(rng, torch.Tensor) and rng.dtype == torch.int64 and rng.shape == (2,) and rng.is_contiguous() and
             rng.device == device, f"{what}: the generator's state is an int64 tensor [2] (seed, offset) on the inputs' device")
    _require(0 <= call < 65536, f"{what}: call {call} (0 to 65535)")


def act_dropout(x, p, rng=None, call=0, act="none"):
    """dropout(act(x), p) with act "none" | "relu" | "gelu" (erf form), differentiable in x.

    rng: int64 [2] (seed, offset) on x's device, what `DropoutState.draw()` returns; it is read when the kernels run, the
    backward pass included, so its contents stay until then.  call (< 65536) tells the dropouts of one pass apart.  p = 0
    needs no rng, p = 1 gives zeros.  The mask depends on (seed, offset, call, element index) only, not on strides.
    Up to 2^35 - 2048 elements."""
    _check("act_dropout", x)
    _require(act in _lib.PN_ACT, f"act_dropout: activation {act!r}")
    _require(x.dim() >= 1, "act_dropout: a tensor of at least one dimension")
    threshold = dropout_threshold(p)
    if threshold:
        _check_rng("act_dropout", rng, x.device, call)
    else:
        if act == "none":
            return x
        rng, call = None, 0
    return _nodes().act_dropout(x, threshold, rng, call, _lib.PN_ACT[act])


# ---- residual join and norms -------------------------------------------------------------------------------------------
class Norm(namedtuple("Norm", "kind weight bias eps")):
    """kind "layer" | "rms" | "affine" (weight and bias only); weight / bias [C] or None (1 / 0)."""

    def __new__(cls, kind, weight=None, bias=None, eps=1e-5):
        _require(kind in ("layer", "rms", "affine"), f"Norm: kind {kind!r}")
        return super().__new__(cls, kind, weight, bias, float(eps))

    @classmethod
    def of(cls, module):
        """of an nn.LayerNorm / nn.RMSNorm over the last dimension."""
        kind = {torch.nn.LayerNorm: "layer", torch.nn.RMSNorm: "rms"}.get(type(module))
        _require(kind is not None and len(module.normalized_shape) == 1, f"Norm.of: {module}")
        eps = module.eps if module.eps is not None else torch.finfo(torch.float32).eps
        return cls(kind, module.weight, getattr(module, "bias", None), eps)


def residual_norm(x, branch=None, gate=None, scale=1.0, post_norm=None, norm=None, dropout=None, act="none"):
    """h = x + scale * gate * dropout(post_norm(branch)), rounded to x's type; y = act(norm(h)).

    x, branch: [..., C], one type (C up to 16384).  gate: None, [C] (layer scale), x's shape, or one row for each leading
    sample -- [B, C] or [B, 1, C] with x [B, ..., C], B up to 2^23.  post_norm: Norm "layer" / "rms" or None; norm: any Norm or None;
    dropout: (p, rng, call) as act_dropout or None; act ("none" | "relu") on y.  Differentiable in x, branch, gate and the norms'
    weights and biases.  Returns (h, y) with branch and norm, h without a norm, y without a branch (h is then x itself).

    The norm reads h as stored, so y is the norm of the returned h; its gradient is that of what was computed."""
    what = "residual_norm"
    _check(what, *[t for t in (x, branch, gate) if t is not None])
    _require(x.dim() >= 1 and 1 <= x.shape[-1] <= _lib.PN_NORM_MAX_COLS, f"{what}: rows of 1 to {_lib.PN_NORM_MAX_COLS} elements")
    C = x.shape[-1]
    _require(branch is not None or norm is not None, f"{what}: neither a branch nor a norm")
    _require(branch is not None or (gate is None and post_norm is None and dropout is None and scale == 1.0),
             f"{what}: gate, scale, post norm and dropout act on a branch")
    _require(branch is None or (branch.shape == x.shape and branch.dtype == x.dtype),
             f"{what}: the branch has another shape or type than x")
    _require(act in ("none", "relu") and (act == "none" or norm is not None), f"{what}: activation {act!r}")
    _require(post_norm is None or post_norm.kind != "affine", f"{what}: the post norm is layer or rms")
    pw, pb = (post_norm.weight, post_norm.bias) if post_norm is not None else (None, None)
    w, b = (norm.weight, norm.bias) if norm is not None else (None, None)
    for t in (pw, pb, w, b):
        if t is not None:
            _check(what, x, t)
            _require(t.shape == (C,), f"{what}: weights and biases have shape [{C}]")
    R = x.numel() // C
    rows_per_gate = max(R, 1)
    if gate is not None:
        if gate.shape == (C,):
            pass
        elif gate.shape == x.shape:
            rows_per_gate = 1
        else:
            _require(x.dim() >= 2 and gate.shape[0] == x.shape[0] and gate.shape[-1] == C and gate.numel() == x.shape[0] * C,
                     f"{what}: a gate of shape {tuple(gate.shape)} for {tuple(x.shape)}")
            rows_per_gate = max(R // max(x.shape[0], 1), 1)
    threshold, rng, call = 0, None, 0
    if dropout is not None:
        p, rng, call = dropout
        threshold = dropout_threshold(p)
        if threshold:
            _check_rng(what, rng, x.device, call)
        else:
            rng, call = None, 0
    first = None
    for t in (gate, pw, pb, w, b):
        if t is not None and (first is not None and t.dtype != first or t.dtype != torch.float32 and x.dtype == torch.float32
                              or not t.is_contiguous()):
            # the kernels read dense parameters of one type, of fp32 where the rows are
            same = x.dtype == torch.bfloat16 and len({q.dtype for q in (gate, pw, pb, w, b) if q is not None}) == 1
            gate, pw, pb, w, b = [None if q is None else (q if same else q.float()).contiguous() for q in (gate, pw, pb, w, b)]
            break
        first = first if t is None else t.dtype
    out = _nodes().residual_norm(
        x, branch, gate, pw, pb, w, b, rng, _lib.PN_NORM[post_norm.kind] if post_norm is not None else 0,
        _lib.PN_NORM[norm.kind] if norm is not None else 0, post_norm.eps if post_norm is not None else 0.0,
        norm.eps if norm is not None else 0.0, scale, threshold, call, _lib.PN_ACT[act], R, rows_per_gate)
    return out[0] if len(out) == 1 else tuple(out)


# ---- products in fp8 ---------------------------------------------------------------------------------------------------
class Fp8Rows:
    """[rows, cols] in e4m3 with block scales, laid out for products along cols (the layout: pn_fp8_quantize)."""
    __slots__ = ("data", "rows", "cols")

    def __init__(self, rows, cols, device):
        self.rows, self.cols = rows, cols
        self.data = torch.empty(_lib.lib().pn_fp8_operand_bytes(rows, cols), dtype=torch.uint8, device=device)

    def _parts(self):
        """(bytes [groups, blocks, plane, quarter, row, 16], scale bytes [words, rows, 4]) as views."""
        g, b = -(-self.rows // 16), -(-self.cols // 128)
        n = g * b * 2048
        return (self.data[:n].view(g, b, 2, 4, 16, 16), self.data[n: n + -(-b // 4) * self.rows * 4].view(-1, self.rows, 4))

    def bytes_and_exponents(self):
        """(uint8 [rows, cols rounded up to 128], int32 [rows, blocks]): e4m3 bytes, and the exponent of each block."""
        q, s = self._parts()
        g, b = q.shape[:2]
        rows = q.permute(0, 4, 1, 3, 2, 5).reshape(g * 16, b * 128)[: self.rows]
        return rows, s.permute(1, 0, 2).reshape(self.rows, -1)[:, :b].to(torch.int32) - 127

    def values(self):
        """What the bytes stand for, fp32 [rows, cols] (for tests and inspection)."""
        q, e = self.bytes_and_exponents()
        s = ((e + 127) << 23).view(torch.float32).repeat_interleave(128, 1)
        return (q.view(torch.float8_e4m3fn).float() * s)[:, : self.cols]


def fp8_quantize(x, block_rows=1, rows=True, transposed=False):
    """x [..., C] -> (Fp8Rows of x or None, Fp8Rows of its transpose or None), in one pass.  block_rows 1: a scale for each 128
    elements along the contraction (the row, or the column for the transpose); 128: one for each 128 x 128 tile (weights)."""
    _check("fp8_quantize", x)
    _require(x.dim() >= 1 and x.shape[-1] >= 1, "fp8_quantize: empty rows")
    _require(block_rows in (1, 128), f"fp8_quantize: blocks of {block_rows} rows (1 or 128)")
    _require(rows or transposed, "fp8_quantize: nothing asked for")
    v = _rows(x.detach())
    M, C = v.shape
    _require(M > 0 or not transposed, "fp8_quantize: no rows to transpose")
    q = Fp8Rows(M, C, x.device) if rows else None
    qt = Fp8Rows(C, M, x.device) if transposed else None
    _call("pn_fp8_quantize", x.device, _DTYPES[x.dtype], v.data_ptr(), M, C, v.stride(0), block_rows, q and q.data.data_ptr(),
          qt and qt.data.data_ptr(), None)
    return q, qt


def _bias_of(what, bias, n, device):
    if bias is None:
        return None, 0
    _check(what, bias)
    _require(bias.shape == (n,) and bias.device == device, f"{what}: the bias has shape [{n}] and lives with the weight")
    return bias.detach().contiguous(), _DTYPES[bias.dtype]


def fp8_matmul(x, w, bias=None, act="none", out_dtype=torch.bfloat16):
    """x, w: Fp8Rows with the same contraction -> act(x @ w.T + bias) [x.rows, w.rows]."""
    _require(isinstance(x, Fp8Rows) and isinstance(w, Fp8Rows) and x.cols == w.cols, "fp8_matmul: two Fp8Rows with one contraction")
    _require(out_dtype in _DTYPES and act in _lib.PN_ACT, f"fp8_matmul: output {out_dtype}, activation {act!r}")
    dev = x.data.device
    _require(dev == w.data.device, f"fp8_matmul: operands on {dev} and {w.data.device}")
    bias, bd = _bias_of("fp8_matmul", bias, w.rows, dev)
    out = torch.empty((x.rows, w.rows), dtype=out_dtype, device=dev)
    _call("pn_fp8_gemm", dev, x.data.data_ptr(), x.rows, w.data.data_ptr(), w.rows, x.cols, _ptr(bias), bd, _lib.PN_ACT[act],
          _DTYPES[out_dtype], out.data_ptr(), w.rows)
    return out


def _scale_bytes(exponents):
    """Exponents of any integer type -> scale bytes e + 127; clamped before the sum, which a narrow type cannot hold."""
    return (exponents.long().clamp(-126, 127) + 127).to(torch.uint8)


class Fp8Weight:
    """A layer's weight [N, K] laid out once for fp8_linear: e4m3 bytes, one scale for each 128 x 128 tile."""

    def __init__(self, weight, bias=None):
        _check("Fp8Weight", weight)
        _require(weight.dim() == 2 and min(weight.shape) >= 1, "Fp8Weight: a weight [out_features, in_features]")
        self._set(fp8_quantize(weight, 128)[0], bias)

    def _set(self, data, bias):
        self.data, self.out_features, self.in_features = data, data.rows, data.cols
        self.bias, self.bias_dtype = _bias_of("Fp8Weight", bias, data.rows, data.data.device)

    @classmethod
    def from_blocks(cls, values, exponents, bias=None):
        """values: float8_e4m3fn [N, K]; exponents: integers [ceil(N / 128), ceil(K / 128)], the weight of tile (i, j) being
        values * 2^exponents[i, j] (-126 to 127; what lies beyond is taken to the nearer end)."""
        _require(values.device.type == "cuda" and exponents.device == values.device,
                 "Fp8Weight: tensors must live on the GPU (no CPU fallback)")
        _require(values.dtype == torch.float8_e4m3fn and values.dim() == 2 and min(values.shape) >= 1,
                 "Fp8Weight: values are float8_e4m3fn [out_features, in_features]")
        N, K = values.shape
        nb, kb = -(-N // 128), -(-K // 128)
        _require(exponents.shape == (nb, kb) and not exponents.is_floating_point(), f"Fp8Weight: exponents are integers [{nb}, {kb}]")
        self, data = cls.__new__(cls), Fp8Rows(N, K, values.device)
        q, s = data._parts()
        pad = torch.nn.functional.pad(values.view(torch.uint8), (0, kb * 128 - K, 0, q.shape[0] * 16 - N))
        q.copy_(pad.view(q.shape[0], 16, kb, 4, 2, 16).permute(0, 2, 4, 3, 1, 5))
        e = torch.nn.functional.pad(_scale_bytes(exponents), (0, s.shape[0] * 4 - kb))
        s.copy_(e.repeat_interleave(128, 0)[:N].view(N, -1, 4).permute(1, 0, 2))
        self._set(data, bias)
        return self


def fp8_linear(x, weight, act="none", out_dtype=None):
    """act(x @ W.T + bias) [..., N] for x [..., K] and an Fp8Weight: x is laid out in blocks of 1 x 128 on the way.
    out_dtype: fp32 or bf16 (default: x's).  Forward only; fp8_linear_train is the form with gradients."""
    _check("fp8_linear", x)
    _require(isinstance(weight, Fp8Weight), "fp8_linear: the weight is an Fp8Weight")
    N, K, dev = weight.out_features, weight.in_features, x.device
    _require(x.dim() >= 1 and x.shape[-1] == K, f"fp8_linear: rows of {tuple(x.shape)} for a weight of {K}")
    _require(dev == weight.data.data.device, f"fp8_linear: x on {dev}, the weight on {weight.data.data.device}")
    _require(not _wants_grad(x), "fp8_linear: forward only (fp8_linear_train has gradients)")
    _no_tangent("fp8_linear", x)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _require(out_dtype in _DTYPES and act in _lib.PN_ACT, f"fp8_linear: output {out_dtype}, activation {act!r}")
    v, ldx = _strided(x)
    M = x.numel() // K
    out = torch.empty((*x.shape[:-1], N), dtype=out_dtype, device=dev)
    size = _lib.lib().pn_fp8_linear_workspace_bytes(M, N, K)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _call("pn_fp8_linear", dev, _DTYPES[x.dtype], v.data_ptr(), M, ldx, weight.data.data.data_ptr(), N, K, _ptr(weight.bias),
          weight.bias_dtype, _lib.PN_ACT[act], _DTYPES[out_dtype], out.data_ptr(), N, _ptr(ws), size)
    return out


def fp8_linear_train(x, weight, bias=None):
    """x @ weight.T + bias for x [..., K], weight [N, K] (fp32 or bf16 master weight), with every product in fp8:
      y = Q(x) Qw(weight)^T + bias,  dx = Q(g) Qw(weight),  dweight = Q(g^T) Q(x^T)^T,  dbias = column sums of g (fp32 sums of g
    itself), where Q rounds in blocks of 1 x 128 along the product's contraction and Qw in 128 x 128 tiles; the rounding's own
    derivative is taken as one.  dweight and dbias come in the parameters' types."""
    _check("fp8_linear_train", *[t for t in (x, weight, bias) if t is not None])
    _require(x.dim() >= 1 and weight.dim() == 2 and min(weight.shape) >= 1 and x.shape[-1] == weight.shape[1],
             f"fp8_linear_train: x {tuple(x.shape)} for a weight {tuple(weight.shape)}")
    _require(bias is None or bias.shape == (weight.shape[0],), f"fp8_linear_train: the bias has shape [{weight.shape[0]}]")
    _require(max(x.numel() // x.shape[-1], *weight.shape) <= 1 << 22, "fp8_linear_train: more than 2^22 rows or features")
    return _nodes().fp8_linear_train(x, weight, bias)
