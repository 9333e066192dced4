"""Feed-forward operators without a GPU: the generator's published test vectors, the oracle's rounding against torch's own
e4m3 conversion, and what the entry points refuse (Python and C ABI)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import ffn_oracle as fo
from pillarnet_lts_amd import _lib, ffn_ops
from pillarnet_lts_amd._lib import PillarnetHipError


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))])
def test_generator_matches_its_published_vectors(counter, key, want):
    got = fo.philox4x32([np.array([c], dtype=np.uint64) for c in counter], key)
    assert tuple(int(v[0]) for v in got) == want


def test_oracle_rounding_equals_the_types_own():
    x = np.concatenate([np.linspace(-460, 460, 40001), 2.0 ** np.arange(-14, 9), -(2.0 ** np.arange(-14, 9)) * 1.0625])
    x = x.astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    inside = np.abs(x) <= 448
    np.testing.assert_array_equal(fo.round_e4m3(x)[inside], want[inside])
    assert np.isnan(fo.round_e4m3(np.array([np.inf, -np.inf, np.nan, 1e4]))).all()


def test_block_exponent_is_the_smallest_that_holds_the_block():
    v = np.array([[448.0], [448.5], [447.0], [1.75], [1.7500001], [0.0], [2.0 ** -140], [3e38]]).astype(np.float32)
    e = fo.block_exponents(v.astype(np.float64), 1)[:, 0]
    assert list(e[:3]) == [0, 1, 0] and list(e[3:5]) == [-8, -7] and list(e[5:7]) == [-126, -126]
    assert (np.abs(v[:, 0]) <= 448 * np.exp2(e.astype(np.float64))).all()


def test_threshold_keeps_its_range():
    t = ffn_ops.dropout_threshold
    assert (t(0.0), t(1.0), t(0.5), t(1e-9), t(1 - 1e-9)) == (0, 65536, 32768, 1, 65535)
    for p in (0.0, 1e-9, 0.1, 0.3, 0.5, 1 - 1e-9, 1.0):
        assert t(p) == fo.threshold(p)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(PillarnetHipError):
            t(p)


def test_host_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(8)
    for call in (lambda: ffn_ops.act_dropout(x, 0.5, torch.zeros(2, dtype=torch.int64)),
                 lambda: ffn_ops.residual_norm(x, x, norm=ffn_ops.Norm("layer", w, w)),
                 lambda: ffn_ops.fp8_quantize(x), lambda: ffn_ops.Fp8Weight(x),
                 lambda: ffn_ops.Fp8Weight.from_blocks(x.to(torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.int32)),
                 lambda: ffn_ops.fp8_linear_train(x, x), lambda: ffn_ops.DropoutState(1, "cpu")):
        with pytest.raises(PillarnetHipError, match="GPU"):
            call()
    with pytest.raises(PillarnetHipError):
        ffn_ops.Norm("group", w, w)


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_scale_bytes_of_any_integer_type_clamp_to_the_nearer_end(dtype):
    lim = torch.iinfo(dtype)
    e = sorted({lim.min, lim.max, 0, 1, 5, 126, 127, *((-127, -126, -125, -1) if lim.min < 0 else (128, 200))})
    got = ffn_ops._scale_bytes(torch.tensor([e], dtype=dtype))
    assert got.dtype == torch.uint8 and got[0].tolist() == [max(-126, min(127, v)) + 127 for v in e]


def test_forward_mode_tangents_are_refused():
    """neither the nodes nor a kernel called beside them drop a tangent in silence (empty tensors launch nothing)."""
    fw, n = torch.autograd.forward_ad, _lib.autograd()
    e, w = torch.zeros(0, 8), torch.zeros(8)
    join = lambda x, f=None, gate=None, w=None: n.residual_norm(x, f, gate, None, None, w, None, None, 0, 1, 0.0, 1e-5, 1.0, 0, 0, 0, 0, 1)
    with fw.dual_level():
        d, dw = fw.make_dual(e, torch.ones(0, 8)), fw.make_dual(w, torch.ones(8))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: n.act_dropout(d, 0, None, 0, 2), lambda: join(d), lambda: join(e, d), lambda: join(e, e, dw),
                             lambda: join(e, w=dw), lambda: n.fp8_linear_train(d, torch.zeros(4, 8), None),
                             lambda: n.fp8_linear_train(e, torch.zeros(8, 8), dw), lambda: ffn_ops._no_tangent("fp8_linear", d)):
                    with pytest.raises(PillarnetHipError, match="no forward-mode derivative"):
                        call()
                assert n.act_dropout(e, 0, None, 0, 2).shape == join(e)[0].shape == (0, 8)      # others go on as ever
                ffn_ops._no_tangent("fp8_linear", e)
    ffn_ops._no_tangent("fp8_linear", d)


def _join(**kw):
    d = dict(dtype=0, param_dtype=0, post_kind=0, norm_kind=1, act=0, cols=8, rows=4, rows_per_gate=4, ldx=8, ldb=8, scale=1.0,
             post_eps=1e-5, norm_eps=1e-5, threshold=0, call=0, x=16, branch=16)
    d.update(kw)
    return _lib.pnResidualNorm(**d)


@pytest.mark.parametrize("bad", [
    dict(dtype=2), dict(param_dtype=7), dict(param_dtype=1), dict(cols=0), dict(cols=16385), dict(rows=-1), dict(post_kind=3), dict(norm_kind=4),
    dict(act=2), dict(branch=None, gate=16), dict(branch=None, post_kind=1), dict(branch=None, threshold=5, rng=16),
    dict(branch=None, norm_kind=0), dict(threshold=65537, rng=16), dict(threshold=1), dict(call=65536), dict(x=None),
    dict(ldx=7), dict(ldb=7), dict(gate=16, rows_per_gate=3), dict(gate=16, rows_per_gate=0),
    dict(gate=16, rows_per_gate=2, rows=(1 << 24) + 2)])
def test_residual_norm_arguments_are_checked_before_the_gpu(bad):
    L = _lib.lib()
    s = _join(**bad)
    assert L.pn_residual_norm_forward(ctypes.byref(s), 16, 16, None, None) == -1 and L.pn_last_error()
    assert L.pn_residual_norm_backward(ctypes.byref(s), 16, 16, 16, 16, 16, None, None, None, None, None, None, 16, 1 << 20, None) == -1
    assert L.pn_residual_norm_workspace_bytes(ctypes.byref(s)) == 0


def test_residual_norm_outputs_and_workspace_are_checked():
    L = _lib.lib()
    s = _join()
    p = ctypes.byref(s)
    assert L.pn_residual_norm_forward(None, 16, 16, None, None) == -1
    assert L.pn_residual_norm_forward(p, None, 16, None, None) == -1 and L.pn_residual_norm_forward(p, 16, None, None, None) == -1
    assert L.pn_residual_norm_forward(p, 16, 16, 20, None) == -1                       # statistics off their alignment
    back = lambda h=16, st=16, gh=16, gy=16, df=None, dg=None, ws=16, n=1 << 20, q=p: L.pn_residual_norm_backward(
        q, h, st, gh, gy, 16, df, None, None, None, None, dg, ws, n, None)
    assert back(gh=None, gy=None) == -1 and back(h=None) == -1 and back(st=None) == -1
    assert back(df=16) == -1                                                            # the branch's gradient is dx here
    assert back(dg=16) == -1
    assert back(n=8) == -2 and b"workspace" in L.pn_last_error() and back(ws=None) == -2
    assert L.pn_residual_norm_workspace_bytes(p) >= 2 * 8 * 4
    none = _join(rows=0)
    assert L.pn_residual_norm_forward(ctypes.byref(none), None, None, None, None) == 0  # nothing to do, nothing launched


def test_dropout_and_fp8_arguments_are_checked_before_the_gpu():
    L = _lib.lib()
    fwd = lambda dt=0, x=16, r=2, c=8, ld=8, act=0, t=5, rng=16, call=0, y=16: L.pn_act_dropout_forward(
        dt, x, r, c, ld, act, t, rng, call, y, None)
    for bad in (dict(dt=3), dict(x=None), dict(r=-1), dict(ld=7), dict(act=3), dict(t=65537), dict(rng=None), dict(call=65536),
                dict(y=None), dict(r=1 << 40, c=1 << 10)):
        assert fwd(**bad) == -1 and L.pn_last_error()
    assert fwd(r=0, x=None, y=None) == 0
    assert L.pn_act_dropout_backward(0, 16, None, 2, 8, 8, 8, 2, 5, 16, 0, 16, None) == -1      # gelu needs x
    assert L.pn_act_dropout_backward(0, None, 16, 2, 8, 8, 8, 1, 5, 16, 0, 16, None) == -1
    assert L.pn_dropout_draw(None, 16, None) == -1
    q = lambda dt=0, x=16, r=4, c=8, ld=8, b=1, q=256, t=None: L.pn_fp8_quantize(dt, x, r, c, ld, b, q, t, None, None)
    for bad in (dict(dt=2), dict(x=None), dict(r=-1), dict(c=0), dict(ld=7), dict(b=64), dict(q=None), dict(q=24), dict(t=16)):
        assert q(**bad) == -1
    assert q(r=0) == 0
    g = lambda x=256, m=4, w=256, n=8, k=8, act=0, od=0, out=16, ldo=8: L.pn_fp8_gemm(x, m, w, n, k, None, 0, act, od, out, ldo, None)
    for bad in (dict(x=None), dict(m=-1), dict(w=None), dict(n=0), dict(k=0), dict(act=3), dict(od=2), dict(out=None), dict(ldo=7),
                dict(x=24), dict(w=16), dict(k=(1 << 22) + 1)):
        assert g(**bad) == -1
    assert g(m=0) == 0
    f = lambda dt=0, x=16, m=5000, ld=256, w=256, n=256, k=256, ws=256, nb=1 << 30: L.pn_fp8_linear(dt, x, m, ld, w, n, k, None, 0, 0, 0, 16, n,
                                                                                                  ws, nb, None)
    assert L.pn_fp8_linear_workspace_bytes(5000, 256, 256) == L.pn_fp8_operand_bytes(5000, 256) > 5000 * 256
    assert L.pn_fp8_linear_workspace_bytes(16, 256, 256) == 0 == L.pn_fp8_operand_bytes(-1, 8)
    for bad in (dict(dt=4), dict(x=None), dict(ld=255), dict(w=None), dict(ws=8)):
        assert f(**bad) == -1
    assert f(ws=None) == -2 and f(nb=100) == -2
    tf = lambda dt=0, x=16, m=4, ld=8, wd=0, w=16, n=8, k=8, lw=8, y=16, sv=256, ws=256: L.pn_fp8_train_forward(
        dt, x, m, ld, wd, w, n, k, lw, None, 0, y, 1, 1, sv, ws, None)
    for bad in (dict(dt=2), dict(wd=3), dict(x=None), dict(m=0), dict(ld=7), dict(lw=7), dict(w=None), dict(y=None), dict(sv=None), dict(ws=8),
                dict(k=1 << 23)):
        assert tf(**bad) == -1
    tb = lambda dt=0, g=16, m=4, ld=8, wd=0, sv=256, dx=None, db=None, bd=0, ws=256: L.pn_fp8_train_backward(
        dt, g, m, ld, wd, 8, 8, sv, dx, None, db, bd, ws, None)
    for bad in (dict(dt=2), dict(g=None), dict(m=0), dict(ld=7), dict(sv=16), dict(ws=None), dict(db=16, bd=7)):
        assert tb(**bad) == -1
    assert tb() == 0                                                            # nothing asked for, nothing launched
    assert L.pn_fp8_train_saved_bytes(0, 8, 8) == 0 and L.pn_fp8_train_workspace_bytes(4, 8, 8, 1) >= 4 * 8


def test_more_elements_than_a_launch_takes_are_refused():
    """a launch holds less than 2^32 threads along a dimension: 256 a workgroup here, for 2048 elements."""
    L = _lib.lib()
    for rows, cols in (((1 << 35) - 2047, 1), (1, (1 << 35) - 2047), (1 << 20, 1 << 15), (1 << 24, 1 << 17)):
        for rc in (L.pn_act_dropout_forward(1, 16, rows, cols, cols, 0, 5, 16, 0, 16, None),
                   L.pn_act_dropout_backward(1, 16, None, rows, cols, cols, cols, 0, 5, 16, 0, 16, None)):
            assert rc == -1 and b"more than one launch takes" in L.pn_last_error()
    for rows, cols in (((1 << 31) - 127, 1), (1 << 27, 2048), (128, (1 << 31) - 127)):        # 2^24 tiles of 128 x 128
        assert L.pn_fp8_quantize(1, 16, rows, cols, cols, 1, None, 256, None, None) == -1
        assert b"more than one launch takes" in L.pn_last_error()


def test_product_cases_take_every_kernel():
    """the sizes that products are tested at on the GPU reach every kernel, also after the rules by size have moved."""
    import fp8_product_cases as pc
    L = _lib.lib()
    for (m, k, n), out, laid, kind, rest in pc.CASES:
        got = L.pn_fp8_kernels(m, n, k, out, laid)
        assert (got & 15, got >> 4) == (kind, rest), ((m, k, n), out, laid, got)
    for (m, k, n), dtype, kinds in pc.TRAIN:
        assert tuple(L.pn_fp8_kernels(*q, 1) for q in pc.products(m, k, n, dtype)) == kinds
    taken = {(out, laid or kind not in (pc.D32, pc.D64), kind) for _, out, laid, kind, _ in pc.CASES}
    assert taken >= {(o, True, kind) for o in (pc.F32, pc.BF16) for kind in (pc.D32, pc.D64, pc.T64, pc.T128, pc.PAIR)}
    assert taken >= {(o, False, kind) for o in (pc.F32, pc.BF16) for kind in (pc.D32, pc.D64)}
    assert {(out, rest) for _, out, _, _, rest in pc.CASES} >= {(o, r) for o in (pc.F32, pc.BF16) for r in (pc.D32, pc.D64, pc.T64)}
    for bad in ((0, 1, 1, 0), (1, 0, 1, 0), (1, 1, 0, 0), (1, 1, 1, 7)):
        assert L.pn_fp8_kernels(*bad, 1) == -1


def test_struct_layout_matches_header():
    assert ctypes.sizeof(_lib.pnResidualNorm) == 6 * 4 + 4 * 8 + 5 * 4 + 4 + 8 * 8      # 4 bytes of padding before the pointers


def test_fp8_plans_follow_replaced_storages():
    """a plan is made anew when a parameter or a buffer gets another storage, also one that a freed storage's address went to."""
    from pillarnet_lts_amd import second_stage
    m = torch.nn.Sequential(torch.nn.Linear(512, 512), torch.nn.BatchNorm1d(512))
    plan = lambda: second_stage.FP8_PLANS.get(m, lambda m: object())
    a = plan()
    assert plan() is a
    m[1].running_mean = torch.ones(512)
    b = plan()
    assert b is not a and plan() is b
    for _ in range(8):
        before = plan()
        m[0].weight.data = torch.zeros(1)
        m[0].weight.data = torch.ones(512, 512)         # where the allocator finds a megabyte: the place just freed, as a rule
        assert plan() is not before
    m[1].running_var.add_(1)
    assert plan() is not before


def test_fp8_plans_go_with_their_modules():
    import gc
    import weakref
    from pillarnet_lts_amd import second_stage
    m = torch.nn.Linear(8, 8)
    for k in range(3):
        m.weight.data = torch.full((8, 8), float(k))
        second_stage.FP8_PLANS.get(m, lambda m: object())
    key, gone = id(m), weakref.ref(m)
    assert key in second_stage.FP8_PLANS._d
    del m
    gc.collect()
    assert gone() is None and key not in second_stage.FP8_PLANS._d


def test_a_head_without_a_fused_path_says_so():
    from pillarnet_lts_amd import legacy
    head = legacy.RoIHead(16, dict(SHARED_FC=[8], CLS_FC=[8], REG_FC=[8], DP_RATIO=0.0))
    for kw in (dict(), dict(fused_ops=False, fp8=True)):
        with pytest.raises(PillarnetHipError, match="RoIHead has no fused path"):
            head.use_fused(**kw)
    assert head.use_fused(False) is head and not head.fused_ops


def test_to_inference_refuses_a_head_without_fp8_before_it_converts():
    from types import SimpleNamespace
    from pillarnet_lts_amd import legacy, second_stage
    converted = []
    stage = SimpleNamespace(to_inference=lambda *a: converted.append(a))
    head = legacy.RoIHead(16, dict(SHARED_FC=[8], CLS_FC=[8], REG_FC=[8], DP_RATIO=0.0))
    with pytest.raises(PillarnetHipError, match="no fused path"):
        second_stage.PillarRCNN.to_inference(SimpleNamespace(single_det=stage, roi_head=head), roi_fp8=True)
    assert not converted
