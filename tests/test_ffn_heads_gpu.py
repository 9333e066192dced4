"""The RoI heads on the feed-forward operators (RoIHeadTemplate.use_fused): against the reference-generated fixtures and the
heads' own torch modules in fp32, their training passes, and the two-stage detector in fp8."""
import copy
import os

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from pillarnet_lts_amd import ffn_ops, second_stage
from pillarnet_lts_amd.config import ConfigDict

pytestmark = pytest.mark.gpu
G = os.path.join(os.path.dirname(__file__), "golden")
CFG = dict(CLASS_AGNOSTIC=True, SHARED_FC=[32, 32], CLS_FC=[32, 32], REG_FC=[32, 32], DP_RATIO=0.3,
           TARGET_CONFIG=dict(ROI_PER_IMAGE=32, FG_RATIO=0.5, SAMPLE_ROI_BY_EACH_CLASS=True, CLS_SCORE_TYPE="roi_iou",
                              CLS_FG_THRESH=0.7, CLS_BG_THRESH=0.25, CLS_BG_THRESH_LO=0.1, HARD_BG_RATIO=0.8, REG_FG_THRESH=0.5),
           LOSS_CONFIG=dict(CLS_LOSS="BinaryCrossEntropy", REG_LOSS="L1", IOU_LOSS="L1",
                            LOSS_WEIGHTS=dict(rcnn_cls_weight=1.0, rcnn_reg_weight=1.0, rcnn_iou_weight=0.7, code_weights=[1.0] * 7)))


def _ffn_head(g, cuda, **kw):
    head = second_stage.RoIFFNHead(model_cfg=ConfigDict(CFG), feedforward_channels=48, content_dim=32, num_class=1, code_size=7, **kw)
    head.load_state_dict({k[len("sd.ffn."):]: torch.from_numpy(g[k]) for k in g.files if k.startswith("sd.ffn.")}, strict=True)
    return head.to(cuda)


def test_ffn_head_fused_matches_reference_outputs(cuda):
    """the same bars as the torch modules: inference 1e-5, training losses and gradients 1e-4 (fp32 sums in another order)."""
    g, t = np.load(os.path.join(G, "rcnn_extra.npz")), np.load(os.path.join(G, "rcnn_train.npz"))
    head = _ffn_head(g, cuda, fused_ops=True).eval()
    tt = lambda a, k: torch.from_numpy(a[k]).to(cuda)
    B = g["bevf.in.rois"].shape[0]
    with torch.no_grad():
        out = head(dict(batch_size=B, rois=tt(g, "bevf.in.rois"), roi_features=tt(g, "ffn.in.roi_features"),
                        roi_scores=tt(g, "ffn.in.roi_scores"), roi_labels=tt(g, "ffn.in.roi_labels")), training=False)
    np.testing.assert_allclose(out["batch_cls_preds"].cpu().numpy(), g["ffn.out.batch_cls_preds"], rtol=1e-5, atol=2e-6)
    np.testing.assert_allclose(out["batch_box_preds"].cpu().numpy(), g["ffn.out.batch_box_preds"], rtol=1e-5, atol=5e-6)
    head.train()
    td = {k: tt(t, "pt." + k) for k in ("rois", "gt_of_rois", "gt_of_rois_src", "roi_scores", "roi_labels", "reg_valid_mask",
                                        "rcnn_cls_labels")}
    head(dict(batch_size=2, rois=td["rois"], roi_labels=td["roi_labels"], roi_scores=td["roi_scores"], roi_targets_dict=td,
              roi_features=tt(g, "ffn.train.in.roi_features")), training=True)
    loss, _ = head.get_loss()
    np.testing.assert_allclose(float(loss.detach()), float(g["ffn.train.loss"]), rtol=1e-4)
    loss.backward()
    np.testing.assert_allclose(head.fc_iou.weight.grad.cpu().numpy(), g["ffn.train.grad.fc_iou.weight"], rtol=1e-3, atol=1e-5)
    np.testing.assert_allclose(head.ffn.layers[0][0].weight.grad.cpu().numpy(), g["ffn.train.grad.ffn.layers.0.0.weight"], rtol=1e-3,
                               atol=1e-5)


@pytest.mark.parametrize("mixer", ["MLPMixer", "ResMLP"])
def test_mixers_fused_match_their_modules(cuda, mixer):
    torch.manual_seed(0)
    head = second_stage.RoIMIXHead(in_channels=64, model_cfg=ConfigDict(CFG), mixer_type=mixer, num_patches=49).to(cuda)
    m = head.mlp_mixer
    with torch.no_grad():
        for p in m.parameters():
            p.add_(torch.randn_like(p) * 0.1)
    head.use_fused(True)
    x = torch.randn(37, 49, 64, device=cuda, requires_grad=True)
    y = head._mix(x)
    want = m(x)
    g = torch.randn_like(y)
    a = torch.autograd.grad(y, [x, *m.parameters()], g)
    b = torch.autograd.grad(want, [x, *m.parameters()], g)
    # two fp32 evaluations of the same expression, torch's GEMMs among both: 1e-5 of each tensor's norm
    for p, q in zip([y, *a], [want, *b]):
        assert (p - q).norm() <= 1e-5 * q.norm()


def _mix_head(cuda, **kw):
    torch.manual_seed(1)
    head = second_stage.RoIMIXHead(in_channels=16, model_cfg=ConfigDict(CFG), mixer_type="MLPMixer", num_patches=49, **kw).to(cuda)
    gen = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=gen).to(cuda)
    batch = dict(batch_size=2, rois=r(2, 32, 7).abs() + 0.5, roi_features=r(2, 32, 49 * 16), roi_scores=r(2, 32).sigmoid(),
                 roi_labels=torch.ones(2, 32, dtype=torch.long, device=cuda))
    td = dict(rois=batch["rois"], roi_scores=batch["roi_scores"], roi_labels=batch["roi_labels"], gt_of_rois=r(2, 32, 8),
              reg_valid_mask=torch.ones(2, 32, dtype=torch.long, device=cuda), rcnn_cls_labels=r(2, 32).sigmoid())
    return head, batch, td


@pytest.mark.parametrize("fp8", [False, True])
def test_mix_head_trains_with_dropout(cuda, fp8):
    """a seed gives one sequence of masks; every parameter gets a finite gradient; evaluation drops nothing."""
    grads = []
    for _ in range(2):
        head, batch, td = _mix_head(cuda, fused_ops=True, fp8=fp8, dropout_seed=11)
        head.train()
        passes = []
        for _ in range(2):
            head.zero_grad()
            head(dict(batch, roi_targets_dict=dict(td)), training=True)
            loss, _ = head.get_loss()
            loss.backward()
            assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in head.parameters())
            passes.append(torch.cat([p.grad.flatten() for p in head.parameters()]))
        assert not torch.equal(passes[0], passes[1])                # the second pass draws other masks
        grads.append(passes)
        assert head._dropout_state.state.tolist() == [11, 2]
    for a, b in zip(*grads):
        assert (a - b).norm() <= 1e-5 * b.norm()                    # (torch's own reductions in BatchNorm's backward may differ)
    head.eval()
    with torch.no_grad():
        a = head(dict(batch), training=False)["batch_cls_preds"]
        assert torch.equal(a, head(dict(batch), training=False)["batch_cls_preds"])


def test_ffn_head_dropout_and_fp8_layers(cuda):
    """RoIFFNHead with dropout: the fused pass equals torch expressions on the same masks; in fp8 each layer is the product of what
    its operands were rounded to."""
    torch.manual_seed(3)
    x = torch.randn(70, 32, device=cuda)
    head = second_stage.RoIFFNHead(model_cfg=ConfigDict(CFG), feedforward_channels=160, content_dim=32, dropout=0.25, dropout_seed=5,
                                   fused_ops=True).to(cuda).train()
    q = head._query_fused(x)
    rng = torch.tensor([5, 0], dtype=torch.int64, device=cuda)
    fc1, fc2 = head.ffn.layers[0][0], head.ffn.layers[1]
    mask = lambda shape, call: ffn_ops.act_dropout(torch.ones(shape, device=cuda), 0.25, rng, call)
    want = head.ffn_norm(x + fc2(fc1(x).relu() * mask((70, 160), 0)) * mask((70, 32), 1))
    assert (q - want).norm() <= 1e-5 * want.norm()
    head.use_fused(fp8=True).eval()
    with torch.no_grad():
        y = head.fused_linear(fc1, x, "relu")
        rounded = lambda t, b: ffn_ops.fp8_quantize(t, b)[0].values()
        want = (rounded(x, 1) @ rounded(fc1.weight, 128).t() + fc1.bias).relu()
        assert (y - want).norm() <= 1e-6 * want.norm()
        old = head.fused_linear(fc1, x)
        fc1.weight.add_(0.25)                                        # a changed weight is laid out anew
        assert not torch.equal(old, head.fused_linear(fc1, x))


def test_fp8_evaluation_with_gradients_enabled(cuda):
    """a folded stack in fp8 gives its rows' gradient, dx = Q(g) Qw(W), and evaluating a head outside of no_grad works as it does
    without fp8."""
    torch.manual_seed(4)
    fc = torch.nn.Linear(96, 40).to(cuda)
    mlp = second_stage.FoldedMLP([fc, torch.nn.ReLU()], fp8=True)
    x, g = torch.randn(70, 96, device=cuda, requires_grad=True), torch.randn(70, 40, device=cuda)
    y = mlp(x)
    dx, = torch.autograd.grad(y, x, g)
    rounded = lambda t, b: ffn_ops.fp8_quantize(t, b)[0].values().double()
    w = rounded(fc.weight, 128)
    # fp32 sums of 96 and 40 products and a bias: K + 2 roundings of 2^-24 of the sum of magnitudes at most
    xq, gq = rounded(x, 1), rounded(g * (y > 0), 1)
    assert ((y - (xq @ w.t() + fc.bias).relu()).abs() <= 200 * 2.0 ** -24 * (xq.abs() @ w.t().abs() + fc.bias.abs())).all()
    assert ((dx - gq @ w).abs() <= 100 * 2.0 ** -24 * (gq.abs() @ w.abs())).all()
    assert not mlp(x.detach()).requires_grad
    head, batch, _ = _mix_head(cuda, fp8=True)
    head.eval()
    feats = batch["roi_features"].clone().requires_grad_()
    out = head(dict(batch, roi_features=feats), training=False)["batch_cls_preds"]
    with torch.no_grad():
        want = head(dict(batch), training=False)["batch_cls_preds"]
    # sums in another order; an input that then falls on the other side of an e4m3 border moves one of some hundred summands of a
    # row by 2^-3 of itself: 1e-2 of the norm has room for many of those
    assert (out - want).norm() <= 1e-2 * want.norm()
    grads = torch.autograd.grad(out.sum(), [feats, *head.mlp_mixer.parameters()])
    assert all(torch.isfinite(q).all() for q in grads) and grads[0].abs().sum() > 0


def test_fp8_plans_follow_replaced_storages(cuda):
    """a weight that moves into a storage at the address that its old one gave back is laid out anew; so is one behind a replaced
    running mean."""
    head = second_stage.RoIHeadTemplate(1, {}).to(cuda).eval()
    head.fp8 = True
    fc, x = torch.nn.Linear(512, 512, bias=False).to(cuda), torch.ones(4, 512, device=cuda)
    with torch.no_grad():
        for k in range(4):
            fc.weight.data = torch.zeros(1, device=cuda)
            fc.weight.data = torch.full((512, 512), 2.0 ** k, device=cuda)
            assert (head.fused_linear(fc, x) == 512 * 2.0 ** k).all(), k
        head, batch, _ = _mix_head(cuda, fp8=True)
        head.eval()
        bn = head.shared_fc_layer[1]
        old = head(dict(batch), training=False)["batch_cls_preds"]
        bn.running_mean = bn.running_mean + 0.5
        assert not torch.equal(old, head(dict(batch), training=False)["batch_cls_preds"])


def test_heads_refuse_host_tensors_when_fused():
    from pillarnet_lts_amd._lib import PillarnetHipError
    head = second_stage.RoIFFNHead(model_cfg=ConfigDict(CFG), feedforward_channels=48, content_dim=32, fused_ops=True)
    with pytest.raises(PillarnetHipError, match="GPU"):
        head._query_fused(torch.zeros(4, 32))


def test_two_stage_detector_with_fp8_head(cuda):
    """PillarRCNN.to_inference(roi_fp8=True): the first stage's detections are what they were, the refined ones move by the rounding;
    eager and in a replayed frame graph alike."""
    from pillarnet_lts_amd import presets, synth
    from pillarnet_lts_amd.frame_graph import FrameGraphs
    from test_rcnn_gpu import small_rcnn
    torch.manual_seed(0)
    model = presets.build(small_rcnn())
    synth.randomize_bn_(model, seed=1)
    plain = copy.deepcopy(model).to_inference(torch.bfloat16)
    model = model.to_inference(torch.bfloat16, roi_fp8=True)
    pts = torch.from_numpy((synth.waymo_frame(6000, seed=3)[:, :5] * np.array([0.17, 0.17, 1, 1, 1], np.float32)).astype(np.float32)).to(cuda)
    ex = dict(points=[pts], metadata=[{}])
    with torch.no_grad():
        a, b = plain(dict(ex), return_loss=False)[0], model(dict(ex), return_loss=False)[0]
    assert a["box3d_lidar"].shape == b["box3d_lidar"].shape and torch.equal(a["label_preds"], b["label_preds"])
    assert torch.isfinite(b["box3d_lidar"]).all() and not torch.equal(a["scores"], b["scores"])
    graphs = FrameGraphs(model, lanes=1)
    for _ in range(3):
        c = graphs.forward_deferred(dict(ex)).result()[0]
        assert torch.equal(c["box3d_lidar"], b["box3d_lidar"]) and torch.equal(c["scores"], b["scores"])
