"""The classifier loss in pieces and the orthogonalised optimiser where the framework's own training uses them."""
import copy
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module")
def job(hip_lib_path):
    from detectron_pytorch_amd.rcnn import config, data, model

    cfg = config.faster_rcnn_r50_fpn()
    torch.manual_seed(cfg.RNG_SEED)
    net = model.GeneralizedRCNN(cfg).to(DEV).train()
    batch = data.to_device(data.synthetic_minibatch(cfg, 2, seed=1, blob_height=256, blob_width=320, image_width=318), DEV)
    return net, cfg, batch


def with_config(net, **changes):
    net = copy.deepcopy(net)
    for section, values in changes.items():
        net.cfg[section].update(values)
    return net


@pytest.mark.parametrize("autocast", [None, torch.bfloat16])
def test_box_head_loss_in_pieces_equals_the_usual_one(job, autocast):
    net, cfg, (data, im_info, roidb, rpn_t) = job
    priority = torch.from_numpy(np.random.RandomState(7).permutation(roidb["gt_boxes"].size(0) + 4000).astype(np.float32)).to(DEV)
    with torch.no_grad():
        blob_conv = net.Conv_Body(data)
        rpn_ret = net.RPN(blob_conv)
        rois = net.proposals(rpn_ret, im_info.to(DEV, torch.float32), static=True)
    blob_conv = [b.detach() for b in blob_conv]
    got = []
    for pieces in (False, True):
        one = with_config(net, FAST_RCNN=dict(CLS_LOSS_IN_PIECES=pieces))
        one.proposals = lambda *a, **k: rois
        pri = priority[:roidb["gt_boxes"].size(0) + rois[0].size(0)]
        if autocast is None:
            ret = one.forward_from_features(blob_conv, rpn_ret, im_info, roidb, rpn_t, pri)
        else:
            with torch.autocast("cuda", dtype=autocast):
                ret = one.forward_from_features(blob_conv, rpn_ret, im_info, roidb, rpn_t, pri)
        (ret["losses"]["loss_cls"] + ret["losses"]["loss_bbox"]).backward()
        got.append((ret, {n: p.grad for n, p in one.named_parameters() if p.grad is not None}))
    (usual, g0), (pieces, g1) = got
    assert torch.equal(usual["blobs"]["labels_int32"], pieces["blobs"]["labels_int32"])
    # the logits' rounding to the autocast type is gone: half a step of logits up to 4 is 2^-7, of gradients 2^-8 a rounding, some ten of them
    tol = 1e-4 if autocast is None else 0.05
    for k in ("loss_cls", "loss_bbox"):
        a, b = usual["losses"][k].detach(), pieces["losses"][k].detach()
        assert abs(float(a) - float(b)) <= tol * max(1.0, abs(float(a)))
    if autocast is None:
        assert float(usual["metrics"]["accuracy_cls"]) == float(pieces["metrics"]["accuracy_cls"])
    assert set(g0) == set(g1) and {"Box_Outs.cls_score.weight", "Box_Outs.cls_score.bias", "Box_Head.fc1.weight"} <= set(g0)
    for n in g0:
        assert float((g0[n] - g1[n]).norm()) <= tol * float(g0[n].norm()) + 1e-9, n


def test_training_steps_with_both(job):
    from detectron_pytorch_amd.muon import Muon
    from detectron_pytorch_amd.rcnn import train as rtrain

    net, cfg, (data, im_info, roidb, rpn_t) = job
    net = with_config(net, FAST_RCNN=dict(CLS_LOSS_IN_PIECES=True), SOLVER=dict(TYPE="MUON"))
    opt = rtrain.make_optimizer(net, net.cfg, lr=1e-4)
    assert isinstance(opt, Muon)
    assert opt.param_groups[0]["lr"] == cfg.SOLVER.MUON.LR and opt.param_groups[1]["sgd_lr"] == 2e-4
    before = {n: p.detach().clone() for n, p in net.named_parameters() if p.requires_grad}
    for _ in range(3):
        ret = rtrain.train_step(net, opt, data, im_info, roidb, rpn_t)
        assert np.isfinite(float(ret["total_loss"]))
    for n, p in net.named_parameters():
        if p.requires_grad:
            assert torch.isfinite(p).all(), n
            assert p.grad is None or not torch.equal(p.detach(), before[n]) or not bool(p.grad.any()), n
    net.cfg.SOLVER.TYPE = "ADAM"
    with pytest.raises(NotImplementedError):
        rtrain.make_optimizer(net, net.cfg)


def test_a_classifier_trained_by_the_operators_follows_the_formulas():
    """Three steps of features -> loss -> gradients -> momentum -> orthogonalised update, all of them in 64 bits on the other side.
    An update's elements are below 1 (its singular values are); the operators' relative errors of 1e-4 of it, three steps and a
    learning rate of 0.02 leave 1e-5 of absolute difference."""
    from detectron_pytorch_amd.linear_cross_entropy import linear_cross_entropy
    from detectron_pytorch_amd.muon import Muon
    from test_orthogonalize_gpu import formula

    gen = torch.Generator(device=DEV)
    gen.manual_seed(5)
    x = torch.randn(300, 48, generator=gen, device=DEV)
    y = torch.randint(-1, 200, (300,), generator=gen, device=DEV)
    weight = torch.nn.Parameter(0.1 * torch.randn(200, 48, generator=gen, device=DEV))
    bias = torch.nn.Parameter(torch.zeros(200, device=DEV))
    w, b = weight.detach().double(), bias.detach().double()
    mw, mb = torch.zeros_like(w), torch.zeros_like(b)
    opt = Muon([weight, bias], lr=0.02, sgd_lr=0.1, weight_decay=0.0)
    keep = y >= 0
    for _ in range(3):
        opt.zero_grad()
        loss = linear_cross_entropy(x, weight, bias, y)
        loss.backward()
        opt.step()
        w.requires_grad_(True), b.requires_grad_(True)
        z = x[keep].double() @ w.t() + b
        want = (torch.logsumexp(z, 1) - z.gather(1, y[keep][:, None])[:, 0]).mean()
        gw, gb = torch.autograd.grad(want, (w, b))
        assert abs(float(loss.detach()) - float(want.detach())) <= 1e-4
        mw, mb = 0.95 * mw + gw, 0.9 * mb + gb
        w = (w.detach() - 0.02 * math.sqrt(200 / 48) * formula(gw + 0.95 * mw))
        b = b.detach() - 0.1 * mb
        assert float((weight.detach().double() - w).abs().max()) <= 1e-5
        assert float((bias.detach().double() - b).abs().max()) <= 1e-5
