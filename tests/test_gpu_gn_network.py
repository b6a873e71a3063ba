"""The network with MODEL.DARKNET.NORM "GN" and the optimizer with SOLVER.CLIP_GRADIENTS: inference, training step, update.

Bars for whole fp32 networks are the ones the BatchNorm network is held to (heads within 1e-3 of their largest value, losses within 1e-3,
gradients cos > 0.998 and 6 % in the 2-norm); single layers go by the roundings counted in test_gpu_gn.py."""
import math

import pytest
import torch
import torch.nn.functional as F

import workload

from .test_gpu_gn import OUT, _check_backward, _check_forward

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _gn_model(dtype, device="cuda", opts=()):
    model, cfg = workload.build_model(config="yolov3.yaml", dtype=dtype, device=device, opts=["MODEL.DARKNET.NORM", "GN"] + list(opts))
    g = torch.Generator().manual_seed(4)
    with torch.no_grad():   # norms that do something
        for n, p in model.named_parameters():
            if n.endswith(".norm.weight"):
                p.copy_(0.7 + 0.6 * torch.rand(p.shape, generator=g))
            elif n.endswith(".norm.bias"):
                p.copy_(0.2 * torch.randn(p.shape, generator=g))
    return model, cfg


def _inputs(cfg, N, S, seed=3):
    from oracle import yolo_train_ref as T
    from yolo_amd.structures import Boxes, Instances
    imgs = workload.synthetic_images(N, S, S, seed=seed)
    gb, gc = T.synthetic_targets(N, S, cfg.MODEL.YOLOV3.NUM_CLASSES, seed=11, max_boxes=6)
    return imgs, gb, gc, [dict(image=im, instances=Instances((S, S), gt_boxes=Boxes(b), gt_classes=c)) for im, b, c in zip(imgs, gb, gc)]


def _rel(got, ref):
    return float((got.double().cpu() - ref.double()).abs().max() / ref.double().abs().max())


@pytest.mark.parametrize("size", [(2, 128, 128), (1, 96, 160)], ids=lambda s: "x".join(map(str, s)))
def test_inference_fp32_matches_the_oracle(cuda, size):
    from oracle import yolo_train_ref as T
    model, cfg = _gn_model("f32")
    sd = {k: v.detach().cpu() for k, v in model.state_dict().items()}
    assert not any("running" in k for k in sd)
    N, H, W = size
    x = workload.synthetic_images(N, H, W, seed=5).float() / 255.0
    with torch.no_grad():
        ref = T.fpn_forward_train(x, sd)
    for _ in range(2):   # twice through one plan: in-place buffers start over
        heads = model.backbone(x.cuda())
        for k in ("p3", "p4", "p5"):
            assert _rel(heads[k], ref[k]) < 1e-3, k
    # new weights reach the plan
    with torch.no_grad():
        model.backbone.fpn_lateral0.blocks[4].norm.bias.add_(0.5)
        sd = {k: v.detach().cpu() for k, v in model.state_dict().items()}
        ref = T.fpn_forward_train(x, sd)
    assert _rel(model.backbone(x.cuda())["p5"], ref["p5"]) < 1e-3


def test_bf16_inference_and_frozen_training_forward_agree_bit_for_bit(cuda):
    """The inference plan (in place, side streams) and a training plan whose backbone is frozen (buffers of their own) run the same
    kernels on the same values; replaying the captured call gives the eager call's detections."""
    model, cfg = _gn_model("bf16", opts=["MODEL.BACKBONE.FREEZE_AT", 6])
    imgs = workload.synthetic_images(2, 160, 160, seed=7).cuda()
    eng = model.backbone.engine()
    eng.split_k = False
    eng._plans.clear()
    mean, std = model._mean, model._std
    P = eng.run_backbone(imgs, mean, std)
    heads = [h.interior().clone() for h in P.heads]
    model.train()
    want = model.backbone.train_engine().forward(imgs, mean, std)
    torch.cuda.synchronize()
    for a, b in zip(heads, want):
        assert torch.equal(a.float(), b.interior().float())
    model.eval()
    eng.split_k = True
    eng._plans.clear()
    model.test_score_thresh = 0.3
    inputs = [dict(image=i) for i in imgs]
    eager = model(inputs)
    model.graph_max_batch = 8
    for _ in range(4):
        got = model(inputs)
        for a, b in zip(eager, got):
            assert torch.equal(a["instances"].scores, b["instances"].scores)
            assert torch.equal(a["instances"].pred_boxes.tensor, b["instances"].pred_boxes.tensor)
        torch.zeros(1000, device="cuda").sum().item()   # eager work between the replays


@pytest.mark.parametrize("freeze_at", [2, 0])
def test_training_step_fp32_matches_the_oracle(cuda, freeze_at):
    from oracle import yolo_train_ref as T
    model, cfg = _gn_model("f32", opts=["MODEL.BACKBONE.FREEZE_AT", freeze_at])
    C = cfg.MODEL.YOLOV3.NUM_CLASSES
    imgs, gb, gc, inputs = _inputs(cfg, 3, 128)
    sd = {k: v.detach().cpu().clone() for k, v in model.state_dict().items()}
    params = {k: v.clone().requires_grad_(True) for k, v in sd.items() if v.dtype.is_floating_point}
    full = dict(sd)
    full.update(params)
    heads_ref = {}
    want = T.forward_training(imgs.float() / 255.0, full, gb, gc, C, freeze_at=freeze_at, heads_out=heads_ref)
    sum(want.values()).backward()
    model.train()
    got = model(inputs)
    sum(got.values()).backward()
    torch.cuda.synchronize()
    for k in want:
        assert abs(float(got[k].detach()) / float(want[k].detach()) - 1) < 1e-3, k
    frozen = set(T.frozen_names(freeze_at))
    n = 0
    for name, p in model.named_parameters():
        layer = name.rsplit(".norm.", 1)[0].rsplit(".weight", 1)[0].rsplit(".bias", 1)[0]
        if layer in frozen:
            assert p.grad is None and not p.requires_grad
            continue
        g, ref = p.grad.double().cpu().flatten(), params[name].grad.double().flatten()
        cos = float(F.cosine_similarity(g, ref, dim=0))
        assert cos > 0.998 and float((g - ref).norm() / ref.norm()) < 0.06, (name, cos)
        n += 1
    assert n == {2: 210, 0: 222}[freeze_at]


@pytest.mark.parametrize("freeze_at", [2, 0])
def test_bf16_layers_of_a_training_step(cuda, freeze_at):
    """Every normalised layer's y from its own z, and its dz, dgamma, dbeta from its own dy, z and statistics."""
    model, cfg = _gn_model("bf16", opts=["MODEL.BACKBONE.FREEZE_AT", freeze_at])
    imgs, gb, gc, inputs = _inputs(cfg, 2, 128)
    model.train()
    losses = model(inputs)
    sum(losses.values()).backward()
    torch.cuda.synchronize()
    assert all(math.isfinite(float(v)) for v in losses.values())
    P = model.backbone.train_engine().plan(2, 128, 128)
    n = 0
    for L in P.layers:
        gn = L.conv.group_norm
        if L.frozen or gn is None:
            continue
        assert L.sums_for is None or L.sums_for.conv.batch_norm is not None
        z, gamma, beta = L.z.interior().cpu(), gn.weight.detach().cpu(), gn.bias.detach().cpu()
        res = None if L.residual is None else L.residual.interior().cpu()
        _check_forward(z, res, gamma, beta, 32, "leaky", 0.1, L.y.interior(), L.stats)
        _check_backward(z, L.dy.interior().cpu(), gamma, beta, L.stats, 32, "leaky", 0.1,
                        (L.dz.interior().double().cpu(), L.dgamma.double().cpu(), L.dbeta.double().cpu()))
        n += 1
    assert n == {2: 68, 0: 72}[freeze_at]


def test_single_modules(cuda):
    """Conv2d and BasicStem called by themselves, against the same layers in fp32 torch on the CPU (1e-3, the fp32 convolution bar)."""
    model, _ = _gn_model("f32")
    b = model.backbone.bottom_up
    x = torch.randn(2, 64, 20, 24, generator=torch.Generator().manual_seed(0))
    block = b.res1[0]

    def ref(conv, t):
        t = F.conv2d(t, conv.weight.detach().cpu(), None, stride=conv.stride, padding=conv.padding)
        return F.leaky_relu(F.group_norm(t, 32, conv.norm.weight.detach().cpu(), conv.norm.bias.detach().cpu()), 0.1)

    t = block.conv1(x.cuda(), slope=0.1)
    assert _rel(t, ref(block.conv1, x)) < 1e-3
    y = block.conv2(t, slope=0.1, residual=x.cuda())
    assert _rel(y, ref(block.conv2, ref(block.conv1, x)) + x) < 1e-3
    img = torch.rand(1, 3, 40, 56, generator=torch.Generator().manual_seed(1))
    assert _rel(b.stem(img.cuda()), ref(b.stem.conv, img)) < 1e-3


@pytest.mark.parametrize("norm", ["GN", "BN"])
@pytest.mark.parametrize("clip", [("full_model", 0.5, 2.0), ("norm", 0.05, 2.0), ("norm", 1e-3, math.inf), ("value", 1e-3, 2.0)],
                         ids=lambda c: f"{c[0]}-{c[2]}")
def test_clipped_update_of_the_network(cuda, clip, norm):
    """Trainer steps with SOLVER.CLIP_GRADIENTS: the parameters after the first step are w - lr (clipped g + wd w), from the gradients
    that backward left; later steps stay finite; torch's own step with clipping in place gives the same parameters."""
    from yolo_amd.trainer import Trainer, synthetic_batches
    kind, value, p = clip

    def make():
        torch.manual_seed(0)
        model, cfg = workload.build_model(config="yolov3.yaml", dtype="bf16", opts=[
            "MODEL.DARKNET.NORM", norm, "SOLVER.IMS_PER_BATCH", 2, "SOLVER.BASE_LR", 1e-2, "SOLVER.WARMUP_ITERS", 0,
            "SOLVER.CLIP_GRADIENTS.ENABLED", True, "SOLVER.CLIP_GRADIENTS.CLIP_TYPE", kind,
            "SOLVER.CLIP_GRADIENTS.CLIP_VALUE", value, "SOLVER.CLIP_GRADIENTS.NORM_TYPE", p])
        return Trainer(cfg, model, synthetic_batches(cfg, 2, 96, seed=5, device=model.device), log=lambda m: None), cfg

    tr, cfg = make()
    before = {n: q.detach().double().cpu() for n, q in tr.model.named_parameters() if q.requires_grad}
    tr.run_step()
    assert tr.optimizer._fused is not None and tr.optimizer._clipper is not None
    named = {n: q for n, q in tr.model.named_parameters() if q.requires_grad}
    grads = {n: q.grad.double().cpu() for n, q in named.items()}
    norm_of = lambda t: float(t.abs().max() if p == math.inf else t.square().sum().sqrt())  # noqa: E731
    total = norm_of(torch.cat([g.flatten() for g in grads.values()]))
    clipped = 0
    for n, g in grads.items():
        if kind == "value":
            want = g.clamp(-value, value)
            clipped += int((want != g).any())
        else:
            k = min(1.0, value / ((norm_of(g) if kind == "norm" else total) + 1e-6))
            want, clipped = g * k, clipped + (k < 1)
        wd = 0.0 if ".norm." in n else cfg.SOLVER.WEIGHT_DECAY
        size = want.abs() + wd * before[n].abs()
        ref = before[n] - 1e-2 * (want + wd * before[n])
        tol = 10 * U * 1e-2 * size + U * (ref.abs() + before[n].abs())
        assert ((named[n].detach().double().cpu() - ref).abs() <= tol).all(), n
    assert clipped > 0
    for _ in range(2):
        assert all(math.isfinite(float(v)) for v in tr.run_step().values())
    # the same first step by torch's SGD: gradients clipped in place (two more roundings), then its own update
    import os
    os.environ["YOLO_FUSED_SGD"] = "0"
    try:
        other, _ = make()
        other.run_step()
    finally:
        del os.environ["YOLO_FUSED_SGD"]
    assert other.optimizer._fused is None
    for n, q in other.model.named_parameters():
        if q.requires_grad:
            g = q.grad.double().cpu()
            wd = 0.0 if ".norm." in n else cfg.SOLVER.WEIGHT_DECAY
            ref = before[n] - 1e-2 * (g + wd * before[n])   # .grad is the clipped gradient here
            tol = 12 * U * 1e-2 * (g.abs() + wd * before[n].abs()) + 2 * U * (ref.abs() + before[n].abs())
            assert ((q.detach().double().cpu() - ref).abs() <= tol).all(), n
            if kind == "value":
                assert float(g.abs().max()) <= value * (1 + 2 * U)
