"""What the GroupNorm and gradient-clipping entry points refuse before any launch, and their host-side parts (no GPU)."""
import ctypes

import pytest
import torch

from yolo_amd import _lib, ops, solver


def _view(H=8, W=8, halo=0, total=64, at=0, ptr=4096):
    return _lib.YoloView(ptr, H, W, halo, total, at)


def _fwd(x=None, y=None, r=None, N=1, C=64, groups=32, eps=1e-5, act=0, slope=0.1, dtype=1, ws=1 << 30, ptr=4096):
    L = _lib.lib()
    x, y = x or _view(), y or _view()
    code = L.yolo_gn_act_fwd(ctypes.byref(x), ptr, ptr, ctypes.byref(r) if r else None, ctypes.byref(y), ptr, N, C, groups, eps,
                             act, slope, dtype, ptr, ws, None)
    return code, L.yolo_last_error().decode()


def _bwd(dy=None, x=None, dx=None, N=1, C=64, groups=32, act=0, slope=0.1, dtype=1, ws=1 << 30, ptr=4096, dgamma=None, dbeta=None):
    L = _lib.lib()
    dy, x, dx = dy or _view(), x or _view(), dx or _view()
    at = lambda i: ptr and ptr + 4096 * i  # noqa: E731
    dgamma, dbeta = at(3) if dgamma is None else dgamma, at(4) if dbeta is None else dbeta
    code = L.yolo_gn_act_bwd(ctypes.byref(dy), ctypes.byref(x), at(1), at(2), ptr, ctypes.byref(dx), dgamma, dbeta, N, C, groups,
                             act, slope, dtype, ptr, ws, None)
    return code, L.yolo_last_error().decode()


@pytest.mark.parametrize("call", [_fwd, _bwd], ids=["fwd", "bwd"])
@pytest.mark.parametrize("kw,says", [
    (dict(ptr=None), "null"), (dict(x=_view(ptr=None)), "null"), (dict(x=_view(H=0)), "expected"), (dict(N=0), "batch"),
    (dict(N=65535), "batch"), (dict(N=32768, C=32768, groups=32768, x=_view(1, 1, total=32768)), "2^30"), (dict(C=60), "channels"), (dict(C=0), "channels"), (dict(groups=0), "groups"),
    (dict(groups=7), "groups"), (dict(act=2), "activation"), (dict(slope=-0.1), "slope"), (dict(slope=float("nan")), "slope"),
    (dict(dtype=2), "dtype"), (dict(ws=16), "workspace"), (dict(x=_view(at=8)), "slice"), (dict(x=_view(total=68)), "slice"),
    (dict(x=_view(ptr=4100)), "aligned"), (dict(x=_view(H=4096, W=4096, total=64)), "2 GiB")],
    ids=lambda v: "-".join(v) if isinstance(v, dict) else v.replace(" ", ""))
def test_gn_refusals(call, kw, says):
    code, message = call(**kw)
    assert code < 0 and says in message, message


def test_gn_refusals_of_one_direction():
    assert "y is 8 x 9" in _fwd(y=_view(W=9))[1] and "residual is 7 x 8" in _fwd(r=_view(H=7))[1]
    assert "eps" in _fwd(eps=-1.0)[1] and "dy is 9 x 8" in _bwd(dy=_view(H=9))[1] and "dx is 8 x 4" in _bwd(dx=_view(W=4))[1]
    assert _fwd(ws=16)[0] == -2
    wide = lambda at, halo=0: _view(halo=halo, total=192, at=at)  # noqa: E731
    for kw in (dict(x=wide(0), y=wide(8)), dict(x=wide(64), y=wide(64, 1)), dict(x=wide(128), y=wide(0), r=wide(56))):
        assert "lies over part" in _fwd(**kw)[1]
    assert "lies over part of dy" in _bwd(x=wide(0), dx=wide(64), dy=wide(72))[1]
    image = 8 * 8 * 64 * 2     # buffers that begin elsewhere: images of one batch, the last byte of a neighbour
    for at in (image, -image, 2 * image - 16, 16 - 2 * image):
        assert "lies over part" in _fwd(N=2, x=_view(ptr=1 << 20), y=_view(ptr=(1 << 20) + at))[1]
        assert "lies over part of dy" in _bwd(N=2, x=_view(ptr=1 << 30), dy=_view(ptr=1 << 20), dx=_view(ptr=(1 << 20) + at))[1]
    for at in (2 * image, -2 * image):
        assert _fwd(N=2, x=_view(ptr=1 << 20), y=_view(ptr=(1 << 20) + at), ws=16)[0] == -2
    for kw in (dict(dgamma=8192), dict(dgamma=3 * 4096), dict(dbeta=8192), dict(dbeta=3 * 4096), dict(dgamma=1 << 16, dbeta=1 << 16)):
        assert "memory of their own" in _bwd(**kw)[1]
    L = _lib.lib()
    assert L.yolo_gn_workspace_bytes(0, 8, 8, 64, 32, 1) == 0 and L.yolo_gn_workspace_bytes(1, 8, 8, 60, 4, 1) == 0
    assert L.yolo_gn_workspace_bytes(64, 208, 208, 64, 32, 1) > 0


def test_grad_refusals():
    L = _lib.lib()
    p = 4096
    inf = float("inf")
    for args, says in (((p, 1, None, 0, 2.0, 1.0, None, p, p, 8), "null"), ((None, 1, None, 0, 2.0, 1.0, p, p, p, 8), "null"),
                       ((p, -1, None, 0, 2.0, 1.0, p, p, p, 8), "blocks"), ((p, 1, p, 0, 2.0, 1.0, p, p, p, 8), "tensors"),
                       ((p, 1, None, 0, 3.0, 1.0, p, p, p, 8), "norm type"), ((p, 1, None, 0, -inf, 1.0, p, p, p, 8), "norm type"),
                       ((p, 1, None, 0, 2.0, -1.0, p, p, p, 8), "max_norm"), ((p, 2, None, 0, inf, 1.0, p, p, p, 8), "workspace")):
        for call in (L.yolo_grad_norm, L.yolo_grad_clip):
            assert call(*args, None) < 0 and says in L.yolo_last_error().decode(), says
    assert L.yolo_grad_clip(p, 1, None, 0, 2.0, 1.0, p, None, p, 8, None) < 0 and L.yolo_grad_clamp(p, 1, -1.0, None) < 0
    assert L.yolo_grad_clamp(p, 1, float("nan"), None) < 0
    step = lambda w, n, coefs, v: L.yolo_sgd_step_clipped(w, p, p, p, n, 0.1, 0.0, 0.1, 0.0, 0.9, coefs, 0, v, None)  # noqa: E731
    assert step(None, 1, p, 0.0) < 0 and step(p, 0, p, 0.0) < 0 and step(p, 1, None, -1.0) < 0 and step(p + 4, 1, p, 0.0) < 0


def test_dense_runs():
    t = torch.zeros(4, 6, 3, 3)
    for v in (t, t.contiguous(memory_format=torch.channels_last), t[:2], t.permute(2, 0, 3, 1), t[:, :1, :1, :1][:1], torch.zeros(())):
        assert ops._dense_run(v)
    for v in (t[:, :2], t[..., ::2], t[:1].expand(5, 6, 3, 3), torch.zeros(8)[::2]):
        assert not ops._dense_run(v)


@pytest.mark.parametrize("segments", [[(0, 5, 0)], [(3, 4096, 1), (4099, 10_000, 0)], [(8, 0, 0), (8, 9000, 1)], [(20_000, 7, 0), (0, 9, 1)]],
                         ids=str)
def test_step_table_covers_each_element_once(segments):
    t = ops.sgd_clip_table(segments, "cpu")
    got = {}
    for first, count, group, tensor in t.blocks.tolist():
        assert 0 < count <= 4096 and segments[tensor][2] == group
        for i in range(first, first + count):
            assert i not in got
            got[i] = tensor
    want = {i: k for k, (a, n, _) in enumerate(segments) for i in range(a, a + n)}
    assert got == want and t.n_blocks == len(t.blocks) and t.end == max(want) + 1 and t.n_tensors == len(segments)


def test_step_table_refusals():
    for bad in ([], [(0, 0, 0)], [(0, 5, 2)], [(-1, 5, 0)], [(0, 5, 0), (4, 2, 1)], [(0, 1 << 31, 0)]):
        with pytest.raises(ValueError):
            ops.sgd_clip_table(bad, "cpu")


def test_clip_settings():
    from yolo_amd.config import get_cfg
    cfg = get_cfg()
    assert cfg.SOLVER.CLIP_GRADIENTS.ENABLED is False and cfg.SOLVER.CLIP_GRADIENTS.CLIP_TYPE == "value"
    model = torch.nn.Sequential(torch.nn.Linear(3, 2))
    assert solver.build_optimizer(cfg, model)._clip is None
    cfg.merge_from_list(["SOLVER.CLIP_GRADIENTS.ENABLED", True, "SOLVER.CLIP_GRADIENTS.CLIP_TYPE", "full_model",
                         "SOLVER.CLIP_GRADIENTS.CLIP_VALUE", 10.0])
    opt = solver.build_optimizer(cfg, model)
    assert opt._clip == ("full_model", 10.0, 2.0)
    for word in ("inf", ".inf", float("inf")):
        c = cfg.clone()
        c.merge_from_list(["SOLVER.CLIP_GRADIENTS.NORM_TYPE", word])
        assert solver.build_optimizer(c, model)._clip == ("full_model", 10.0, float("inf"))
    opt.step()                     # no gradients: nothing to clip
    with pytest.raises(RuntimeError, match="closure"):
        opt.step(lambda: 0.0)
    model[0].weight.grad = torch.ones(2, 3)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        opt.step()
    for key, value in (("CLIP_TYPE", "each"), ("CLIP_VALUE", -1.0), ("NORM_TYPE", 3.0)):
        c = cfg.clone()
        c.merge_from_list([f"SOLVER.CLIP_GRADIENTS.{key}", value])
        with pytest.raises(ValueError):
            solver.build_optimizer(c, model)
    assert float(solver.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0)) == 0.0


def test_group_norm_network_is_built_and_refuses_what_it_cannot(tmp_path):
    import workload
    from yolo_amd.checkpoint import YOLOV3Checkpointer
    from yolo_amd.checkpoint.load_darknet import save_darknet_weights
    from yolo_amd.modeling.backbone.layers import GroupNorm, get_norm
    from yolo_amd.utils.calibrate import calibrate_norm_stats
    model, cfg = workload.build_model(config="yolov3.yaml", device="cpu", opts=["MODEL.DARKNET.NORM", "GN"])
    convs = dict(model.backbone.darknet_modules())
    norms = [c.norm for c in convs.values() if c.norm is not None]
    assert len(norms) == 72 and all(isinstance(n, GroupNorm) and n.num_groups == 32 for n in norms)
    keys = [k for k in model.state_dict() if ".norm." in k]
    assert len(keys) == 144 and all(k.endswith((".norm.weight", ".norm.bias")) for k in keys)
    w, b = convs["bottom_up.res2.0.conv1"].folded()
    assert torch.equal(w, convs["bottom_up.res2.0.conv1"].weight) and float(b.abs().max()) == 0.0
    opt = solver.build_optimizer(cfg, model)
    assert sum(len(g["params"]) for g in opt.param_groups) == 210 and opt.param_groups[1]["weight_decay"] == 0.0
    bn, _ = workload.build_model(config="yolov3.yaml", device="cpu")
    path = str(tmp_path / "x.weights")
    with open(path, "wb") as f:
        save_darknet_weights(f, bn.backbone.darknet_modules())
    with pytest.raises(ValueError, match="BatchNorm parameters"):
        YOLOV3Checkpointer(model).load(path)
    with open(path, "wb") as f, pytest.raises(ValueError, match="BatchNorm parameters"):
        save_darknet_weights(f, model.backbone.darknet_modules())
    with pytest.raises(ValueError, match="no running statistics"):
        calibrate_norm_stats(model.backbone, torch.zeros(1, 3, 32, 32))
    with pytest.raises(ValueError, match="do not divide"):
        get_norm("GN", 48)
    with pytest.raises(ValueError, match="not supported"):
        get_norm("LN", 64)
    # a checkpoint of the same network round-trips
    torch.save({"model": model.state_dict()}, str(tmp_path / "gn.pth"))
    other, _ = workload.build_model(config="yolov3.yaml", device="cpu", seed=1, opts=["MODEL.DARKNET.NORM", "GN"])
    YOLOV3Checkpointer(other).load(str(tmp_path / "gn.pth"))
    assert all(torch.equal(a, b) for a, b in zip(model.state_dict().values(), other.state_dict().values()))
