"""Every form of the GroupNorm kernels (gn_forms.py) against the formulas in 64 bits, in place, over slices, next to the kink of the
leaky activation, with values that are not finite, and captured into a graph.

Tolerances as counted in test_gpu_gn.py, but the mean's part of the output is its own rounding: with s = gamma / sqrt(var + eps),
u (|mean s| + 256 max|x - mean| |s|) + 144 u (|(x - mean) s| + |beta| + |residual|)."""
import math

import pytest
import torch

from . import gn_forms
from .test_gpu_gn import OUT, U, _act, _ref_backward, _ref_stats, _spread, ids

pytestmark = pytest.mark.gpu
name = lambda c: ids(c[1]) + ("-bf16" if c[0] == torch.bfloat16 else "-f32") if isinstance(c[0], torch.dtype) else str(c)  # noqa: E731


def _inputs(cuda, shape, dtype, seed):
    N, H, W, C, G = shape
    g = torch.Generator(cuda).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    x = (rand(N, H, W, C) * (0.5 + torch.rand(C, generator=g, device=cuda)) + rand(C)).to(dtype)
    return x, rand(N, H, W, C).to(dtype), rand(N, H, W, C).to(dtype), 1 + 0.3 * rand(C), 0.3 * rand(C)


def _view(t, halo=0, extra=0, at=0):
    """A view over a copy of t in a buffer whose other elements are 7."""
    from yolo_amd import ops
    N, H, W, C = t.shape
    v = ops.View(torch.full((N, H + 2 * halo, W + 2 * halo, C + extra), 7.0, dtype=t.dtype, device=t.device), H, W, halo, C, at)
    v.interior().copy_(t)
    return v


def _only_inside(v):
    """Whether the buffer's other elements are still 7."""
    b = v.buf.clone()
    h = v.halo
    b[:, h:h + v.H, h:h + v.W, v.ch_offset:v.ch_offset + v.C] = 7
    return bool((b == 7).all())


def _ws(shape, dtype, cuda):
    from yolo_amd import ops
    return torch.full((ops.gn_workspace_bytes(*shape, dtype),), 255, dtype=torch.uint8, device=cuda)


def _forward(cuda, shape, x, r, gamma, beta, act="leaky", slope=0.1, views=(0, 0, 0), out=None, extra=0):
    """out: "x" or "r", the output over that one.  Returns y, stats."""
    from yolo_amd import ops
    N, H, W, C, G = shape
    xv, rv = _view(x, views[0], extra, extra // 8 * 4), None if r is None else _view(r, views[2])
    yv = {"x": xv, "r": rv, None: None}[out] or _view(torch.zeros_like(x), views[1], extra, extra)
    stats = torch.full((2, N, G), -1.0, device=cuda)
    ops.gn_act_fwd(xv, gamma, beta, yv, stats, _ws(shape, x.dtype, cuda), groups=G, act=act, slope=slope, residual=rv)
    assert _only_inside(yv) and (out == "x" or torch.equal(xv.interior().nan_to_num(), x.nan_to_num()))
    return yv.interior().clone(), stats


def _backward(cuda, shape, x, dy, gamma, beta, stats, act="leaky", slope=0.1, views=(0, 0, 0), out=None, extra=0):
    from yolo_amd import ops
    N, H, W, C, G = shape
    xv, dyv = _view(x, views[0], extra, extra // 8 * 4), _view(dy, views[1])
    dxv = {"x": xv, "dy": dyv, None: None}[out] or _view(torch.zeros_like(x), views[2], extra, extra)
    dg, db = torch.full((C,), 9.0, device=cuda), torch.full((C,), 9.0, device=cuda)
    ops.gn_act_bwd(dyv, xv, gamma, beta, stats, dxv, dg, db, _ws(shape, x.dtype, cuda), groups=G, act=act, slope=slope)
    assert _only_inside(dxv)
    return dxv.interior().clone(), dg, db


def _check_backward(shape, x, dy, gamma, beta, stats, act, slope, got):
    ref = _ref_backward(x, dy, gamma, beta, stats[0], stats[1], shape[4], act, slope)
    for what, a, b, tol in zip(("dx", "dgamma", "dbeta"), got, ref[:3], ref[3:]):
        tol = tol + OUT[x.dtype] * b.abs() if what == "dx" else tol
        over = float(((a.double() - b).abs() / tol.clamp_min(1e-300)).max())
        assert over <= 1, (what, over)


@pytest.mark.parametrize("act,slope", [("leaky", 0.1), ("silu", 0.0)], ids=["leaky", "silu"])
@pytest.mark.parametrize("case", gn_forms.FORWARD, ids=name)
def test_forward(cuda, case, act, slope):
    dtype, shape = case
    N, H, W, C, G = shape
    x, r, _, gamma, beta = _inputs(cuda, shape, dtype, 1)
    mean, rs = _ref_stats(x, G)
    xm = x.double() - _spread(mean, C)
    far = xm.abs().reshape(N, H * W, G, -1).amax((1, 3))
    s = gamma.double() * _spread(rs, C)
    t = xm * s + beta.double()
    size = 144 * ((xm * s).abs() + beta.double().abs()) + (_spread(mean, C).abs() + 256 * _spread(far, C)) * s.abs()
    del xm
    want = _act(t, act, slope)
    for res in (None, r):
        y, stats = _forward(cuda, shape, x, res, gamma, beta, act, slope, (1, 0, 1))
        got = stats.double()
        assert ((got[0] - mean).abs() <= U * (mean.abs() + 256 * far)).all()
        assert ((got[1] - rs).abs() <= 128 * U * rs).all()
        if res is not None:
            want, size = want + r.double(), size + 144 * r.double().abs()
        assert float(((y.double() - want).abs() / (OUT[dtype] * want.abs() + U * size)).max()) <= 1


@pytest.mark.parametrize("case", gn_forms.FORWARD, ids=name)
def test_forward_in_place_and_over_slices(cuda, case):
    """The same bits over x, over the residual, and between channel slices of wider buffers."""
    dtype, shape = case
    x, r, _, gamma, beta = _inputs(cuda, shape, dtype, 2)
    for res in (None, r):
        y, stats = _forward(cuda, shape, x, res, gamma, beta)
        for kw in (dict(out="x", views=(1, 0, 0)), dict(out="x" if res is None else "r", views=(0, 0, 1)), dict(extra=16, views=(0, 1, 0))):
            y2, stats2 = _forward(cuda, shape, x, res, gamma, beta, **kw)
            assert torch.equal(y2, y) and torch.equal(stats2, stats), kw


@pytest.mark.parametrize("act,slope", [("leaky", 0.1), ("silu", 0.0)], ids=["leaky", "silu"])
@pytest.mark.parametrize("case", gn_forms.BACKWARD, ids=name)
def test_backward(cuda, case, act, slope):
    dtype, shape = case
    x, _, dy, gamma, beta = _inputs(cuda, shape, dtype, 3)
    stats = torch.stack(_ref_stats(x, shape[4])).float()
    _check_backward(shape, x, dy, gamma, beta, stats, act, slope, _backward(cuda, shape, x, dy, gamma, beta, stats, act, slope, (1, 0, 1)))


@pytest.mark.parametrize("case", gn_forms.BACKWARD, ids=name)
def test_backward_in_place_and_over_slices(cuda, case):
    dtype, shape = case
    x, _, dy, gamma, beta = _inputs(cuda, shape, dtype, 4)
    stats = torch.stack(_ref_stats(x, shape[4])).float()
    got = _backward(cuda, shape, x, dy, gamma, beta, stats)
    for kw in (dict(out="x", views=(1, 0, 0)), dict(out="dy", views=(0, 1, 0)), dict(extra=16, views=(0, 0, 1))):
        again = _backward(cuda, shape, x, dy, gamma, beta, stats, **kw)
        assert all(torch.equal(a, b) for a, b in zip(again, got)), kw


@pytest.mark.parametrize("case", [c for c in gn_forms.BACKWARD if c[0] == gn_forms.F32], ids=name)
def test_the_side_of_the_kink_is_exact(cuda, case):
    """Every t within a few roundings of zero (see the test of this name in test_gpu_gn.py), in every form."""
    _, shape = case
    N, H, W, C, G = shape
    g = torch.Generator(cuda).manual_seed(C)
    rand = lambda *s: torch.rand(*s, generator=g, device=cuda)  # noqa: E731
    gamma, beta = 0.5 + rand(C), 0.5 + rand(C)
    beta[0] = 0.0
    stats = torch.stack([torch.randn(N, G, generator=g, device=cuda), 0.5 + rand(N, G)])
    zero = _spread(stats[0], C) - beta.double() / (gamma.double() * _spread(stats[1], C))
    x = zero.expand(N, H, W, C).float().contiguous()
    x = (x.view(torch.int32) + torch.randint(-3, 4, x.shape, generator=g, device=cuda, dtype=torch.int32)).view(torch.float32)
    x[:, 0, 0, 0] = stats[0, :, 0]       # t == 0 exactly: xh = 0, beta = 0
    dy = 1 + rand(N, H, W, C)
    t = (x.double() - _spread(stats[0], C)) * _spread(stats[1], C) * gamma.double() + beta.double()
    t32 = ((x - _spread(stats[0], C).float()) * _spread(stats[1], C).float()) * gamma + beta
    assert ((t > 0) != (t32 > 0)).sum() > 10     # the inputs do reach it
    _check_backward(shape, x, dy, gamma, beta, stats, "leaky", 0.1, _backward(cuda, shape, x, dy, gamma, beta, stats))


# one shape of each form; the bad values lie in its last image's second group: at pixel 0, and in the last pixel's last channel
BAD_FORWARD = [(F, s) for F, s in gn_forms.FORWARD if s in [(2, 13, 11, 128, 32), (64, 26, 26, 256, 32), (64, 46, 45, 128, 32), (64, 46, 45, 256, 32),
                                                           (128, 141, 20, 80, 5), (32, 95, 115, 32, 4), (9, 208, 207, 64, 32)]]
BAD_BACKWARD = [(F, s) for F, s in gn_forms.BACKWARD if s in [(64, 13, 13, 512, 32), (64, 31, 32, 256, 32), (130, 38, 37, 32, 32),
                                                             (130, 38, 37, 64, 32), (2, 20, 20, 192, 2), (9, 208, 207, 64, 32)]]


def _hit(shape, cuda):
    N, H, W, C, G = shape
    group = torch.zeros(N, 1, 1, C, dtype=torch.bool, device=cuda)
    group[-1, :, :, C // G:2 * C // G] = True
    return group.expand(N, H, W, C)


@pytest.mark.parametrize("at", ["first", "last"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
@pytest.mark.parametrize("case", BAD_FORWARD, ids=name)
def test_a_bad_value_stays_in_its_image_and_group_forward(cuda, case, bad, at):
    dtype, shape = case
    N, H, W, C, G = shape
    x, r, _, gamma, beta = _inputs(cuda, shape, dtype, 5)
    clean, stats0 = _forward(cuda, shape, x, r, gamma, beta)
    x[(-1, 0, 0, C // G) if at == "first" else (-1, H - 1, W - 1, 2 * C // G - 1)] = bad
    y, stats = _forward(cuda, shape, x, r, gamma, beta)
    hit = _hit(shape, cuda)
    assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], clean[~hit])
    assert not torch.isfinite(stats[:, -1, 1]).any()
    stats[:, -1, 1] = stats0[:, -1, 1]
    assert torch.equal(stats, stats0)


@pytest.mark.parametrize("at", ["first", "last"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
@pytest.mark.parametrize("case", BAD_BACKWARD, ids=name)
def test_a_bad_value_stays_in_its_image_and_group_backward(cuda, case, bad, at):
    dtype, shape = case
    N, H, W, C, G = shape
    x, _, dy, gamma, beta = _inputs(cuda, shape, dtype, 6)
    stats = torch.stack(_ref_stats(x, G)).float()
    d0, g0, b0 = _backward(cuda, shape, x, dy, gamma, beta, stats)
    c = C // G if at == "first" else 2 * C // G - 1
    dy[(-1, 0, 0, c) if at == "first" else (-1, H - 1, W - 1, c)] = bad
    dx, dg, db = _backward(cuda, shape, x, dy, gamma, beta, stats)
    hit, ch = _hit(shape, cuda), torch.arange(C, device=cuda) == c
    assert not torch.isfinite(dx[hit]).any() and torch.equal(dx[~hit], d0[~hit])
    assert not torch.isfinite(dg[ch]).any() and not torch.isfinite(db[ch]).any()
    assert torch.equal(dg[~ch], g0[~ch]) and torch.equal(db[~ch], b0[~ch])


@pytest.mark.parametrize("shape", [(64, 13, 13, 512, 32), (64, 46, 45, 256, 32), (9, 208, 207, 64, 32)], ids=ids)
def test_captured_forward_and_backward(cuda, shape):
    """Replays over new inputs, with eager work between them on the same buffers, give the eager calls' bits."""
    from yolo_amd import ops
    G, bf16 = shape[4], torch.bfloat16
    sets = [_inputs(cuda, shape, bf16, s)[:3] for s in (7, 8)]
    gamma, beta = _inputs(cuda, shape, bf16, 7)[3:]
    xv, rv, dyv = (_view(t, 1) for t in sets[0])
    yv, dxv = _view(torch.zeros_like(sets[0][0]), 1), _view(torch.zeros_like(sets[0][0]), 1)
    stats, dg, db = torch.empty(2, shape[0], G, device=cuda), torch.empty(shape[3], device=cuda), torch.empty(shape[3], device=cuda)
    ws = _ws(shape, bf16, cuda)

    def both():
        ops.gn_act_fwd(xv, gamma, beta, yv, stats, ws, groups=G, residual=rv)
        ops.gn_act_bwd(dyv, xv, gamma, beta, stats, dxv, dg, db, ws, groups=G)

    def run(i, go):
        for v, t in zip((xv, rv, dyv), sets[i]):
            v.interior().copy_(t)
        torch.cuda.synchronize()
        go()
        torch.cuda.synchronize()
        return [t.clone() for t in (yv.interior(), stats, dxv.interior(), dg, db)]

    want = [run(i, both) for i in range(2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for i in (1, 0, 0, 1):
        assert all(torch.equal(a, b) for a, b in zip(run(i, graph.replay), want[i])), i
        run(1 - i, both)


def test_adjacent_memory_is_taken(cuda):
    """Everything of a call end to end in one buffer: nothing is shared, nothing is refused, and the bits are the same."""
    from yolo_amd import ops
    shape = N, H, W, C, G = 2, 4, 4, 64, 8
    x, r, dy, gamma, beta = _inputs(cuda, shape, torch.float32, 9)
    y, stats = _forward(cuda, shape, x, r, gamma, beta)
    want = _backward(cuda, shape, x, dy, gamma, beta, stats)
    sizes = [x.numel()] * 5 + [C] * 4 + [2 * N * G, ops.gn_workspace_bytes(*shape, torch.float32) // 4]
    bx, br, bdy, by, bdx, bg, bb, dg, db, st, ws = torch.zeros(sum(sizes), device=cuda).split(sizes)
    for b, t in ((bx, x), (br, r), (bdy, dy), (bg, gamma), (bb, beta)):
        b.copy_(t.flatten())
    v = lambda b: ops.View(b.view(N, H, W, C), H, W, 0, C)  # noqa: E731
    ops.gn_act_fwd(v(bx), bg, bb, v(by), st, ws, groups=G, residual=v(br))
    ops.gn_act_bwd(v(bdy), v(bx), bg, bb, st, v(bdx), dg, db, ws, groups=G)
    assert torch.equal(by.view_as(y), y) and torch.equal(st.view_as(stats), stats)
    assert all(torch.equal(a.view_as(b), b) for a, b in zip((bdx, dg, db), want))
