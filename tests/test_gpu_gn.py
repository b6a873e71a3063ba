"""Group normalisation + activation (forward, backward) through ops.gn_act_fwd / gn_act_bwd against the formulas in 64 bits.

Tolerances are sums of roundings (u = 2^-24 for fp32 arithmetic; the output's own rounding is 2^-8 relative in bf16):
  statistics   a thread sums at most 128 values in fp32 (differences from the first one it sees), fp64 follows: the mean is
               off by at most u (|mean| + 2 * 128 max|x - mean|), 1/sqrt(var + eps) by 128 u relative
  y            with s = gamma / sqrt(var + eps): u * 144 * (|mean s| + |(x - mean) s| + |beta| + |residual|): the statistics'
               128 u, the half dozen roundings of the expression, and for silu (|t| + 6) u for exp and reciprocal, |t| < 10
  sums of d    at most 128 values in a thread and 256 threads in fp32: 512 u times the sum of absolute values
  dx           r * (u * 64 * |gamma d| + 512 u * (mean|gamma d| + |xh| mean|gamma d xh|)) (d itself: the derivative of silu
               is off by at most (|t| + 16) u)
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
OUT = {torch.float32: U, torch.bfloat16: 2.0 ** -8}

# (N, H, W, C, groups): one pixel, one value in a group, groups across vectors (3, 12, 257 channels), one group, a slab that is
# not full, more chunks than one, the network's own stages
SHAPES = [(1, 1, 1, 8, 8), (2, 1, 1, 8, 1), (3, 2, 3, 24, 8), (2, 5, 7, 96, 32), (1, 13, 13, 1024, 32), (2, 13, 13, 512, 32),
          (1, 3, 5, 1024, 1), (2, 4, 3, 2056, 8), (5, 26, 25, 256, 32), (1, 52, 52, 128, 32), (2, 61, 47, 64, 32),
          (1, 104, 90, 32, 32), (70, 6, 5, 384, 32), (3, 17, 1, 40, 5), (2, 1, 300, 72, 6), (1, 208, 200, 16, 2),
          (1, 208, 200, 64, 32), (64, 96, 50, 16, 2), (3, 50, 45, 96, 4), (8, 52, 40, 256, 32)]
ids = lambda s: "x".join(map(str, s)) if isinstance(s, tuple) else str(s).replace("torch.", "")  # noqa: E731


def _inputs(shape, dtype, seed=0):
    N, H, W, C, G = shape
    g = torch.Generator().manual_seed(seed + C + H)
    x = (torch.randn(N, H, W, C, generator=g) * (0.5 + torch.rand(C, generator=g)) + torch.randn(C, generator=g)).to(dtype)
    r = torch.randn(N, H, W, C, generator=g).to(dtype)
    dy = torch.randn(N, H, W, C, generator=g).to(dtype)
    return x, r, dy, 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)


def _act(t, act, slope):
    if act == "silu":
        return t * torch.sigmoid(t)
    return torch.where(t > 0, t, t * slope)


def _grp(t, G):
    """[N, H, W, C] -> its mean over each (image, group), broadcast back."""
    N, H, W, C = t.shape
    m = t.reshape(N, H * W, G, C // G).mean((1, 3))
    return m.repeat_interleave(C // G, 1).view(N, 1, 1, C)


def _ref_stats(x, G, eps=1e-5):
    N, H, W, C = x.shape
    v = x.double().reshape(N, H * W, G, C // G)
    return v.mean((1, 3)), 1 / (v.var((1, 3), unbiased=False) + eps).sqrt()


def _spread(t, C):
    N, G = t.shape
    return t.double().repeat_interleave(C // G, 1).view(N, 1, 1, C)


def _view(t, cuda, halo=0, extra=0, at=0):
    """A view of a buffer with ``extra`` more channels (the slice begins at channel ``at``), everything around it 7."""
    from yolo_amd import ops
    N, H, W, C = t.shape
    buf = torch.full((N, H + 2 * halo, W + 2 * halo, C + extra), 7.0, dtype=t.dtype, device=cuda)
    v = ops.View(buf, H, W, halo, C, at)
    v.interior().copy_(t.to(cuda))
    return v


def _around(v):
    """The buffer with the view's own elements set to zero."""
    b = v.buf.float().cpu().clone()
    h = v.halo
    b[:, h:h + v.H, h:h + v.W, v.ch_offset:v.ch_offset + v.C] = 0
    return b


def _forward(cuda, x, r, gamma, beta, G, act="leaky", slope=0.1, halo=(0, 0, 0), extra=0, at=0, eps=1e-5):
    from yolo_amd import ops
    N, H, W, C = x.shape
    xv, yv = _view(x, cuda, halo[0], extra, at), _view(torch.zeros_like(x), cuda, halo[1])
    rv = None if r is None else _view(r, cuda, halo[2])
    stats = torch.full((2, N, G), -1.0, device=cuda)
    ws = torch.full((ops.gn_workspace_bytes(N, H, W, C, G, x.dtype),), 255, dtype=torch.uint8, device=cuda)
    before = _around(yv)
    ops.gn_act_fwd(xv, gamma.to(cuda), beta.to(cuda), yv, stats, ws, groups=G, eps=eps, act=act, slope=slope, residual=rv)
    torch.cuda.synchronize()
    assert torch.equal(_around(yv), before)     # nothing outside the view is written
    return xv, yv, stats, ws


def _check_forward(x, r, gamma, beta, G, act, slope, y, stats, eps=1e-5):
    N, H, W, C = x.shape
    mean, rs = _ref_stats(x, G, eps)
    xm = (x.double() - _spread(mean, C))
    spread = xm.abs().reshape(N, H * W, G, -1).amax((1, 3))
    got = stats.double().cpu()
    assert ((got[0] - mean).abs() <= U * (mean.abs() + 256 * spread)).all()
    assert ((got[1] - rs).abs() <= 128 * U * rs).all()
    s = gamma.double() * _spread(rs, C)
    want = _act(xm * s + beta.double(), act, slope)
    size = (_spread(mean, C) * s).abs() + (xm * s).abs() + beta.double().abs()
    if r is not None:
        want, size = want + r.double(), size + r.double().abs()
    err = (y.double().cpu() - want).abs()
    tol = OUT[x.dtype] * want.abs() + 144 * U * size
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())


@pytest.mark.parametrize("act,slope", [("leaky", 0.1), ("silu", 0.0)], ids=["leaky", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=ids)
def test_forward(cuda, shape, dtype, act, slope):
    x, r, _, gamma, beta = _inputs(shape, dtype)
    G = shape[4]
    for res in (None, r):
        _, yv, stats, _ = _forward(cuda, x, res, gamma, beta, G, act, slope, halo=(1, 0, 2))
        _check_forward(x, res, gamma, beta, G, act, slope, yv.interior(), stats)


# every CU has a slab that its registers do not hold: the rest in LDS, or read again too; far means as well
@pytest.mark.parametrize("dtype,shape,act,far", [(torch.bfloat16, (256, 59, 51, 64, 32), "leaky", 0.0),
                                                 (torch.float32, (256, 59, 51, 32, 8), "silu", 100.0),
                                                 (torch.bfloat16, (256, 66, 61, 64, 4), "silu", 0.0)], ids=ids)
def test_forward_of_tall_slabs(cuda, dtype, shape, act, far):
    from yolo_amd import ops
    x, r, _, gamma, beta = _inputs(shape, dtype)
    N, H, W, C, G = shape
    x = x + far
    for res in (None, r):
        _, yv, stats, ws = _forward(cuda, x, res, gamma, beta, G, act, 0.1, halo=(1, 0, 2))
        _check_forward(x, res, gamma, beta, G, act, 0.1, yv.interior(), stats)
    for over_x in (False, True):   # in place: the same bits
        xv, rv = _view(x, cuda, 1), _view(r, cuda, 1)
        out, again = (xv if over_x else rv), torch.empty_like(stats)
        ops.gn_act_fwd(xv, gamma.to(cuda), beta.to(cuda), out, again, ws, groups=G, act=act, slope=0.1, residual=rv)
        assert torch.equal(out.interior(), yv.interior()) and torch.equal(again, stats)


def _ref_backward(x, dy, gamma, beta, mean, rs, G, act, slope):
    """The formulas at given statistics, in 64 bits; (dx, dgamma, dbeta) and their tolerances' sizes."""
    N, H, W, C = x.shape
    mean, rs, gamma, beta = _spread(mean, C), _spread(rs, C), gamma.double(), beta.double()
    xh = (x.double() - mean) * rs
    t = xh * gamma + beta
    if act == "silu":
        sg = torch.sigmoid(t)
        k = sg * (1 + t * (1 - sg))
        kerr = (t.abs() + 16) * 1.1     # |silu'| < 1.1, |silu''| <= 0.5
    else:
        k = torch.where(t > 0, torch.ones_like(t), torch.full_like(t, slope))
        kerr = torch.zeros_like(t)
    d = dy.double() * k
    size = d.abs() + kerr / 64 * dy.double().abs()
    dx = rs * (gamma * d - _grp(gamma * d, G) - xh * _grp(gamma * d * xh, G))
    g = gamma.abs() * size
    dx_tol = rs * U * (64 * g + 512 * (_grp(g, G) + xh.abs() * _grp(g * xh.abs(), G)))
    return (dx, (d * xh).sum((0, 1, 2)), d.sum((0, 1, 2)),
            dx_tol, 512 * U * (size * xh.abs()).sum((0, 1, 2)), 512 * U * size.sum((0, 1, 2)))


def _backward(cuda, x, dy, gamma, beta, stats, G, act, slope, halo=(0, 0, 0), extra=0, at=0):
    from yolo_amd import ops
    N, H, W, C = x.shape
    xv, dyv, dxv = _view(x, cuda, halo[0]), _view(dy, cuda, halo[1], extra, at), _view(torch.zeros_like(x), cuda, halo[2])
    dg, db = torch.full((C,), 9.0, device=cuda), torch.full((C,), 9.0, device=cuda)
    ws = torch.full((ops.gn_workspace_bytes(N, H, W, C, G, x.dtype),), 255, dtype=torch.uint8, device=cuda)
    before = _around(dxv)
    ops.gn_act_bwd(dyv, xv, gamma.to(cuda), beta.to(cuda), stats.to(cuda), dxv, dg, db, ws, groups=G, act=act, slope=slope)
    torch.cuda.synchronize()
    assert torch.equal(_around(dxv), before)
    return dxv.interior().double().cpu(), dg.double().cpu(), db.double().cpu()


def _check_backward(x, dy, gamma, beta, stats, G, act, slope, got):
    ref = _ref_backward(x, dy, gamma, beta, stats[0].cpu(), stats[1].cpu(), G, act, slope)
    for what, a, b, tol in zip(("dx", "dgamma", "dbeta"), got, ref[:3], ref[3:]):
        if what == "dx":
            tol = tol + OUT[x.dtype] * b.abs()
        err = (a - b).abs()
        assert (err <= tol).all(), (what, float((err / tol.clamp_min(1e-300)).max()))


@pytest.mark.parametrize("act,slope", [("leaky", 0.1), ("leaky", 0.0), ("leaky", 1.0), ("silu", 0.0)],
                         ids=["leaky", "relu", "none", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=ids)
def test_backward(cuda, shape, dtype, act, slope):
    x, _, dy, gamma, beta = _inputs(shape, dtype, seed=3)
    G = shape[4]
    stats = torch.stack(_ref_stats(x, G)).float()
    _check_backward(x, dy, gamma, beta, stats, G, act, slope, _backward(cuda, x, dy, gamma, beta, stats, G, act, slope, (1, 0, 2)))


# images whose slabs are held in part: each thread's last pixels in LDS or read again; few and many of them, slabs of 80 bytes
TALL = [(128, 33, 35, 64, 32), (128, 43, 41, 64, 16), (130, 40, 40, 40, 5), (256, 64, 62, 16, 1)]


@pytest.mark.parametrize("act,slope", [("leaky", 0.1), ("silu", 0.0)], ids=["leaky", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", TALL, ids=ids)
def test_backward_of_tall_slabs(cuda, shape, dtype, act, slope):
    from yolo_amd import ops
    x, _, dy, gamma, beta = _inputs(shape, dtype, seed=4)
    N, H, W, C, G = shape
    stats = torch.stack(_ref_stats(x, G)).float()
    got = _backward(cuda, x, dy, gamma, beta, stats, G, act, slope, (1, 0, 2))
    _check_backward(x, dy, gamma, beta, stats, G, act, slope, got)
    for over_x in (False, True):   # in place: the same bits
        xv, dyv = _view(x, cuda, 1), _view(dy, cuda, 1)
        dg, db = torch.empty(C, device=cuda), torch.empty(C, device=cuda)
        ws = torch.empty(ops.gn_workspace_bytes(N, H, W, C, G, dtype), dtype=torch.uint8, device=cuda)
        out = xv if over_x else dyv
        ops.gn_act_bwd(dyv, xv, gamma.to(cuda), beta.to(cuda), stats.to(cuda), out, dg, db, ws, groups=G, act=act, slope=slope)
        for a, b in zip((out.interior(), dg, db), got):
            assert torch.equal(a.double().cpu(), b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_views_slices_halos_and_buffers_used_twice(cuda, dtype):
    """Channel slices of wider buffers, in-place outputs: the same bits as separate buffers, nothing else written."""
    from yolo_amd import ops
    x, r, dy, gamma, beta = _inputs((2, 9, 11, 64, 32), dtype, seed=5)
    _, yv, stats, ws = _forward(cuda, x, r, gamma, beta, 32)
    want = yv.interior().clone()
    _, sl, _, _ = _forward(cuda, x, r, gamma, beta, 32, halo=(1, 1, 0), extra=24, at=16)
    assert torch.equal(sl.interior(), want)
    ga, be = gamma.to(cuda), beta.to(cuda)
    # into a slice of a wider buffer
    wide = ops.View(torch.full((2, 11, 13, 96), 7.0, dtype=dtype, device=cuda), 9, 11, 1, 64, 32)
    around = _around(wide)
    xv, rv = _view(x, cuda), _view(r, cuda, 1)
    ops.gn_act_fwd(xv, ga, be, wide, stats, ws, groups=32, residual=rv)
    assert torch.equal(wide.interior(), want) and torch.equal(_around(wide), around)
    # over the residual, over the input
    ops.gn_act_fwd(xv, ga, be, rv, stats, ws, groups=32, residual=rv)
    assert torch.equal(rv.interior(), want)
    rv, xi = _view(r, cuda), _view(x, cuda, 1)
    ops.gn_act_fwd(xi, ga, be, xi, stats, ws, groups=32, residual=rv)
    assert torch.equal(xi.interior(), want)
    # backward: over dy, over x
    dg, db = torch.empty(64, device=cuda), torch.empty(64, device=cuda)
    dx, dg0, db0 = _backward(cuda, x, dy, gamma, beta, stats, 32, "leaky", 0.1, (1, 1, 0), 40, 8)
    for which in ("dy", "x"):
        xv, dyv = _view(x, cuda, 1), _view(dy, cuda)
        out = dyv if which == "dy" else xv
        ops.gn_act_bwd(dyv, xv, ga, be, stats, out, dg, db, ws, groups=32)
        assert torch.equal(out.interior().double().cpu(), dx)
        assert torch.equal(dg.double().cpu(), dg0) and torch.equal(db.double().cpu(), db0)


@pytest.mark.parametrize("shape", [(2, 13, 13, 64, 32), (1, 40, 40, 32, 8), (2, 208, 104, 16, 2), (128, 43, 41, 64, 16)],
                         ids=ids)
def test_the_side_of_the_kink_is_exact(cuda, shape):
    """Leaky derivative next to t = 0: every t is within a few roundings of zero, so that fp32 arithmetic takes the wrong side for
    many of them; a wrong one moves dx by 0.9 |gamma d r|, far above the tolerance.  t == 0 takes the slope."""
    N, H, W, C, G = shape
    g = torch.Generator().manual_seed(C)
    gamma, beta = 0.5 + torch.rand(C, generator=g), 0.5 + torch.rand(C, generator=g)
    beta[0] = 0.0
    stats = torch.stack([torch.randn(N, G, generator=g), 0.5 + torch.rand(N, G, generator=g)])
    zero = _spread(stats[0], C) - beta.double() / (gamma.double() * _spread(stats[1], C))
    x = zero.expand(N, H, W, C).float()
    steps = torch.randint(-3, 4, (N, H, W, C), generator=g, dtype=torch.int32)
    x = (x.contiguous().view(torch.int32) + steps).view(torch.float32)
    x[:, 0, 0, 0] = stats[0, :, 0]       # t == 0 exactly: xh = 0, beta = 0
    dy = 1 + torch.rand(N, H, W, C, generator=g)
    got = _backward(cuda, x, dy, gamma, beta, stats, G, "leaky", 0.1)
    t = (x.double() - _spread(stats[0], C)) * _spread(stats[1], C) * gamma.double() + beta.double()
    t32 = ((x - _spread(stats[0], C).float()) * _spread(stats[1], C).float()) * gamma + beta
    assert ((t > 0) != (t32 > 0)).sum() > 10     # the inputs do reach it
    _check_backward(x, dy, gamma, beta, stats, G, "leaky", 0.1, got)


def test_gradient_against_differences(cuda):
    """(L(x + h v) - L(x - h v)) / 2h of the kernel's own forward against <dx, v>, and the same for gamma and beta: apart by what
    the difference quotient of the 64-bit formula is apart from its gradient, and the forward's tolerance over h."""
    N, H, W, C, G = shape = (2, 5, 4, 48, 8)
    x, _, dy, gamma, beta = _inputs(shape, torch.float32, seed=11)
    g = torch.Generator().manual_seed(1)
    h = 2.0 ** -6
    stats = torch.stack(_ref_stats(x, G)).float()
    grads = _backward(cuda, x, dy, gamma, beta, stats, G, "silu", 0.0)

    def ref(x, gamma, beta):
        m, rs = _ref_stats(x, G)
        return (_act((x.double() - _spread(m, C)) * _spread(rs, C) * gamma.double() + beta.double(), "silu", 0) * dy.double()).sum()

    def ours(x, gamma, beta):
        return (_forward(cuda, x, None, gamma, beta, G, "silu")[1].interior().double().cpu() * dy.double()).sum()

    for i, base in enumerate((x, gamma, beta)):
        v = (torch.randint(0, 2, base.shape, generator=g) * 2 - 1).float()
        args = [x, gamma, beta]
        shift = lambda s: [a + s * h * v if k == i else a for k, a in enumerate(args)]  # noqa: E731
        leaf = base.double().requires_grad_(True)
        ref(*[leaf if k == i else a.double() for k, a in enumerate(args)]).backward()
        slope64 = float((leaf.grad * v.double()).sum())
        quotient64 = float(ref(*shift(1)) - ref(*shift(-1))) / (2 * h)
        quotient = float(ours(*shift(1)) - ours(*shift(-1))) / (2 * h)
        ours_slope = float((grads[i] * v.double()).sum())
        size = float((dy.double().abs() * 8).sum())     # |y| and the terms of its tolerance stay below 8
        assert abs(quotient - quotient64) <= 2 * 144 * U * size / (2 * h)
        assert abs(ours_slope - slope64) <= 1e-4 * float((leaf.grad * v.double()).abs().sum())
        assert abs(quotient - ours_slope) <= abs(quotient64 - slope64) + 144 * U * size / h + 1e-4 * float((leaf.grad * v.double()).abs().sum())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hw", [(13, 13), (104, 100)], ids=ids)
def test_a_far_mean_keeps_the_variance(cuda, hw, dtype):
    """Values at 300 +- 1 (fp32 squares about zero would keep a hundredth of the variance's digits), the first pixel far out."""
    g = torch.Generator().manual_seed(2)
    x = 300 + torch.randn(2, *hw, 64, generator=g)
    x[:, 0, 0] = 340.0
    x = x.to(dtype)
    gamma, beta = torch.ones(64), torch.zeros(64)
    _, yv, stats, _ = _forward(cuda, x, None, gamma, beta, 16, "leaky", 1.0)
    _check_forward(x, None, gamma, beta, 16, "leaky", 1.0, yv.interior(), stats)


@pytest.mark.parametrize("hw", [(13, 13), (104, 100)], ids=ids)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
def test_a_bad_value_stays_in_its_image_and_group(cuda, bad, hw):
    x, _, dy, gamma, beta = _inputs((3, *hw, 64, 8), torch.float32, seed=9)
    _, clean, st, _ = _forward(cuda, x, None, gamma, beta, 8)
    xb = x.clone()
    xb[1, 2, 3, 19] = bad          # image 1, group 2
    _, yv, stats, _ = _forward(cuda, xb, None, gamma, beta, 8)
    y, c = yv.interior().cpu(), clean.interior().cpu()
    hit = torch.zeros(3, 1, 1, 64, dtype=torch.bool)
    hit[1, :, :, 16:24] = True
    hit = hit.expand_as(y)
    assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], c[~hit])
    dyb = dy.clone()
    dyb[1, 2, 3, 19] = bad
    dx, dg, db = _backward(cuda, x, dyb, gamma, beta, st, 8, "leaky", 0.1)
    d0, g0, b0 = _backward(cuda, x, dy, gamma, beta, st, 8, "leaky", 0.1)
    assert not torch.isfinite(dx[hit]).any() and torch.equal(dx[~hit], d0[~hit])
    ch = torch.arange(64) == 19
    assert not torch.isfinite(dg[ch]).any() and not torch.isfinite(db[ch]).any()
    assert torch.equal(dg[~ch], g0[~ch]) and torch.equal(db[~ch], b0[~ch])


def test_constant_image_and_zero_gamma(cuda):
    """var = 0: y = act(beta), dx = d's deviation from the group's mean over sqrt(eps); gamma = 0: dx = 0 exactly."""
    x = torch.full((2, 4, 4, 16), 2.5)
    gamma, beta = torch.ones(16), torch.linspace(-1, 1, 16)
    _, yv, stats, _ = _forward(cuda, x, None, gamma, beta, 4)
    _check_forward(x, None, gamma, beta, 4, "leaky", 0.1, yv.interior(), stats)
    dy = torch.randn(2, 4, 4, 16, generator=torch.Generator().manual_seed(4))
    got = _backward(cuda, x, dy, gamma, beta, stats, 4, "leaky", 0.1)
    _check_backward(x, dy, gamma, beta, stats, 4, "leaky", 0.1, got)
    got = _backward(cuda, x, dy, torch.zeros(16), beta, stats, 4, "leaky", 0.1)
    assert float(got[0].abs().max()) == 0.0


@pytest.mark.parametrize("shape", [(4, 13, 13, 256, 32), (2, 104, 104, 64, 32)], ids=ids)
def test_forward_and_backward_together_streams_and_graphs(cuda, shape):
    """A layer's forward and backward as a training step makes them: on a stream of their own the same bits; captured into a graph
    that is replayed with new inputs between other work the same bits as eager calls; the same bits from call to call."""
    from yolo_amd import ops
    N, H, W, C, G = shape
    sets = [_inputs(shape, torch.bfloat16, seed=s) for s in (20, 21, 22)]
    gamma, beta = sets[0][3].to(cuda), sets[0][4].to(cuda)
    xv, rv, dyv = (_view(t, cuda, 1) for t in sets[0][:3])
    yv, dxv = _view(torch.zeros_like(sets[0][0]), cuda, 1), _view(torch.zeros_like(sets[0][0]), cuda, 1)
    stats = torch.empty(2, N, G, device=cuda)
    dg, db = torch.empty(C, device=cuda), torch.empty(C, device=cuda)
    ws = torch.empty(ops.gn_workspace_bytes(N, H, W, C, G, torch.bfloat16), dtype=torch.uint8, device=cuda)

    def both():
        ops.gn_act_fwd(xv, gamma, beta, yv, stats, ws, groups=G, residual=rv)
        ops.gn_act_bwd(dyv, xv, gamma, beta, stats, dxv, dg, db, ws, groups=G)

    def load(s):
        for v, t in zip((xv, rv, dyv), s[:3]):
            v.interior().copy_(t.to(cuda))

    def results():
        torch.cuda.synchronize()
        return [t.clone() for t in (yv.interior(), stats, dxv.interior(), dg, db)]

    want = []
    for s in sets:
        load(s)
        both()
        want.append(results())
        both()
        assert all(torch.equal(a, b) for a, b in zip(results(), want[-1]))
    side = torch.cuda.Stream()
    load(sets[1])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(results(), want[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for i in (2, 0, 1, 2):
        load(sets[i])
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip(results(), want[i]):
            assert torch.equal(a, b), i
        load(sets[(i + 1) % 3])
        both()          # eager work on the same buffers between the replays
        torch.cuda.synchronize()


def test_refusals(cuda):
    from yolo_amd import ops
    from yolo_amd._lib import YoloHipError
    x = torch.zeros(2, 4, 4, 32)
    xv, yv = _view(x, cuda), _view(x, cuda)
    ga, be = torch.ones(32, device=cuda), torch.zeros(32, device=cuda)
    st = torch.zeros(2, 2, 4, device=cuda)
    ws = torch.empty(ops.gn_workspace_bytes(2, 4, 4, 32, 4, torch.float32), dtype=torch.uint8, device=cuda)
    ok = dict(groups=4)
    with pytest.raises(YoloHipError, match="do not divide"):
        ops.gn_act_fwd(xv, ga, be, yv, torch.zeros(2, 2, 5, device=cuda), ws, groups=5)
    with pytest.raises(YoloHipError, match="workspace of"):
        ops.gn_act_fwd(xv, ga, be, yv, st, ws[:64], **ok)
    with pytest.raises(YoloHipError, match="slope"):
        ops.gn_act_fwd(xv, ga, be, yv, st, ws, slope=1.5, **ok)
    with pytest.raises(ValueError, match="activation"):
        ops.gn_act_fwd(xv, ga, be, yv, st, ws, act="tanh", **ok)
    with pytest.raises(ValueError, match="stats"):
        ops.gn_act_fwd(xv, ga, be, yv, torch.zeros(2, 2, 3, device=cuda), ws, **ok)
    with pytest.raises(ValueError, match="gamma"):
        ops.gn_act_fwd(xv, ga[:16], be, yv, st, ws, **ok)
    with pytest.raises(ValueError, match="gamma"):
        ops.gn_act_fwd(xv, ga.double(), be, yv, st, ws, **ok)
    with pytest.raises(ValueError, match="y is"):
        ops.gn_act_fwd(xv, ga, be, _view(x.bfloat16(), cuda), st, ws, **ok)
    with pytest.raises(ValueError, match="residual is"):
        ops.gn_act_fwd(xv, ga, be, yv, st, ws, residual=_view(x[:1], cuda), **ok)
    with pytest.raises(YoloHipError, match="expected 4 x 4"):
        ops.gn_act_fwd(xv, ga, be, _view(torch.zeros(2, 5, 4, 32), cuda), st, ws, **ok)
    with pytest.raises(ValueError, match="does not describe"):
        ops.gn_act_fwd(ops.View(xv.buf, 4, 4, 1, 32), ga, be, yv, st, ws, **ok)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.gn_act_fwd(ops.View(x, 4, 4, 0, 32), ga, be, yv, st, ws, **ok)
    with pytest.raises(ValueError, match="dy is"):
        ops.gn_act_bwd(_view(x.bfloat16(), cuda), xv, ga, be, st, yv, ga.clone(), be.clone(), ws, **ok)
    with pytest.raises(YoloHipError, match="workspace of"):
        ops.gn_act_bwd(yv, xv, ga, be, st, yv, ga.clone(), be.clone(), ws[:64], **ok)
