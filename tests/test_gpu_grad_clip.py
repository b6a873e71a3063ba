"""Gradient norms, clipping and the clipped momentum step against the formulas in 64 bits.

Tolerances in roundings u = 2^-24: a norm is a 64-bit sum rounded once (2 u allowed); a factor adds the roundings of its sum and
quotient (4 u), a clipped gradient that of its product (6 u), plus 2^-8 relative where it is stored in bf16; the step's
momentum adds two products and two sums: 8 u of the sum of its terms' sizes.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SETS = {"one": [1], "small": [3, 1, 255, 0, 5], "ragged": [4097, 70001, 33, 16384, 16385, 1023], "empty": [0, 0],
        "many": [17 + 13 * i for i in range(300)], "large": [5_000_011, 12]}


def _tensors(cuda, sizes, dtype, seed=0, scale=0.1):
    """Views of one arena, some of them not at a 16-byte boundary."""
    g = torch.Generator().manual_seed(seed)
    flat = (torch.randn(sum(sizes) + 1, generator=g) * scale).to(dtype)
    arena = flat.to(cuda)
    out, at = [], 1
    for n in sizes:
        out.append(arena[at:at + n])
        at += n
    return arena, flat, out


def _ref_norm(t, kind):
    t = t.double()
    if not t.numel():
        return 0.0
    return float(t.abs().max() if kind == math.inf else t.abs().sum() if kind == 1 else t.square().sum().sqrt())


@pytest.mark.parametrize("each", [False, True], ids=["all", "each"])
@pytest.mark.parametrize("kind", [1.0, 2.0, math.inf], ids=["l1", "l2", "inf"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("name", list(SETS))
def test_norm_and_clip(cuda, name, dtype, kind, each):
    from yolo_amd.solver import GradientClipper
    sizes = SETS[name]
    arena, flat, grads = _tensors(cuda, sizes, dtype)
    parts = [t.double() for t in flat[1:].split(sizes)]
    want = [_ref_norm(p, kind) for p in parts] if each else [_ref_norm(flat[1:], kind)]
    max_norm = 0.5 * (sorted(want)[len(want) // 2] or 1.0)
    c = GradientClipper(grads, "norm" if each else "full_model", max_norm, kind)
    norms = c.measure().double().cpu()
    assert torch.equal(arena.cpu(), flat)      # measuring writes nothing
    want = torch.tensor(want, dtype=torch.float64)
    assert ((norms - want).abs() <= 2 * U * want).all()
    k = (max_norm / (want + 1e-6)).clamp(max=1.0)
    assert ((c.coefs.double().cpu() - k).abs() <= 4 * U * k).all()
    again = c.clip_()
    assert torch.equal(again.double().cpu(), norms)
    got = arena.double().cpu()
    assert float(got[0]) == float(flat[0])     # the element in front of the first tensor
    ref = torch.cat([p * (k[i] if each else k[0]) for i, p in enumerate(parts)])
    tol = (6 * U + (2.0 ** -8 if dtype == torch.bfloat16 else 0)) * ref.abs()
    assert ((got[1:] - ref).abs() <= tol).all()


def test_mixed_types_layouts_and_separate_tensors(cuda):
    from yolo_amd.solver import GradientClipper, clip_grad_norm_, clip_grad_value_
    g = torch.Generator().manual_seed(3)
    host = [torch.randn(64, 32, 3, 3, generator=g).contiguous(memory_format=torch.channels_last), torch.randn(7, generator=g),
            torch.randn(130, 3, generator=g).bfloat16(), torch.randn(5, 9, generator=g).t()]
    dev = [h.to(cuda) for h in host]
    assert [d.stride() for d in dev] == [h.stride() for h in host]
    want = math.sqrt(sum(float(h.double().square().sum()) for h in host))
    norm = GradientClipper(dev, "full_model", 1.0).clip_()
    assert abs(float(norm) - want) <= 2 * U * want
    for d, h in zip(dev, host):
        ref = h.double() / (want + 1e-6)
        assert ((d.double().cpu() - ref).abs() <= (6 * U + (2.0 ** -8 if d.dtype == torch.bfloat16 else 0)) * ref.abs()).all()
    # the functions torch has
    ps = [torch.nn.Parameter(torch.zeros(n, device=cuda)) for n in (5, 1000, 1)] + [torch.nn.Parameter(torch.zeros(3, device=cuda))]
    for p in ps[:3]:
        p.grad = torch.randn(p.shape, generator=g).to(cuda)
    kept = [p.grad.cpu().clone() for p in ps[:3]]
    total = clip_grad_norm_(ps + [ps[0]], 0.25, 1.0)      # one without a gradient, one listed twice
    want = sum(float(t.double().abs().sum()) for t in kept)
    assert total.shape == () and abs(float(total) - want) <= 2 * U * want
    for p, t in zip(ps, kept):
        ref = t.double() * 0.25 / (want + 1e-6)
        assert ((p.grad.double().cpu() - ref).abs() <= 6 * U * ref.abs()).all()
        p.grad.copy_(t)
    assert ps[3].grad is None
    clip_grad_value_(ps, 0.5)
    for p, t in zip(ps, kept):
        assert torch.equal(p.grad.cpu(), t.clamp(-0.5, 0.5))


def test_values_outside_what_fp32_squares_hold(cuda):
    """2-norms of values whose squares overflow or vanish in fp32, and the values a norm cannot bound."""
    from yolo_amd.solver import GradientClipper
    for scale in (1e30, 1e-30, 1e-41):
        t = (torch.randn(5000, generator=torch.Generator().manual_seed(1)) * scale)
        want = _ref_norm(t, 2.0)
        got = float(GradientClipper([t.to(cuda)], "full_model", 1.0).measure())
        assert abs(got - want) <= 2 * U * want + 2.0 ** -149
    for kind in (1.0, 2.0, math.inf):
        t = torch.randn(9000, device=cuda)
        t[4321] = math.nan
        c = GradientClipper([t, torch.ones(3, device=cuda)], "full_model", 1.0, kind)
        assert math.isnan(float(c.clip_())) and torch.isnan(t).all()
        t = torch.randn(9000, device=cuda)
        t[77] = -math.inf
        c = GradientClipper([t], "full_model", 1.0, kind)
        assert float(c.clip_()) == math.inf and float(c.coefs) == 0.0
        keep = torch.arange(9000, device=cuda) != 77
        assert torch.isnan(t[77]) and float(t[keep].abs().max()) == 0.0
    t = torch.tensor([math.nan, math.inf, -math.inf, 2.0, -0.25], device=cuda)
    GradientClipper([t], "value", 0.5).clip_()
    assert math.isnan(float(t[0])) and t[1:].tolist() == [0.5, -0.5, 0.5, -0.25]


@pytest.mark.parametrize("how", ["full_model", "norm", "value"])
@pytest.mark.parametrize("sizes", [[1], [5, 4096, 3], [70001, 255, 8200, 33], [1_000_003, 64]], ids=lambda s: f"{len(s)}x{s[0]}")
def test_clipped_step(cuda, sizes, how):
    from yolo_amd import ops
    from yolo_amd.solver import GradientClipper
    n = sum(sizes)
    g = torch.Generator().manual_seed(n)
    w, d, m = (torch.randn(n, generator=g) for _ in range(3))
    segs, at = [], 0
    for i, s in enumerate(sizes):
        segs.append((at, s, i % 2))
        at += s
    pd, gd, md = w.to(cuda), d.to(cuda), m.to(cuda)
    clip_value = {"full_model": 0.7, "norm": 0.7, "value": 0.3}[how]
    c = GradientClipper([gd[a:a + s] for a, s, _ in segs] if how == "norm" else [gd], how, clip_value)
    c.measure()
    lr, wd, mu = (0.1, 0.02), (0.01, 0.0), 0.9
    ops.sgd_step_clipped(pd, gd, md, ops.sgd_clip_table(segs, cuda), lr[0], wd[0], lr[1], wd[1], mu, coefs=c.coefs,
                         per_tensor=how == "norm", clip_value=clip_value if how == "value" else None)
    assert torch.equal(gd.cpu(), d)
    total = _ref_norm(d, 2.0)
    for a, s, grp in segs:
        x, dd, mm = w[a:a + s].double(), d[a:a + s].double(), m[a:a + s].double()
        if how == "value":
            dd = dd.clamp(-clip_value, clip_value)
        else:
            dd = dd * min(1.0, clip_value / ((_ref_norm(d[a:a + s], 2.0) if how == "norm" else total) + 1e-6))
        m_ref = mu * mm + dd + wd[grp] * x
        size = (mu * mm).abs() + dd.abs() + (wd[grp] * x).abs()
        w_ref = x - lr[grp] * m_ref
        assert ((md[a:a + s].double().cpu() - m_ref).abs() <= 8 * U * size).all()
        assert ((pd[a:a + s].double().cpu() - w_ref).abs() <= 10 * U * lr[grp] * size + U * (w_ref.abs() + x.abs())).all()


def test_a_factor_of_one_is_the_plain_step(cuda):
    """Nothing to clip: bit for bit sgd_step's result; segments that leave elements out leave them alone."""
    from yolo_amd import ops
    g = torch.Generator().manual_seed(0)
    n = 50_021
    w, d, m = (torch.randn(n, generator=g).to(cuda) for _ in range(3))
    segs = [(0, 20_000, 0), (20_003, 30_000, 1)]
    a, b, am, bm = w.clone(), w.clone(), m.clone(), m.clone()
    ops.sgd_step(a, d, am, *ops.sgd_block_table(segs, cuda), 0.1, 0.01, 0.2, 0.0, 0.9)
    ops.sgd_step_clipped(b, d, bm, ops.sgd_clip_table(segs, cuda), 0.1, 0.01, 0.2, 0.0, 0.9, coefs=torch.ones(1, device=cuda))
    assert torch.equal(a, b) and torch.equal(am, bm)
    assert torch.equal(b[20_000:20_003], w[20_000:20_003]) and torch.equal(b[50_003:], w[50_003:])


def test_norm_clip_and_step_in_a_graph(cuda):
    """Norm + step captured, replayed over new gradients with eager work between: each replay as the eager call, twice the same."""
    from yolo_amd import ops
    from yolo_amd.solver import GradientClipper
    n = 300_007
    g = torch.Generator().manual_seed(8)
    grads = [torch.randn(n, generator=g) for _ in range(3)]
    w0, m0 = torch.randn(n, generator=g).to(cuda), torch.randn(n, generator=g).to(cuda)
    w, m, d = w0.clone(), m0.clone(), grads[0].to(cuda)
    clipper, table = GradientClipper([d], "full_model", 1.0), ops.sgd_clip_table([(0, 200_000, 0), (200_000, n - 200_000, 1)], cuda)
    own = GradientClipper([d], "full_model", 0.5)

    def step():
        clipper.measure()
        ops.sgd_step_clipped(w, d, m, table, 0.1, 0.01, 0.1, 0.0, 0.9, coefs=clipper.coefs)
        own.clip_()

    def run(i, go):
        w.copy_(w0)
        m.copy_(m0)
        d.copy_(grads[i].to(cuda))
        torch.cuda.synchronize()
        go()
        torch.cuda.synchronize()
        return [t.clone() for t in (w, m, d, clipper.norms, own.norms)]

    want = [run(i, step) for i in range(3)]
    assert all(torch.equal(a, b) for a, b in zip(run(1, step), want[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in (2, 0, 1, 1):
        assert all(torch.equal(a, b) for a, b in zip(run(i, graph.replay), want[i])), i
        run((i + 1) % 3, step)


def test_refusals(cuda):
    from yolo_amd import ops
    from yolo_amd._lib import YoloHipError
    from yolo_amd.solver import GradientClipper
    t = torch.zeros(100, device=cuda)
    with pytest.raises(ValueError, match="share memory"):
        ops.grad_table([t[:60], t[50:]])
    with pytest.raises(ValueError, match="share memory"):
        ops.grad_table([t, t])
    with pytest.raises(ValueError, match="one run of memory"):
        ops.grad_table([t[::2]])
    with pytest.raises(ValueError, match="one run of memory"):
        ops.grad_table([torch.zeros(1, device=cuda).expand(5)])
    with pytest.raises(ValueError, match="dtype"):
        ops.grad_table([t.half()])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.grad_table([t.cpu()])
    with pytest.raises(ValueError, match="no tensors"):
        GradientClipper([], "norm", 1.0)
    with pytest.raises(ValueError, match="clipping by"):
        GradientClipper([t], "agc", 1.0)
    with pytest.raises(ValueError, match="NORM_TYPE"):
        GradientClipper([t], "norm", 1.0, 3.0)
    with pytest.raises(ValueError, match="CLIP_VALUE"):
        GradientClipper([t], "value", -1.0)
    table = ops.grad_table([t])
    with pytest.raises(YoloHipError, match="norm type"):
        ops.grad_norm(table, t[:1], torch.empty(64, dtype=torch.uint8, device=cuda), norm_type=0.5)
    with pytest.raises(YoloHipError, match="workspace of"):
        ops.grad_norm(table, t[:1], torch.empty(4, dtype=torch.uint8, device=cuda))
    with pytest.raises(ValueError, match="norms"):
        ops.grad_norm(table, t[:2], torch.empty(64, dtype=torch.uint8, device=cuda))
    sgd = ops.sgd_clip_table([(0, 50, 0), (50, 50, 1)], cuda)
    one = torch.ones(1, device=cuda)
    with pytest.raises(ValueError, match="covers 100"):
        ops.sgd_step_clipped(t[:96], t[:96].clone(), t[:96].clone(), sgd, 0.1, 0, 0.1, 0, 0.9, coefs=one)
    with pytest.raises(ValueError, match="one of the two"):
        ops.sgd_step_clipped(t, t.clone(), t.clone(), sgd, 0.1, 0, 0.1, 0, 0.9)
    with pytest.raises(ValueError, match="coefs"):
        ops.sgd_step_clipped(t, t.clone(), t.clone(), sgd, 0.1, 0, 0.1, 0, 0.9, coefs=one, per_tensor=True)
    with pytest.raises(ValueError, match="two segments"):
        ops.sgd_clip_table([(0, 50, 0), (40, 50, 1)], cuda)
