"""Group normalisation of groups that are constant, or nearly so, far from zero: the sums, the differences from the mean and the
output lose nothing to the mean's size beyond the rounding of the stored fp32 mean itself, whichever kernel the size selects.

Tolerances are sums of roundings (u = 2^-24): as in test_gpu_gn.py, but what goes with the mean is its own rounding alone.
  statistics   mean u (|mean| + 256 max|x - mean|); 1/sqrt(var + eps) 128 u relative
  y            with s = gamma / sqrt(var + eps): u (|mean s| + 256 max|x - mean| |s|) for the mean,
               144 u (|(x - mean) s| + |beta| + |residual|) for the expression, and the output's own rounding
A constant group: its mean is stored exactly and x - mean is zero, so that y is act(beta) [+ residual], 4 u and the output's rounding.
"""
import pytest
import torch

from .test_gpu_gn import OUT, U, _act, ids

pytestmark = pytest.mark.gpu

# one shape for each form of the forward pass: vectors of 16 bytes that a thread of the whole form holds (4, 11, 16, 22), tall slabs,
# chunked passes of two launches and of three; (N, H, W, bytes of a pixel, groups)
FORMS = {"whole4": (2, 13, 13, 128, 8), "whole11": (32, 26, 26, 1024, 32), "whole16": (256, 40, 40, 128, 8),
         "whole22": (256, 46, 45, 128, 8), "tall": (256, 59, 51, 128, 8), "joined": (1, 52, 52, 512, 32),
         "chunked": (4, 208, 208, 256, 8), "chunked_split_group": (2, 31, 30, 8224, 8)}
DTYPES = [torch.float32, torch.bfloat16]


def _case(cuda, form, dtype, residual, seed):
    N, H, W, row, G = FORMS[form]
    C = row // torch.finfo(dtype).bits * 8
    g = torch.Generator(cuda).manual_seed(seed)
    mean = (10 ** (4 * torch.rand(N, G, generator=g, device=cuda) - 1)).to(dtype).float()      # 0.1 to 1000
    mean *= 1 - 2 * torch.randint(0, 2, (N, G), generator=g, device=cuda)
    x = mean.repeat_interleave(C // G, 1).view(N, 1, 1, C).expand(N, H, W, C).to(dtype).contiguous()
    r = torch.randn(N, H, W, C, generator=g, device=cuda).to(dtype) if residual else None
    gamma, beta = (torch.randn(C, generator=g, device=cuda) * 0.3 + k for k in (1, 0))
    return x, mean, r, gamma, beta, G


def _forward(x, r, gamma, beta, G):
    from yolo_amd import ops
    N, H, W, C = x.shape
    view = lambda t: ops.View(t, H, W, 0, C)  # noqa: E731
    y, stats = torch.full_like(x, 7.0), torch.full((2, N, G), -1.0, device=x.device)
    ws = torch.full((ops.gn_workspace_bytes(N, H, W, C, G, x.dtype),), 255, dtype=torch.uint8, device=x.device)
    ops.gn_act_fwd(view(x), gamma, beta, view(y), stats, ws, groups=G, act="leaky", slope=0.1, residual=None if r is None else view(r))
    torch.cuda.synchronize()
    return y, stats


@pytest.mark.parametrize("residual", [False, True], ids=["alone", "residual"])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("form", list(FORMS))
def test_constant_groups(cuda, form, dtype, residual):
    x, mean, r, gamma, beta, G = _case(cuda, form, dtype, residual, 1)
    y, stats = _forward(x, r, gamma, beta, G)
    assert torch.equal(stats[0], mean)
    rs = 1e-5 ** -0.5
    want = _act(beta.double(), "leaky", 0.1) if r is None else _act(beta.double(), "leaky", 0.1) + r.double()
    size = beta.double().abs() if r is None else beta.double().abs() + r.double().abs()
    over = (y.double() - want).abs() / (OUT[dtype] * want.abs() + 4 * U * size)
    assert float(over.max()) <= 1
    assert float((stats[1].double() - rs).abs().max()) <= 128 * U * rs


@pytest.mark.parametrize("residual", [False, True], ids=["alone", "residual"])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("form", list(FORMS))
def test_groups_constant_but_for_a_few_values(cuda, form, dtype, residual):
    """Some values an eighth off, the first pixel's among them in every other image."""
    x, mean, r, gamma, beta, G = _case(cuda, form, dtype, residual, 2)
    N, H, W, C = x.shape
    x[:, H // 2, W // 3] *= 1.125
    x[:, H - 1, :, :: C // G] *= 0.875
    x[::2, 0, 0] *= 1.125
    y, stats = _forward(x, r, gamma, beta, G)
    spread = lambda t: t.repeat_interleave(C // G, 1).view(N, 1, 1, C)  # noqa: E731
    v = x.double().view(N, H * W, G, C // G)
    m = v.mean((1, 3))
    v = v - m.view(N, 1, G, 1)
    far = v.abs().amax((1, 3))
    rs = 1 / (v.square().mean((1, 3)) + 1e-5).sqrt()
    assert ((stats[0].double() - m).abs() <= U * (m.abs() + 256 * far)).all()
    assert ((stats[1].double() - rs).abs() <= 128 * U * rs).all()
    s = gamma.double() * spread(rs)
    t = v.view(N, H, W, C) * s
    want, size = _act(t + beta.double(), "leaky", 0.1), 144 * (t.abs() + beta.double().abs()) + (spread(m).abs() + 256 * spread(far)) * s.abs()
    if r is not None:
        want, size = want + r.double(), size + 144 * r.double().abs()
    over = (y.double() - want).abs() / (OUT[dtype] * want.abs() + U * size)
    assert float(over.max()) <= 1
