"""The shape lists of gn_forms.py take every kernel form and instance, so that a change of the rules that choose one cannot leave
another without a test (no GPU: the name query runs on the host)."""
import pytest

from yolo_amd import _lib, ops

from . import gn_forms

DTYPES = {gn_forms.BF16: "bf16", gn_forms.F32: "float"}


def _names(cases, backward):
    return {ops.gn_kernel_name(*s, dt, residual=r, backward=backward) for dt, s in cases for r in ((False,) if backward else (False, True))}


@pytest.mark.parametrize("dtype", list(DTYPES.values()))
def test_every_form_has_a_shape(dtype):
    fwd, bwd = _names(gn_forms.FORWARD, False), _names(gn_forms.BACKWARD, True)
    plain = lambda names: {n.replace(",stream", "") for n in names}  # noqa: E731
    want = {f"gn_whole_kernel<{dtype},{k},whole>" for k in (1, 2, 4, 6, 8, 11, 16, 22)}
    want |= {f"gn_whole_kernel<{dtype},12,tall>", f"gn_kernel<{dtype},joined>", f"gn_kernel<{dtype},chunked>"}
    assert plain(n for n in fwd if dtype in n) == want
    want = {f"gn_whole_bwd_kernel<{dtype},{k},whole>" for k in (1, 2, 4, 6, 8)}
    want |= {f"gn_whole_bwd_kernel<{dtype},8,tall>", f"gn_bwd_kernel<{dtype},joined>", f"gn_bwd_kernel<{dtype},chunked>"}
    assert plain(n for n in bwd if dtype in n) == want
    for names in (fwd, bwd):   # past the caches and through them
        for form in ("whole", "tall", "joined", "chunked"):
            mine = [n for n in names if dtype in n and f",{form}" in n]
            assert any(",stream" in n for n in mine)
            assert form == "tall" and names is fwd or any(",stream" not in n for n in mine)


def test_a_tall_call_is_one_instance_with_a_residual_and_one_without():
    for dt, s in gn_forms.FORWARD:   # both are run by the GPU tests for every shape; neither leaves the tall form
        names = {ops.gn_kernel_name(*s, dt, residual=r) for r in (False, True)}
        assert len({n.split(",", 1)[1].replace(",stream", "") for n in names}) == 1


def test_name_query_refusals():
    L = _lib.lib()
    import ctypes
    out = ctypes.create_string_buffer(128)
    ask = lambda N=1, H=8, W=8, C=64, G=32, dt=1, buf=out, n=128: L.yolo_gn_kernel_name(N, H, W, C, G, dt, 0, 0, buf, n)  # noqa: E731
    assert ask() == 0 and out.value == b"gn_whole_kernel<bf16,1,whole>"
    for bad in (dict(N=0), dict(H=0), dict(W=-1), dict(C=60), dict(G=7), dict(dt=2), dict(buf=None), dict(n=0), dict(H=1 << 15, W=1 << 15)):
        assert ask(**bad) < 0
    short = ctypes.create_string_buffer(8)
    assert ask(buf=short, n=8) == 0 and short.value == b"gn_whol"
