"""GroupNorm calls whose statistics, workspace, vectors and views share memory, in part too, are refused before any launch, and so are
gradient norms whose outputs and workspace do (no GPU)."""
import ctypes

import pytest

from yolo_amd import _lib

N, H, W, C, G, BF16 = 2, 4, 4, 64, 8, 1
IMAGES, VEC, STATS = N * H * W * C * 2, C * 4, 2 * N * G * 4


def _call(backward, **moved):
    """The call with memory that nothing shares, but for what ``moved`` gives another address."""
    need = _lib.lib().yolo_gn_workspace_bytes(N, H, W, C, G, BF16)
    size = dict(x=IMAGES, y=IMAGES, r=IMAGES, gamma=VEC, beta=VEC, dgamma=VEC, dbeta=VEC, stats=STATS, ws=need)
    at = {k: (i + 1) << 20 for i, k in enumerate(size)}
    for k, (other, shift) in moved.items():   # "end": the last 16 bytes, "start": the first 16 in front of it
        at[k] = at[other] + {"same": 0, "end": size[other] - 16, "start": 16 - size[k]}[shift]
    v = {k: ctypes.byref(_lib.YoloView(at[k], H, W, 0, C, 0)) for k in "xyr"}
    L = _lib.lib()
    if backward:
        code = L.yolo_gn_act_bwd(v["r"], v["x"], at["gamma"], at["beta"], at["stats"], v["y"], at["dgamma"], at["dbeta"], N, C, G, 0,
                                 0.1, BF16, at["ws"], need, None)
    else:
        code = L.yolo_gn_act_fwd(v["x"], at["gamma"], at["beta"], v["r"], v["y"], at["stats"], N, C, G, 1e-5, 0, 0.1, BF16, at["ws"],
                                 need, None)
    return code, L.yolo_last_error().decode()


FWD = [(a, b) for a in ("stats", "ws") for b in ("x", "y", "r", "gamma", "beta")] + [("stats", "ws"), ("y", "gamma"), ("y", "beta")]
BWD = [(a, b) for a in ("dgamma", "dbeta", "ws") for b in ("x", "y", "r", "gamma", "beta", "stats")]
BWD += [("dgamma", "ws"), ("dbeta", "ws"), ("dgamma", "dbeta"), ("y", "gamma"), ("y", "beta"), ("y", "stats")]


@pytest.mark.parametrize("shift", ["same", "end", "start"])
@pytest.mark.parametrize("backward,pair", [(False, p) for p in FWD] + [(True, p) for p in BWD], ids=str)
def test_shared_memory_is_refused(backward, pair, shift):
    code, message = _call(backward, **{pair[0]: (pair[1], shift)})
    assert code == -1 and ("share memory" in message or "memory of their own" in message), message


@pytest.mark.parametrize("each", [False, True], ids=["all", "each"])
@pytest.mark.parametrize("clip", [False, True], ids=["norm", "clip"])
@pytest.mark.parametrize("norms,coefs,ws", [(0, 0, 4096), (0, 4096, 0), (4096, 0, 0), (16, 4096, 0), (4096, 48, 0)], ids=str)
def test_gradient_norms_over_factors_or_workspace_are_refused(norms, coefs, ws, clip, each):
    L, base = _lib.lib(), 1 << 20
    call = L.yolo_grad_clip if clip else L.yolo_grad_norm
    code = call(2 << 20, 8, 3 << 20 if each else None, 5 if each else 0, 2.0, 1.0, base + norms, base + coefs, base + ws, 64, None)
    assert code == -1 and "share memory" in L.yolo_last_error().decode()
