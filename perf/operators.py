"""Cases for measuring the training operators of the GroupNorm network and of gradient clipping.

Four operators:

* ``gn_fwd``  group normalisation + activation (+ residual) of a pixel-major activation, with the statistics that the
  backward pass reads: what follows every convolution of a network built with MODEL.DARKNET.NORM "GN";
* ``gn_bwd``  its gradient with respect to the input, the weights and the biases;
* ``clip``    the norm of the gradients of many tensors (of all of them together, or of each) and their scaling in place;
* ``step``    the norm of a flat gradient arena and the momentum step of the optimizer on the clipped gradients.

``own`` says which form ``run`` takes: elementary torch operations, or this repository's kernels.  Both take what
``prepare`` gives.  ``exact`` is the operator's definition in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-5
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
LARGEST = 64 * 208 * 208 * 64          # elements of the largest activation
NET = 62_000_000                       # elements of the largest gradient set


# ------------------------------------------------------------------------------------------------------ the cases
def listed():
    gn = lambda name, op, n, h, w, c, groups=32, dtype="bf16", act="leaky", slope=0.1, halo=1, residual=False: dict(  # noqa: E731
        name=name, op=op, n=n, h=h, w=w, c=c, groups=groups, dtype=dtype, act=act, slope=slope, halo=halo, residual=residual)
    return [
        # one 416 x 416 image in inference: the last stage (stride 32), where the call's latency counts
        gn("gn_fwd_b1_13x13x1024", "gn_fwd", 1, 13, 13, 1024, residual=True),
        # a training batch of 64 at 416 x 416: the middle stage (stride 8) ...
        gn("gn_fwd_b64_52x52x256", "gn_fwd", 64, 52, 52, 256, residual=True),
        # ... and the first one (stride 2), two channels to a group
        gn("gn_fwd_b64_208x208x64", "gn_fwd", 64, 208, 208, 64),
        # the fp32 plan on a small odd-sized batch (a 608 x 416 image, stride 32), SiLU, twelve channels to a group
        gn("gn_fwd_b3_19x13x384_f32", "gn_fwd", 3, 19, 13, 384, dtype="f32", act="silu", slope=0.0, halo=0),
        # the same training batch backwards: last stage, middle stage, first stage
        gn("gn_bwd_b64_13x13x1024", "gn_bwd", 64, 13, 13, 1024),
        gn("gn_bwd_b64_52x52x256", "gn_bwd", 64, 52, 52, 256),
        gn("gn_bwd_b64_208x208x64", "gn_bwd", 64, 208, 208, 64),
        # fp32, the stem's output of two images: one channel to a group
        gn("gn_bwd_b2_208x208x32_f32", "gn_bwd", 2, 208, 208, 32, dtype="f32"),
        # every gradient of the network (its 75 convolutions with their norms), clipped by their common norm
        dict(name="clip_network", op="clip", tensors=-1, numel=0, dtype="f32", norm_type=2.0, each=False, max_norm=10.0),
        # the gradients of a head alone, each tensor by its own largest value (all else is frozen)
        dict(name="clip_heads_each", op="clip", tensors=6, numel=261_120, dtype="f32", norm_type=math.inf, each=True, max_norm=1e-3),
        # the optimizer's step of the whole network
        dict(name="step_network", op="step", weights=61_895_776, norms=53_000, norm_type=2.0, max_norm=10.0),
        # the optimizer's step where only the neck and the heads train, an odd number of elements
        dict(name="step_neck", op="step", weights=2_097_155, norms=4_096, norm_type=2.0, max_norm=1.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gn_fwd", "gn_bwd", "gn_fwd", "gn_bwd", "clip", "step"])
    if op == "clip":
        return dict(op=op, tensors=_log(rng, 1, 60), numel=_log(rng, 1, 1_000_000), dtype=rng.choice(["f32", "f32", "bf16"]),
                    norm_type=rng.choice([1.0, 2.0, 2.0, math.inf]), each=rng.random() < 0.5, max_norm=rng.choice([1e-3, 0.1, 1.0, 10.0]))
    if op == "step":
        return dict(op=op, weights=_log(rng, 1000, NET), norms=_log(rng, 16, 50_000), norm_type=rng.choice([1.0, 2.0, 2.0, math.inf]),
                    max_norm=rng.choice([0.1, 1.0, 10.0]))
    per = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 32])            # channels to a group
    groups = rng.choice([8, 16, 32, 32, 32])
    c = per * groups
    h, w = _log(rng, 4, 208), _log(rng, 4, 208)
    if rng.random() < 0.7:
        w = max(4, min(208, int(h * rng.uniform(0.6, 1.7))))     # images are not strips
    n = _log(rng, 1, max(1, min(64, LARGEST // (c * h * w))))
    act = rng.choice(["leaky", "leaky", "silu"])
    return dict(op=op, n=n, h=h, w=w, c=c, groups=groups, dtype=rng.choice(["bf16", "bf16", "f32"]), act=act,
                slope=rng.choice([0.1, 0.1, 0.0, 1.0]) if act == "leaky" else 0.0, halo=rng.choice([0, 1]),
                residual=op == "gn_fwd" and rng.random() < 0.4)


def _network():
    """Elements of the network's trainable tensors: the convolutions of the backbone, the neck and the heads with the weight
    and the bias of each one's norm."""
    convs, cin = [(3, 32, 3)], 32
    for blocks in (1, 2, 8, 8, 4):
        convs += [(cin, 2 * cin, 3)] + [(2 * cin, cin, 1), (cin, 2 * cin, 3)] * blocks
        cin *= 2
    for c, extra in ((512, 1024), (256, 768), (128, 384)):
        convs += [(extra, c, 1), (c, 2 * c, 3), (2 * c, c, 1), (c, 2 * c, 3), (2 * c, c, 1), (c, 2 * c, 3), (2 * c, 255, 1)]
        convs += [(c, c // 2, 1)] if c > 128 else []
    sizes = []
    for i, o, k in convs:
        sizes += [i * o * k * k] + ([o, o] if o != 255 else [o])
    return sizes


# ---------------------------------------------------------------------------------------------------- their inputs
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if case["op"] in ("gn_fwd", "gn_bwd"):
        return _prepare_gn(case, rand)
    if case["op"] == "clip":
        sizes = _network() if case["tensors"] < 0 else [case["numel"] + 3 * i for i in range(case["tensors"])]
        flat = (rand(sum(sizes)) * 0.01).to(DT[case["dtype"]])
        grads = list(flat.split(sizes))                          # as in the engine: one arena, a view for each tensor
        s = dict(case=case, flat=flat, grads=grads)
        if own:
            from yolo_amd.solver import GradientClipper
            s["clipper"] = GradientClipper(grads, "norm" if case["each"] else "full_model", case["max_norm"], case["norm_type"])
        return s
    n = case["weights"] + case["norms"]
    s = dict(case=case, param=rand(n) * 0.05, grad=rand(n) * 0.01, mom=rand(n) * 0.01, lr=0.01, decay=0.0005, momentum=0.9)
    if own:
        from yolo_amd import ops
        from yolo_amd.solver import GradientClipper
        s["clipper"] = GradientClipper([s["grad"]], "full_model", case["max_norm"], case["norm_type"])
        s["blocks"] = ops.sgd_clip_table([(0, case["weights"], 0), (case["weights"], case["norms"], 1)], s["param"].device)
    return s


def _prepare_gn(case, rand):
    n, h, w, c, pad, dt = (case[k] for k in ("n", "h", "w", "c", "halo", "dtype"))
    dt = DT[dt]
    inner = lambda b: b[:, pad:pad + h, pad:pad + w]  # noqa: E731
    buffer = lambda: torch.zeros(n, h + 2 * pad, w + 2 * pad, c, dtype=dt, device="cuda")  # noqa: E731
    x, y = buffer(), buffer()
    inner(x).copy_(rand(n, h, w, c) * (0.5 + rand(c).abs()) + 0.5 * rand(c))   # a convolution's output: channels differ
    s = dict(case=case, x=x, y=y, gamma=1 + 0.2 * rand(c), beta=0.2 * rand(c))
    if case["residual"]:
        s["residual"] = buffer()
        inner(s["residual"]).copy_(rand(n, h, w, c))
    if case["op"] == "gn_fwd":
        s["stats"] = torch.empty(2, n, case["groups"], device="cuda")
    else:                                                        # what the forward pass left
        s["dy"] = buffer()
        inner(s["dy"]).copy_(rand(n, h, w, c) * 0.01)
        r = inner(x).reshape(n, h * w, case["groups"], -1).double()
        mean = r.mean((1, 3), keepdim=True)
        s["stats"] = torch.stack([mean.view(n, -1), ((r - mean).square().mean((1, 3)) + EPS).rsqrt()]).float()
        s["dgamma"], s["dbeta"] = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    if own:
        from yolo_amd import ops
        s["workspace"] = torch.empty(ops.gn_workspace_bytes(n, h, w, c, case["groups"], dt), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return {"gn_fwd": _own_gn_fwd, "gn_bwd": _own_gn_bwd, "clip": _own_clip, "step": _own_step}[case["op"]](state, case)
    return {"gn_fwd": _plain_gn_fwd, "gn_bwd": _plain_gn_bwd, "clip": _plain_clip, "step": _plain_step}[case["op"]](state, case)


def _inner(buf, case):
    p = case["halo"]
    return buf[:, p:p + case["h"], p:p + case["w"]]


def _own_gn_fwd(s, case):
    from yolo_amd import ops
    v = lambda b: ops.View(b, case["h"], case["w"], case["halo"], case["c"])  # noqa: E731
    ops.gn_act_fwd(v(s["x"]), s["gamma"], s["beta"], v(s["y"]), s["stats"], s["workspace"], groups=case["groups"], eps=EPS,
                   act=case["act"], slope=case["slope"], residual=v(s["residual"]) if case["residual"] else None)
    return {"y": _inner(s["y"], case), "stats": s["stats"]}


def _own_gn_bwd(s, case):
    from yolo_amd import ops
    v = lambda b: ops.View(b, case["h"], case["w"], case["halo"], case["c"])  # noqa: E731
    ops.gn_act_bwd(v(s["dy"]), v(s["x"]), s["gamma"], s["beta"], s["stats"], v(s["y"]), s["dgamma"], s["dbeta"], s["workspace"],
                   groups=case["groups"], act=case["act"], slope=case["slope"])
    return {"dx": _inner(s["y"], case), "dgamma": s["dgamma"], "dbeta": s["dbeta"]}


def _own_clip(s, case):
    return {"norm": s["clipper"].clip_(), "grads": s["flat"]}


def _own_step(s, case):
    from yolo_amd import ops
    norm = s["clipper"].measure()
    ops.sgd_step_clipped(s["param"], s["grad"], s["mom"], s["blocks"], s["lr"], s["decay"], s["lr"], 0.0, s["momentum"],
                         coefs=s["clipper"].coefs)
    return {"norm": norm, "param": s["param"], "momentum": s["mom"]}


def _plain_gn_fwd(s, case):
    n, h, w, c, groups = (case[k] for k in ("n", "h", "w", "c", "groups"))
    x = _inner(s["x"], case).float().reshape(n, h * w, groups, c // groups)
    mean = x.mean((1, 3), keepdim=True)
    xm = x - mean
    invstd = (xm.square().mean((1, 3), keepdim=True) + EPS).rsqrt()
    t = (xm * invstd).view(n, h, w, c) * s["gamma"] + s["beta"]
    t = t * torch.sigmoid(t) if case["act"] == "silu" else torch.where(t > 0, t, t * case["slope"])
    if case["residual"]:
        t = t + _inner(s["residual"], case).float()
    return {"y": t.to(s["x"].dtype), "stats": torch.stack([mean.view(n, groups), invstd.view(n, groups)])}


def _plain_gn_bwd(s, case):
    n, h, w, c, groups = (case[k] for k in ("n", "h", "w", "c", "groups"))
    mean, invstd = (t.repeat_interleave(c // groups, 1).view(n, 1, 1, c) for t in s["stats"])
    xhat = (_inner(s["x"], case).float() - mean) * invstd
    dy = _inner(s["dy"], case).float()
    if case["act"] == "silu":
        t = xhat * s["gamma"] + s["beta"]
        sig = torch.sigmoid(t)
        g = dy * (sig * (1 + t * (1 - sig)))
    else:   # which side of the kink a value is on: in 64 bits, where 32 would take the wrong one next to it
        t = (_inner(s["x"], case).double() - mean) * invstd.double() * s["gamma"] + s["beta"]
        g = torch.where(t > 0, dy, dy * case["slope"])
    dbeta = g.sum((1, 2))
    dgamma = (g * xhat).sum((1, 2))
    count = h * w * (c // groups)
    spread = lambda t: ((t * s["gamma"]).view(n, groups, -1).sum(2) / count).repeat_interleave(c // groups, 1).view(n, 1, 1, c)  # noqa: E731
    dx = invstd * (g * s["gamma"] - spread(dbeta) - xhat * spread(dgamma))
    return {"dx": dx.to(s["x"].dtype), "dgamma": dgamma.sum(0), "dbeta": dbeta.sum(0)}


def _norm(t, kind):
    t = t.float()
    return t.abs().max() if kind == math.inf else t.abs().sum() if kind == 1.0 else t.square().sum().sqrt()


def _plain_clip(s, case):
    if case["each"]:
        norms = torch.stack([_norm(t, case["norm_type"]) for t in s["grads"]])
        for t, k in zip(s["grads"], (case["max_norm"] / (norms + 1e-6)).clamp(max=1.0)):
            t.copy_(t.float() * k)
        return {"norm": norms, "grads": s["flat"]}
    norm = _norm(s["flat"], case["norm_type"])
    s["flat"].copy_(s["flat"].float() * (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0))
    return {"norm": norm.view(1), "grads": s["flat"]}


def _plain_step(s, case):
    norm = _norm(s["grad"], case["norm_type"])
    d = s["grad"] * (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    d[:case["weights"]] += s["decay"] * s["param"][:case["weights"]]
    s["mom"].mul_(s["momentum"]).add_(d)
    s["param"].sub_(s["lr"] * s["mom"])
    return {"norm": norm.view(1), "param": s["param"], "momentum": s["mom"]}


# --------------------------------------------------------------------------------------------- what a pass has to do
def work(case):
    if case["op"] in ("gn_fwd", "gn_bwd"):
        m = case["n"] * case["h"] * case["w"] * case["c"]
        es = 4 if case["dtype"] == "f32" else 2
        tensors = (3 if case["residual"] else 2) if case["op"] == "gn_fwd" else 3
        return {"bytes": tensors * m * es + 8 * case["n"] * case["groups"] + (8 if case["op"] == "gn_fwd" else 16) * case["c"],
                "flops": (9 if case["op"] == "gn_fwd" else 18) * m}
    if case["op"] == "clip":
        m = sum(_network()) if case["tensors"] < 0 else sum(case["numel"] + 3 * i for i in range(case["tensors"]))
        return {"bytes": 2 * m * (4 if case["dtype"] == "f32" else 2), "flops": 3 * m}
    m = case["weights"] + case["norms"]
    return {"bytes": 5 * 4 * m, "flops": 8 * m}


# -------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "clip":
        return _exact_clip(s, case)
    if case["op"] == "step":
        g = s["grad"].double()
        norm = torch.linalg.vector_norm(g, case["norm_type"])
        g = g * min(1.0, case["max_norm"] / (float(norm) + 1e-6))
        w = s["param"].double()
        decay = torch.zeros_like(w)
        decay[:case["weights"]] = s["decay"]
        mom = s["momentum"] * s["mom"].double() + g + decay * w
        return {"norm": norm.view(1), "param": w - s["lr"] * mom, "momentum": mom}
    # rows of one (image, group) each
    n, h, w, c, groups = (case[k] for k in ("n", "h", "w", "c", "groups"))
    rows = lambda t: t.view(n, h, w, groups, -1).permute(0, 3, 1, 2, 4).reshape(n * groups, h * w, -1)  # noqa: E731
    back = lambda t: t.view(n, groups, h, w, -1).permute(0, 2, 3, 1, 4).reshape(n, h, w, c)  # noqa: E731
    one = lambda t: t.double().view(1, groups, 1, -1).expand(n, -1, -1, -1).reshape(n * groups, 1, -1)  # noqa: E731
    x = rows(_inner(s["x"], case).double())
    gamma, beta = one(s["gamma"]), one(s["beta"])
    if case["op"] == "gn_fwd":
        mean = x.mean((1, 2), keepdim=True)
        invstd = 1 / torch.sqrt(((x - mean) ** 2).mean((1, 2), keepdim=True) + EPS)
        t = (x - mean) * invstd * gamma + beta
        y = t / (1 + torch.exp(-t)) if case["act"] == "silu" else t.clamp(min=0) + case["slope"] * t.clamp(max=0)
        y = back(y)
        if case["residual"]:
            y = y + _inner(s["residual"], case).double()
        return {"y": y, "stats": torch.stack([mean.view(n, groups), invstd.view(n, groups)])}
    mean, invstd = (t.double().view(n * groups, 1, 1) for t in s["stats"])
    xhat = (x - mean) * invstd
    t = xhat * gamma + beta
    if case["act"] == "silu":
        e = torch.exp(-t)
        slope = (1 + e + t * e) / (1 + e) ** 2
    else:
        slope = (t > 0).double() * (1 - case["slope"]) + case["slope"]
    d = rows(_inner(s["dy"], case).double()) * slope
    up = d * gamma
    dx = invstd * (up - up.mean((1, 2), keepdim=True) - xhat * (up * xhat).mean((1, 2), keepdim=True))
    per_channel = lambda t: t.sum(1).view(n, c).sum(0)  # noqa: E731
    return {"dx": back(dx), "dgamma": per_channel(d * xhat), "dbeta": per_channel(d)}


def _exact_clip(s, case):
    if not case["each"]:
        norm = torch.linalg.vector_norm(s["flat"].double(), case["norm_type"])
        return {"norm": norm.view(1), "grads": s["flat"].double() * min(1.0, case["max_norm"] / (float(norm) + 1e-6))}
    norms = torch.stack([torch.linalg.vector_norm(t.double(), case["norm_type"]) for t in s["grads"]])
    return {"norm": norms, "grads": torch.cat([t.double() * min(1.0, case["max_norm"] / (float(m) + 1e-6)) for t, m in zip(s["grads"], norms)])}
