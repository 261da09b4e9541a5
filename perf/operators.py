"""Cases of the operators that end a training step: the global norm of a list of gradients, clipping by it, and Adam's update.

A list is the parameters of one of this framework's modules, held the way training programs hold them: views of one arena per
quantity (parameters, gradients, first and second moments), each view starting at a multiple of `align` elements (64: an allocator's
or a padded arena's, 1: a packed communication bucket's, where most views are not aligned to anything).  What lies between the views
is zero, stays zero and adds nothing to a norm, so the plain forms work on whole arenas, in a few long operations.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BETAS, EPS = (0.9, 0.999), 1e-8
STEPS_TAKEN = 1000


def _dense_block(cin, grow, cout):
    """Five densely connected 3x3 convolutions with biases."""
    got = []
    for i in range(4):
        got += [(grow, cin + i * grow, 3, 3), (grow,)]
    return got + [(cout, cin + 4 * grow, 3, 3), (cout,)]


def _double_conv(cin, cout, mid=None):
    """Two 3x3 convolutions, each before a batch norm."""
    mid = mid or cout
    return [(mid, cin, 3, 3), (mid,), (mid,), (cout, mid, 3, 3), (cout,), (cout,)]


def shapes(case):
    """The parameters of the module that the case names, in order."""
    if case["module"] == "prior":         # the learned prior (a U-Net between dense input blocks and a 1x1 output)
        chans, dim, depth = case["chans"], case["dim"], case["depth"]
        half = dim // 2
        got = _dense_block(chans, half, half) + [(chans, 3, 3, 3), (chans,)] + _dense_block(chans, half, half)
        for i in range(depth):
            got += _double_conv(dim << i, (dim << (i + 1)) // (2 if i == depth - 1 else 1))
        for i in range(depth):
            cin = dim << (depth - i)
            got += _double_conv(cin, (dim << (depth - i - 1)) // (2 if i < depth - 1 else 1), cin // 2)
        return got + _double_conv(dim, dim) + [(chans, dim, 1, 1), (chans,)]
    f = case["feats"]
    if case["module"] == "dense":         # the RRDB encoder: three dense blocks in each of `blocks`, and its head and tail
        got = [(f, 3, 3, 3), (f,)]
        for _ in range(3 * case["blocks"]):
            got += _dense_block(f, case["grow"], f)
        return got + 4 * [(f, f, 3, 3), (f,)] + [(3, f, 3, 3), (3,)]
    return [(f, 3, 3, 3), (f,)] + (2 * case["blocks"] + 1) * [(f, f, 3, 3), (f,)]      # "residual": the EDSR encoder


def _count(case):
    return sum(math.prod(s) for s in shapes(case))


def listed():
    prior = {"module": "prior", "chans": 27, "dim": 64, "depth": 3}          # the shipped learned prior: 4.6 M in 66 tensors
    dense = {"module": "dense", "feats": 64, "grow": 32, "blocks": 23}       # the shipped RRDB encoder: 16.7 M in 702 tensors
    small = {"module": "residual", "feats": 16, "blocks": 1}                 # a latent module of a few small layers
    odd = {"module": "residual", "feats": 37, "blocks": 2}
    wide = {"module": "residual", "feats": 512, "blocks": 32}                # 153 M: more than the caches hold
    middle = {"module": "residual", "feats": 256, "blocks": 32}              # 38 M
    return [
        # monitoring a step: the norm alone.  A small module, where only latency counts
        {"name": "norm small fp32", "op": "norm", **small, "grads": "fp32", "kind": "l2", "align": 64},
        # ... the module that this framework trains, in its own type
        {"name": "norm prior fp32", "op": "norm", **prior, "grads": "fp32", "kind": "l2", "align": 64},
        # ... many tensors of 16 bits from a packed bucket
        {"name": "norm dense bf16 packed", "op": "norm", **dense, "grads": "bf16", "kind": "l2", "align": 1},
        # ... the largest magnitude of a larger encoder's half-precision gradients, as a check for overflow
        {"name": "max-norm middle fp16", "op": "norm", **middle, "grads": "fp16", "kind": "max", "align": 64},
        # clipping into the buffer that goes on to an optimizer or a collective.  Few, odd and unaligned tensors
        {"name": "clip odd fp32 packed", "op": "clip", **odd, "grads": "fp32", "kind": "l2", "align": 1, "most": 0.1},
        # ... the trained module's
        {"name": "clip prior fp32", "op": "clip", **prior, "grads": "fp32", "kind": "l2", "align": 64, "most": 1.0},
        # ... by the largest magnitude, many tensors of 16 bits
        {"name": "max-clip dense fp16", "op": "clip", **dense, "grads": "fp16", "kind": "max", "align": 64, "most": 0.01},
        # ... the largest list
        {"name": "clip wide bf16", "op": "clip", **wide, "grads": "bf16", "kind": "l2", "align": 64, "most": 1.0},
        # Adam's update, alone and after clipping.  A small module
        {"name": "adam small fp32", "op": "adam", **small, "params": "fp32", "grads": "fp32", "align": 64, "most": 0.0, "decay": 0.0,
         "decoupled": False},
        # ... the trained module, clipped
        {"name": "adam prior fp32 clipped", "op": "adam", **prior, "params": "fp32", "grads": "fp32", "align": 64, "most": 1.0, "decay": 0.0,
         "decoupled": False},
        # ... parameters and gradients of 16 bits with moments of 32, decoupled decay
        {"name": "adam dense bf16 packed", "op": "adam", **dense, "params": "bf16", "grads": "bf16", "align": 1, "most": 0.0, "decay": 0.01,
         "decoupled": True},
        # ... the largest list, clipped
        {"name": "adam wide fp32 clipped", "op": "adam", **wide, "params": "fp32", "grads": "fp32", "align": 64, "most": 1.0, "decay": 0.01,
         "decoupled": True},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    cap = _count({"module": "residual", "feats": 512, "blocks": 32})
    while True:
        case = {"op": rng.choice(["norm", "clip", "adam"]), "module": rng.choice(["prior", "dense", "residual"])}
        if case["module"] == "prior":
            case |= {"chans": rng.choice([3, 6, 27, 96, spread(3, 96)]), "dim": 2 * spread(8, 64), "depth": rng.randint(1, 4)}
        elif case["module"] == "dense":
            case |= {"feats": spread(8, 128), "grow": spread(4, 64), "blocks": spread(1, 23)}
        else:
            case |= {"feats": spread(8, 512), "blocks": spread(1, 32)}
        if _count(case) <= cap:
            break
    case |= {"grads": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "align": rng.choice([1, 2, 16, 64])}
    if case["op"] == "adam":
        case |= {"params": rng.choice(["fp32", case["grads"]]), "most": rng.choice([0.0, spread(1, 1000) / 100]), "decay": rng.choice([0.0, 0.01, 0.1]),
                 "decoupled": rng.random() < 0.5}
    else:
        case["kind"] = rng.choice(["l2", "l2", "max"])
        if case["op"] == "clip":
            case["most"] = spread(1, 1000) / 100
    return case


_ops = None


def _framework():
    global _ops
    if _ops is None:
        from bfsr_amd.ops import HipOps
        _ops = HipOps(DEVICE)
    return _ops


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    shp, align = shapes(case), case["align"]
    sizes = [math.prod(s) for s in shp]
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // align) * align
    total = at
    spans = [b - a for a, b in zip(starts, starts[1:] + [total])]
    # each layer's gradients have a scale of their own, over two decades
    host = torch.Generator().manual_seed(seed)
    scale = (10.0 ** (-3.0 + 2.0 * torch.rand(len(shp), generator=host))).to(DEVICE)
    filled = torch.ones(total, dtype=torch.bool, device=DEVICE)
    if align > 1:
        gaps = [torch.arange(a + n, a + s) for a, n, s in zip(starts, sizes, spans) if s > n]
        if gaps:
            filled[torch.cat(gaps).to(DEVICE)] = False
    scale = torch.repeat_interleave(scale, torch.tensor(spans, device=DEVICE), output_size=total) * filled

    def arena(kind, values):
        return values.to(TYPES[kind])

    def views(a):
        return [a[o:o + n].view(s) for o, n, s in zip(starts, sizes, shp)]

    state = {"case": case}
    grads = arena(case["grads"], torch.randn(total, generator=g, device=DEVICE) * scale)
    state["grads"], lists = grads, {"grads": views(grads)}
    if case["op"] == "clip":
        state["out"] = torch.zeros_like(grads)
        lists["out"] = views(state["out"])
    elif case["op"] == "adam":
        state["params"] = arena(case["params"], torch.randn(total, generator=g, device=DEVICE) * 0.05 * filled)
        state["m"] = 0.3 * torch.randn(total, generator=g, device=DEVICE) * scale
        state["v"] = (0.2 + torch.rand(total, generator=g, device=DEVICE)) * scale * scale
        state["step"] = torch.full((len(shp),), float(STEPS_TAKEN), device=DEVICE)
        state["norm"] = torch.zeros((), device=DEVICE)
        for k in ("params", "m", "v"):
            lists[k] = views(state[k])
    if own:
        ops = _framework()
        if case["op"] == "norm":
            state["plan"] = ops.tensor_list(lists["grads"])
        elif case["op"] == "clip":
            state["plan"] = ops.tensor_list(lists["grads"], out=lists["out"])
        else:
            state["plan"] = ops.adam(lists["params"], lists["grads"], lists["m"], lists["v"], state["step"])
    return state


def _norm(g, kind):
    return g.abs().max() if kind == "max" else torch.sum(g * g, dtype=torch.float64).sqrt().float()


def _share(norm, most):
    """What the gradients are multiplied by so that their norm is at most `most`."""
    return (most / (norm + 1e-6)).clamp(max=1.0)


def _run_own(state):
    case, ops = state["case"], _framework()
    if case["op"] == "norm":
        return [ops.grad_norm(state["plan"], math.inf if case["kind"] == "max" else 2.0)]
    if case["op"] == "clip":
        return [ops.clip_grads(state["plan"], case["most"], math.inf if case["kind"] == "max" else 2.0), state["out"]]
    norm = state["plan"].run(lr=1e-4, betas=BETAS, eps=EPS, weight_decay=case["decay"], decoupled=case["decoupled"], max_norm=case["most"] or None)
    return [state["norm"] if norm is None else norm, state["params"], state["m"], state["v"], state["step"]]


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    g = state["grads"].float()
    if case["op"] == "norm":
        return [_norm(g, case["kind"])]
    if case["op"] == "clip":
        norm = _norm(g, case["kind"])
        state["out"].copy_(g * _share(norm, case["most"]))
        return [norm, state["out"]]
    norm, lr, (b1, b2) = state["norm"], 1e-4, BETAS
    if case["most"]:
        norm = _norm(g, "l2")
        g = g * _share(norm, case["most"])
    state["step"] += 1
    t = state["step"][0].double()
    p, m, v = state["params"].float(), state["m"], state["v"]
    if case["decay"]:
        if case["decoupled"]:
            p = p * (1 - lr * case["decay"])
        else:
            g = g + case["decay"] * p
    m.mul_(b1).add_(g * (1 - b1))
    v.mul_(b2).add_(g * g * (1 - b2))
    size, root = (lr / (1 - b1 ** t)).float(), (1 / (1 - b2 ** t).sqrt()).float()
    state["params"].copy_(p - size * m / (v.sqrt() * root + EPS))
    return [norm, state["params"], m, v, state["step"]]


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    g = s["grads"].double()
    if case["op"] != "adam":
        norm = torch.linalg.vector_norm(g, math.inf if case["kind"] == "max" else 2)
        if case["op"] == "norm":
            return [norm]
        return [norm, g * min(1.0, case["most"] / (float(norm) + 1e-6))]
    norm = torch.zeros((), dtype=torch.float64, device=DEVICE)
    if case["most"]:
        norm = torch.linalg.vector_norm(g)
        g *= min(1.0, case["most"] / (float(norm) + 1e-6))
    x, t = s["params"].double(), STEPS_TAKEN + 1
    if case["decoupled"]:
        x *= 1 - 1e-4 * case["decay"]
    else:
        g += case["decay"] * x
    first = BETAS[0] * s["m"].double() + (1 - BETAS[0]) * g
    second = BETAS[1] * s["v"].double() + (1 - BETAS[1]) * g ** 2
    x -= 1e-4 * (first / (1 - BETAS[0] ** t)) / (torch.sqrt(second / (1 - BETAS[1] ** t)) + EPS)
    return [norm, x, first, second, s["step"].double() + 1]


def work(case):
    n = _count(case)
    width = {"fp32": 4, "fp16": 2, "bf16": 2}
    g = width[case["grads"]]
    if case["op"] == "norm":
        return {"bytes": n * g + 4, "flops": 2 * n}
    if case["op"] == "clip":
        return {"bytes": 2 * n * g + 4, "flops": 3 * n}
    # parameters and both moments are read and written, gradients read
    return {"bytes": n * (2 * width[case["params"]] + g + 16) + 8 * len(shapes(case)), "flops": n * (14 + (3 if case["most"] else 0))}
