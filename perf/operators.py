"""Cases that time the gradient-conditioning operators of the optimizer path.

Four operators work on the list of a model's gradient tensors between the
backward pass and the end of the optimizer step:

* ``norm``       the global norm over all tensors (2-norm or largest magnitude);
* ``clip_norm``  the same norm, then every tensor scaled by
                 ``min(1, max_norm / (norm + 1e-6))`` in place;
* ``clip_value`` every value bounded to ``[-clip_value, clip_value]`` in place;
* ``lamb``       one LAMB step (moments, trust ratio for each tensor, update),
                 with the global norm clipped inside it where the case says so.

The tensors of a case are views into one arena, so that whole results come back
as few outputs: ``flat`` puts them next to each other, as ``FlatParamSpace``
does, ``padded`` leaves one to seven unused values between them, which shifts
every tensor's alignment and shows a write outside of a tensor.
"""

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BETA1, BETA2, EPS = 0.9, 0.999, 1e-6
# the bounds shrink a little from pass to pass, as a bound that follows the
# training's running norm does: otherwise the first pass on a state would be
# the only one that clips
ANNEAL = 0.999


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------

def _resnet(blocks, bottleneck, width=64):
    """(numel, is matrix-like) of an encoder's parameters, in module order."""
    out = [(3 * 64 * 49, True), (64, False), (64, False)]
    cin, expansion = 64, 4 if bottleneck else 1
    for stage, count in enumerate(blocks):
        planes = 64 << stage
        mid = planes * width // 64
        for i in range(count):
            cout = planes * expansion
            convs = ([(cin, mid, 1), (mid, mid, 9), (mid, cout, 1)]
                     if bottleneck else [(cin, planes, 9),
                                         (planes, planes, 9)])
            if i == 0 and (stage > 0 or cin != cout):
                convs.append((cin, cout, 1))
            for a, b, taps in convs:
                out += [(a * b * taps, True), (b, False), (b, False)]
            cin = cout
    return out, cin


def _mlp(inner, latent, outer):
    return [(inner * latent, True), (latent, False), (latent, False),
            (latent, False), (latent * outer, True), (outer, False)]


def _heads(features):
    return _mlp(features, 4096, 256) + _mlp(256, 4096, 256)


def _model(name):
    if name == "probe":  # the linear classifier alone
        return [(2048 * 1000, True), (1000, False)]
    if name == "heads":  # projector and predictor of a 2048-wide encoder
        return _heads(2048)
    encoder, features = {
        "resnet18": lambda: _resnet((2, 2, 2, 2), False),
        "resnet50": lambda: _resnet((3, 4, 6, 3), True),
        "resnet200": lambda: _resnet((3, 24, 36, 3), True),
        "wide_resnet50_2": lambda: _resnet((3, 4, 6, 3), True, 128),
    }[name]()
    return (encoder + _heads(features)
            + [(features * 1000, True), (1000, False)])


def _sizes(case):
    """The case's tensors: a model of this framework, or drawn lengths."""
    if case["model"] != "drawn":
        return _model(case["model"])
    rng = random.Random(case["split"])
    weights = [rng.lognormvariate(0.0, 2.0) for _ in range(case["tensors"])]
    scale = case["total"] / sum(weights)
    sizes = [int(w * scale) for w in weights]
    sizes[rng.randrange(len(sizes))] += case["total"] - sum(sizes)
    return [(n, rng.random() < 0.4) for n in sizes]


def listed():
    return [
        # logging the gradient norm of a linear probe that is trained alone:
        # little data, the call's own latency counts
        {"name": "norm probe fp32", "op": "norm", "model": "probe",
         "dtype": "fp32", "layout": "flat", "norm_type": 2.0},
        # the default encoder with its heads, gradients in the flat buffer
        {"name": "norm resnet50 fp32", "op": "norm", "model": "resnet50",
         "dtype": "fp32", "layout": "flat", "norm_type": 2.0},
        # many small tensors of a deep encoder, half-precision gradients
        {"name": "norm resnet200 bf16", "op": "norm", "model": "resnet200",
         "dtype": "bf16", "layout": "padded", "norm_type": 2.0},
        # the largest magnitude, as a guard before a cast to half precision
        {"name": "norm wide50 fp16 inf", "op": "norm",
         "model": "wide_resnet50_2", "dtype": "fp16", "layout": "padded",
         "norm_type": math.inf},
        # only the heads are trained: a dozen tensors
        {"name": "clip norm heads fp32", "op": "clip_norm", "model": "heads",
         "dtype": "fp32", "layout": "flat", "norm_type": 2.0, "bites": True},
        # every step of a clipped run of the default encoder
        {"name": "clip norm resnet50 fp32", "op": "clip_norm",
         "model": "resnet50", "dtype": "fp32", "layout": "flat",
         "norm_type": 2.0, "bites": True},
        {"name": "clip norm resnet200 bf16", "op": "clip_norm",
         "model": "resnet200", "dtype": "bf16", "layout": "padded",
         "norm_type": 2.0, "bites": True},
        # a bound that is not reached, as in most steps of a settled run
        {"name": "clip norm resnet18 idle", "op": "clip_norm",
         "model": "resnet18", "dtype": "fp32", "layout": "flat",
         "norm_type": 2.0, "bites": False},
        # the engine's clipping by value, small and half-precision encoders
        {"name": "clip value resnet18 fp32", "op": "clip_value",
         "model": "resnet18", "dtype": "fp32", "layout": "flat"},
        {"name": "clip value resnet50 fp16", "op": "clip_value",
         "model": "resnet50", "dtype": "fp16", "layout": "padded"},
        # large-batch training with LAMB: the default encoder, and the deepest
        # one with the global norm clipped in the same step
        {"name": "lamb resnet50 fp32", "op": "lamb", "model": "resnet50",
         "dtype": "fp32", "layout": "flat", "step": 1000, "clip": False},
        {"name": "lamb resnet200 clipped", "op": "lamb",
         "model": "resnet200", "dtype": "fp32", "layout": "flat",
         "step": 0, "clip": True},
    ]


def draw(rng):
    op = rng.choice(["norm", "clip_norm", "clip_value", "lamb"])
    tensors = int(math.exp(rng.uniform(0.0, math.log(400))))
    total = int(math.exp(rng.uniform(math.log(100), math.log(60e6))))
    case = {"op": op, "model": "drawn", "tensors": tensors, "total": total,
            "split": rng.randrange(1 << 30),
            "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]),
            "layout": rng.choice(["flat", "padded"])}
    if op in ("norm", "clip_norm"):
        case["norm_type"] = rng.choice([2.0, 2.0, math.inf])
    if op == "clip_norm":
        case["bites"] = rng.random() < 0.75
    if op == "lamb":
        case["step"] = rng.choice([0, 1, 30, 5000])
        case["clip"] = rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _spans(case):
    rng = random.Random(len(case["layout"]))
    spans, at = [], 0
    for n, _ in _sizes(case):
        if case["layout"] == "padded":
            at += rng.randint(1, 7)
        spans.append((at, n))
        at += n
    return spans, at


def prepare(case, seed):
    spans, total = _spans(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lengths = torch.tensor([n for _, n in spans], device="cuda")
    place = torch.tensor([a for a, _ in spans], device="cuda")

    def spread(values, rest):
        """One value for each tensor, over the tensor's part of the arena."""
        out = torch.full((total,), rest, device="cuda")
        tensor = torch.repeat_interleave(
            torch.arange(len(spans), device="cuda"), lengths)
        first = (torch.cumsum(lengths, 0) - lengths)[tensor]
        index = place[tensor] + torch.arange(len(tensor), device="cuda") \
            - first
        out[index] = values[tensor]
        return out

    def normal():
        return torch.randn(total, generator=gen, device="cuda")

    # a layer's gradients share a magnitude, layers differ by a thousand
    level = 10 ** torch.empty(len(spans), device="cuda").uniform_(
        -4, -1, generator=gen)
    scale = spread(level, 1.0)
    dtype = DTYPES[case["dtype"]]
    grad = (normal() * scale).to(dtype)
    views = [grad[a:a + n] for a, n in spans]
    state = {"op": case["op"], "arena": grad, "grads": views}
    if "norm_type" in case:
        state["norm_type"] = case["norm_type"]
    if case["op"] == "clip_norm":
        flat = torch.cat(views).double()
        size = (flat.abs().max() if case["norm_type"] == math.inf
                else flat.square().sum().sqrt()).item()
        # rounded to a number that a person would set
        state["bound"] = float("%.1g" % (
            size / 4 if case["bites"] else size * 1e9)) or 1.0
        state["anneal"] = ANNEAL if case["bites"] else 1.0
    if case["op"] == "clip_value":
        state["bound"], state["anneal"] = 0.02, ANNEAL
    if case["op"] == "lamb":
        fresh = case["step"] == 0
        # bias and norm parameters: near zero or one, weights near 1/sqrt(fan)
        matrix = torch.tensor([m for _, m in _sizes(case)], device="cuda")
        param = normal() * spread(torch.where(matrix, 0.03, 0.3), 1.0)
        first = torch.zeros_like(param) if fresh \
            else normal() * scale * 0.3
        second = torch.zeros_like(param) if fresh \
            else scale.square() * (0.1 + normal().square())
        for key, arena in (("param", param), ("first", first),
                           ("second", second)):
            state[key + "_arena"] = arena
            state[key + "s"] = [arena[a:a + n] for a, n in spans]
        state["decay"] = [1e-2 if m else 0.0 for _, m in _sizes(case)]
        state["step"] = case["step"]
        state["lr"] = 1e-4
        state["max_grad_norm"] = 1.0 if case["clip"] else 0.0
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _joined(tensors):
    return torch.cat(tensors).float()


def _norm(flat, norm_type):
    if norm_type == math.inf:
        return flat.abs().max()
    return flat.square().sum(dtype=torch.float64).sqrt()


def _factor(norm, bound):
    return torch.clamp(bound / (norm + 1e-6), max=1.0).float()


def _write_back(tensors, flat):
    parts = flat.to(tensors[0].dtype).split([t.numel() for t in tensors])
    [t.copy_(x) for t, x in zip(tensors, parts)]


def _plain_lamb(s, step):
    sizes = [t.numel() for t in s["grads"]]
    ends = torch.tensor(sizes, device="cuda").cumsum(0)
    tensor = torch.bucketize(
        torch.arange(sum(sizes), device="cuda"), ends, right=True)
    p, g, m, v = (_joined(s[k]) for k in ("params", "grads", "firsts",
                                          "seconds"))

    def norms(flat):
        return torch.stack([x.square().sum(dtype=torch.float64)
                            for x in flat.split(sizes)]).sqrt()

    if s["max_grad_norm"] > 0:
        g = g * _factor(_norm(g, 2.0), s["max_grad_norm"])
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    u = (m / (1 - BETA1 ** step)) / ((v / (1 - BETA2 ** step)).sqrt() + EPS)
    u = u + torch.tensor(s["decay"], device="cuda")[tensor] * p
    p_norm, u_norm = norms(p), norms(u)
    trust = torch.where((p_norm > 0) & (u_norm > 0), p_norm / u_norm, 1.0)
    p = p - s["lr"] * trust.float()[tensor] * u
    _write_back(s["params"], p)
    _write_back(s["firsts"], m)
    _write_back(s["seconds"], v)


def run(state):
    s = state
    op, grads = s["op"], s["grads"]
    if own:
        from byol_amd import ops
    if op == "norm":
        if own:
            return ops.global_grad_norm(grads, s["norm_type"])
        return _norm(_joined(grads), s["norm_type"]).float()
    if op == "clip_norm":
        bound = s["bound"]
        s["bound"] *= s["anneal"]
        if own:
            norm = ops.clip_grads_by_norm_(grads, bound, s["norm_type"])
        else:
            flat = _joined(grads)
            norm = _norm(flat, s["norm_type"])
            _write_back(grads, flat * _factor(norm, bound))
        return {"norm": norm.float(), "grads": s["arena"]}
    if op == "clip_value":
        bound = s["bound"]
        s["bound"] *= s["anneal"]
        if own:
            ops.clip_grads_by_value_(grads, bound)
        else:
            _write_back(grads, _joined(grads).clamp(-bound, bound))
        return s["arena"]
    s["step"] += 1
    if own:
        ops.fused_lamb_step(
            s["params"], grads, s["firsts"], s["seconds"], step=s["step"],
            lr=s["lr"], betas=(BETA1, BETA2), eps=EPS,
            weight_decay=s["decay"], max_grad_norm=s["max_grad_norm"])
    else:
        _plain_lamb(s, s["step"])
    return {"params": s["param_arena"], "exp_avg": s["first_arena"],
            "exp_avg_sq": s["second_arena"]}


# ---------------------------------------------------------------------------
# cost and the value in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    n = sum(k for k, _ in _sizes(case))
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        return {"bytes": n * size, "flops": 2 * n}
    if case["op"] == "clip_norm":
        # nothing changes, and nothing has to be written, below the bound
        return {"bytes": n * size * (2 if case["bites"] else 1),
                "flops": 3 * n}
    if case["op"] == "clip_value":
        return {"bytes": n * size * 2, "flops": 2 * n}
    # parameters and both moments read and written, gradients read
    return {"bytes": n * (24 + size), "flops": 20 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] != "lamb":
        values = s["arena"].double()
        inside = torch.zeros(values.numel(), dtype=torch.bool, device="cuda")
        for a, n in _spans(case)[0]:
            inside[a:a + n] = True
        if case["op"] == "clip_value":
            over = inside & (values.abs() > s["bound"])
            values[over] = torch.sign(values[over]) * s["bound"]
            return values
        inner = values[inside]
        norm = torch.linalg.vector_norm(inner, s["norm_type"])
        if case["op"] == "norm":
            return norm
        if norm.item() + 1e-6 > s["bound"]:
            values[inside] = inner / (norm + 1e-6) * s["bound"]
        return {"norm": norm, "grads": values}
    out = {k: s[k + "_arena"].double() for k in ("param", "first", "second")}
    step, shrink = case["step"] + 1, 1.0
    if s["max_grad_norm"] > 0:
        total = math.sqrt(sum(
            t.double().pow(2).sum().item() for t in s["grads"]))
        shrink = min(1.0, s["max_grad_norm"] / (total + 1e-6))
    for (a, n), grad, decay in zip(_spans(case)[0], s["grads"], s["decay"]):
        p, m, v = (out[k][a:a + n] for k in ("param", "first", "second"))
        g = grad.double() * shrink
        m.lerp_(g, 1 - BETA1)
        v.lerp_(g.pow(2), 1 - BETA2)
        rate = m.div(1 - BETA1 ** step).div_(
            v.div(1 - BETA2 ** step).sqrt_().add_(EPS)).add_(p, alpha=decay)
        p_size = torch.linalg.vector_norm(p).item()
        u_size = torch.linalg.vector_norm(rate).item()
        ratio = p_size / u_size if p_size > 0 and u_size > 0 else 1.0
        p.sub_(rate, alpha=s["lr"] * ratio)
    return {"params": out["param"], "exp_avg": out["first"],
            "exp_avg_sq": out["second"]}
