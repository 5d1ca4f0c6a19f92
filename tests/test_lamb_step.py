"""The fused LAMB step against 64-bit values, its refusals, and the optimizer
and engine paths that call it.

Tolerances, e = 2^-24 (half an fp32 step), from the step's own operations:

* the clipping factor: the norm is rounded to fp32 (e), so is the factor (e);
* g' = factor * g: one more rounding, 3e in all;
* m = b1 m + (1-b1) g': both constants rounded (e each), two products and the
  sum (e each): e (3 |b1 m| + 6 |(1-b1) g'|);
* v alike, with g' twice: e (3 b2 v + 11 (1-b2) g'^2) <= 11 e v;
* u = (m k1) / (sqrt(v k2) + eps) + wd p: with a the first summand, m k1 takes
  2e, the root (11 + 2) / 2 + 1 e, the sum with a rounded eps 2e, the division
  e: 13 e |a| beside m's own error; wd p: 2e; the sum e |u|;
* r = |p| / |u|: |p| is summed in 64 bits; |u| is off by the norm of u's
  errors; lr r takes 2e (lr and the product rounded);
* p - lr r u: product and sum, e each.

The CPU form takes its norms from torch in fp32: n e more for n elements, at
the small sizes where it is tested.  1.01 covers products of these terms.
"""

import math
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from byol_amd import ops
from byol_amd.optim.lamb import LAMB

E = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
B1, B2 = 0.9, 0.999


def make(sizes, device, dtype=torch.float32, seed=0, fresh=False, gap=0):
    """params, grads, exp_avgs, exp_avg_sqs as views of four buffers of
    sevens, `gap` values between the views."""
    gen = torch.Generator().manual_seed(seed)
    total = sum(sizes) + gap * (len(sizes) + 1)
    arenas = [torch.full((total,), 7.0,
                         dtype=dtype if k == 1 else torch.float32)
              for k in range(4)]
    spans, at = [], gap
    for i, n in enumerate(sizes):
        scale = 10.0 ** (-(i % 3))
        values = [torch.randn(n, generator=gen) * 0.1,
                  torch.randn(n, generator=gen) * scale,
                  torch.randn(n, generator=gen) * scale * 0.3,
                  torch.rand(n, generator=gen) * scale ** 2]
        if fresh:
            values[2:] = [torch.zeros(n), torch.zeros(n)]
        for arena, value in zip(arenas, values):
            arena[at:at + n] = value
        spans.append((at, n))
        at += n + gap
    arenas = [a.to(device) for a in arenas]
    return arenas, [[a[s:s + n] for s, n in spans] for a in arenas]


def exact(p, g, m, v, step, lr, eps, wd, factor):
    """The step in 64 bits, and how far p, m and v may be from it."""
    p, g, m, v = (t.detach().cpu().double() for t in (p, g, m, v))
    g = g * factor
    m_old, v_old = m, v
    m = B1 * m_old + (1 - B1) * g
    v = B2 * v_old + (1 - B2) * g * g
    k1 = 1 / (1 - B1 ** step)
    den = (v / (1 - B2 ** step)).sqrt() + eps
    a = m * k1 / den
    u = a + wd * p
    p_norm, u_norm = p.norm(), u.norm()
    r = (p_norm / u_norm).item() if p_norm > 0 and u_norm > 0 else 1.0
    out = p - lr * r * u
    m_off = E * (3 * (B1 * m_old).abs() + 6 * ((1 - B1) * g).abs())
    u_off = m_off * k1 / den + E * (13 * a.abs() + 2 * (wd * p).abs()
                                    + u.abs())
    r_off = (u_off.norm() / u_norm).item() if r != 1.0 else 0.0
    p_off = lr * r * (u_off + u.abs() * (r_off + 3 * E)) + E * out.abs()
    return (out, 1.01 * p_off), (m, 1.01 * m_off), (v, 1.01 * 11 * E * v), \
        lr * r * u.abs()


def check(lists, before, step, lr, eps, decay, factor=1.0, slack=False):
    for i in range(len(lists[0])):
        p, m, v, moved = exact(*(b[i] for b in before), step, lr, eps,
                               decay[i], factor)
        norm_slack = moved * 2 * moved.numel() * E if slack else 0.0
        for name, k, (want, off), more in (("p", 0, p, norm_slack),
                                           ("m", 2, m, 0.0),
                                           ("v", 3, v, 0.0)):
            far = (lists[k][i].detach().cpu().double() - want).abs()
            # 1e-44: results among the subnormal numbers
            assert (far <= off + more + 1e-44).all(), (name, i,
                                                       far.max().item())


LISTS = {
    "one value": [1],
    "one bias": [257],
    "no values among some": [0, 5, 0, 64],
    "around a pack": [3, 4, 5, 7, 8, 9],
    "around a block's share": [8191, 8192, 8193, 16383, 24577],
    "more tensors than a table": [1 + (i * 37) % 300 for i in range(200)],
}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize("step,clip", [(1, 0.0), (1, 0.5), (40, 0.0),
                                       (3000, 0.5), (3000, 1e6)])
@pytest.mark.parametrize("sizes", LISTS.values(), ids=LISTS.keys())
def test_step(device, dtype, step, clip, sizes):
    arenas, lists = make(sizes, device, dtype, fresh=step == 1, gap=1)
    before = [[t.clone() for t in ts] for ts in lists]
    decay = [0.01 * (i % 2) for i in range(len(sizes))]
    norm = torch.cat([g.cpu().double() for g in before[1]]).norm().item()
    ops.fused_lamb_step(*lists, step=step, lr=0.1, weight_decay=decay,
                        max_grad_norm=clip)
    factor = min(1.0, clip / (norm + 1e-6)) if clip else 1.0
    check(lists, before, step, 0.1, 1e-6, decay, factor, device == "cpu")
    for g, b in zip(lists[1], before[1]):
        assert torch.equal(g, b)
    edges = sum(1 for _ in sizes) + 1
    for a in arenas:  # the values between the tensors
        assert int((a == 7).sum()) >= edges


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[5_000_001, 3, 700_000],
                                   [70_000] * 100,
                                   [70_000_003, 32768, 32769, 14_000_000]])
def test_large_lists(sizes):
    _, lists = make(sizes, "cuda", gap=1)
    before = [[t.clone() for t in ts] for ts in lists]
    decay = [0.01] * len(sizes)
    ops.fused_lamb_step(*lists, step=7, lr=0.01, weight_decay=decay)
    check(lists, before, 7, 0.01, 1e-6, decay)
    again = [[t.clone() for t in ts] for ts in before]
    ops.fused_lamb_step(*again, step=7, lr=0.01, weight_decay=decay)
    for a, b in zip(lists, again):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("wait_ticks", [0, 20000])
def test_every_alignment(wait_ticks):
    """Each place in a cache line, lengths around it and around a block's
    share in short and in long lists; parameters aligned unlike moments."""
    for n in (1, 2, 3, 4, 5, 31, 32, 33, 8191, 8192, 8193, 70_000, 163_840,
              196_607):
        sizes = [n + i for i in range(9)] * 3
        arenas, lists = make(sizes, "cuda", gap=3)
        moved = [torch.empty(sum(sizes) + 40, device="cuda") for _ in "gm"]
        for k, buffer in zip((1, 2), moved):  # gradients and exp_avgs moved
            at = 2 * k
            for i, t in enumerate(lists[k]):
                lists[k][i] = buffer[at:at + t.numel()].copy_(t)
                at += t.numel()
        before = [[t.clone() for t in ts] for ts in lists]
        ops.extension().lamb_step(*lists, [0.01] * len(sizes), 3, 0.1, B1, B2,
                                  1e-6, 0.0, None, wait_ticks)
        check(lists, before, 3, 0.1, 1e-6, [0.01] * len(sizes))
        for a in (arenas[0], arenas[3]):
            assert int((a == 7).sum()) >= 3 * (len(sizes) + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("wait_ticks", [0, 1, 1000])
@pytest.mark.parametrize("sizes", [
    [3_000_001, 32768, 32769, 20_000, 5, 100_000] * 3 + [15_000_000],
    [400_001, 8192, 8193, 5, 100_000] * 3])
def test_second_pass_gives_the_same_bits(dtype, wait_ticks, sizes):
    """Blocks that do not wait for the rest of their tensor, or give up, leave
    it to a pass that computes the same."""
    results = []
    for ticks in (20000, wait_ticks):
        _, lists = make(sizes, "cuda", dtype, gap=1)
        ops.extension().lamb_step(*lists, [0.01] * len(sizes), 3, 0.1, B1, B2,
                                  1e-6, 0.0, None, ticks)
        results.append(lists)
    for a, b in zip(*results):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("device", DEVICES)
def test_norms_of_zero(device):
    """A zero parameter, and one whose update is zero, step with ratio 1."""
    _, lists = make([300, 300], device)
    lists[0][0].zero_()
    for k in (1, 2):
        lists[k][1].zero_()
    before = [[t.clone() for t in ts] for ts in lists]
    ops.fused_lamb_step(*lists, step=2, lr=0.1)
    check(lists, before, 2, 0.1, 1e-6, [0.0, 0.0], slack=device == "cpu")
    assert torch.equal(lists[0][1], before[0][1])


@pytest.mark.parametrize("device", DEVICES)
def test_nan_stays_in_its_tensor(device):
    _, lists = make([300, 300], device)
    lists[1][0][7] = math.nan
    before = [[t.clone() for t in ts] for ts in lists]
    ops.fused_lamb_step(*lists, step=2, lr=0.1)
    assert lists[0][0][7].isnan() and lists[2][0][7].isnan()
    assert int(lists[0][0].isnan().sum()) == 1
    check([t[1:] for t in lists], [b[1:] for b in before], 2, 0.1, 1e-6,
          [0.0], slack=device == "cpu")


@pytest.mark.parametrize("device", DEVICES)
def test_layouts(device):
    """Channels-last parameters, and gradients laid out unlike them."""
    torch.manual_seed(0)
    shapes = [(8, 6, 3, 3), (8, 6, 1, 1), (5, 40)]
    def like():
        return [torch.rand(shapes[0]).to(memory_format=torch.channels_last),
                torch.rand(shapes[1]), torch.rand(shapes[2]).t()]
    lists = [[t.to(device) for t in like()] for _ in range(4)]
    lists[1] = [g.contiguous() for g in lists[1]]
    lists[1][1] = lists[1][1].to(memory_format=torch.channels_last)
    before = [[t.clone() for t in ts] for ts in lists]
    ops.fused_lamb_step(*lists, step=3, lr=0.1, weight_decay=0.01)
    check(lists, before, 3, 0.1, 1e-6, [0.01] * 3, slack=device == "cpu")


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    _, (p, g, m, v) = make([64, 8], device)
    before = [t.clone() for t in p + m + v]
    for bad in (dict(step=0), dict(step=1, betas=(1.0, 0.9)),
                dict(step=1, betas=(0.9, -0.1)), dict(step=1, eps=-1.0),
                dict(step=1, max_grad_norm=-1.0),
                dict(step=1, max_grad_norm=math.nan),
                dict(step=1, weight_decay=[0.1])):
        with pytest.raises(ValueError):
            ops.fused_lamb_step(p, g, m, v, lr=0.1, **bad)
    with pytest.raises(ValueError):
        ops.fused_lamb_step(p, g, m[:1], v, step=1, lr=0.1)
    with pytest.raises(ValueError, match="shape"):
        ops.fused_lamb_step(p, [g[0], g[0]], m, v, step=1, lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        ops.fused_lamb_step(p, g, m, m, step=1, lr=0.1)
    with pytest.raises(TypeError):
        ops.fused_lamb_step([t.double() for t in p], g, m, v, step=1, lr=0.1)
    with pytest.raises(TypeError):
        ops.fused_lamb_step(p, g, [t.half() for t in m], v, step=1, lr=0.1)
    for a, b in zip(p + m + v, before):
        assert torch.equal(a, b)


@pytest.mark.skipif(not ops.has_extension(), reason="extension not built")
def test_binding_refuses_before_any_launch():
    """The checks of the binding itself, on CPU tensors: it never launches
    for them."""
    ext = ops.extension()

    def call(p, g, m, v, step=1, norm=None):
        ext.lamb_step(p, g, m, v, [0.0] * len(p), step, 0.1, B1, B2, 1e-6,
                      1.0, norm)

    _, (p, g, m, v) = make([64, 8], "cpu")
    sides = torch.rand(8, 8)
    for bad, text in (
            ((p, g, m, v), "GPU"),
            ((p, g, m, v, 0), "step"),
            ((p, g, m, m), "twice"),
            ((p, g, p, v), "twice"),
            (([p[0], p[0]], [g[0]] * 2, m, v), "strides|twice"),
            ((p, p, m, v), "gradient shares memory"),
            ((p, g, m, [v[1], v[0]]), "strides"),
            (([sides], [sides.clone()], [sides.t().clone(
                memory_format=torch.preserve_format)],
              [torch.rand(8, 8)]), "strides"),
            (([p[0][::2]], [g[0][::2]], [m[0][::2]], [v[0][::2]]), "dense"),
            ((p, g[::-1], m, v), "shape")):
        with pytest.raises(ValueError, match=text):
            call(*bad)
    for bad in (([t.double() for t in p], g, m, v),
                (p, [t.double() for t in g], m, v),
                (p, [g[0], g[1].half()], m, v)):
        with pytest.raises(TypeError):
            call(*bad)


def small_model(device, seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(
        torch.nn.Conv2d(3, 8, 3), torch.nn.BatchNorm2d(8), torch.nn.ReLU(),
        torch.nn.Flatten(), torch.nn.Linear(8 * 36, 5)).to(device)


def train(model, opt, steps=4, seed=3):
    gen = torch.Generator().manual_seed(seed)
    device = next(model.parameters()).device
    for _ in range(steps):
        opt.zero_grad()
        x = torch.randn(16, 3, 8, 8, generator=gen).to(device)
        model(x).square().mean().backward()
        opt.step()


@pytest.mark.parametrize("device", DEVICES)
def test_optimizer_clips_like_clipping_first(device):
    """max_grad_norm inside the step is clipping the gradients before it:
    alike within a rounding of each gradient."""
    from byol_amd.optim import clip_grad_norm_
    grads = [torch.randn(40, 9), torch.randn(9)]
    results = []
    for inside in (True, False):
        params = [torch.nn.Parameter((torch.ones(g.shape) * 0.1).to(device))
                  for g in grads]
        opt = LAMB(params, lr=0.1, weight_decay=0.01,
                   max_grad_norm=0.25 if inside else 0.0)
        assert opt.max_grad_norm == (0.25 if inside else 0.0)
        for p, g in zip(params, grads):
            p.grad = g.to(device)
        if not inside:
            clip_grad_norm_(params, 0.25)
        opt.step()
        results.append(params)
    # the first step's update is g' / (|g'| + eps) in each element
    for a, b in zip(*results):
        assert torch.allclose(a, b, rtol=16 * E, atol=16 * E * 0.1)


@pytest.mark.gpu
def test_optimizer_matches_its_cpu_form():
    """One step from the same gradients; then state dicts move between the
    devices and the next step still agrees."""
    cpu, gpu = small_model("cpu"), small_model("cuda")
    groups = [[{"params": [p for p in m.parameters() if p.ndim > 1],
                "weight_decay": 0.01},
               {"params": [p for p in m.parameters() if p.ndim <= 1],
                "weight_decay": 0.0}] for m in (cpu, gpu)]
    opts = [LAMB(g, lr=0.05, max_grad_norm=1.0) for g in groups]
    gen = torch.Generator().manual_seed(1)
    for turn in range(3):
        for p, q in zip(cpu.parameters(), gpu.parameters()):
            q.data.copy_(p.data)
            p.grad = torch.randn(p.shape, generator=gen)
            q.grad = p.grad.to("cuda")
        for o in opts:
            o.step()
        for p, q in zip(cpu.parameters(), gpu.parameters()):
            # the steps' own bounds, doubled for two forms; sums of up to
            # 1440 elements in fp32 on the CPU
            far = (q.detach().cpu() - p.detach()).abs()
            assert (far <= 2 * (p.detach().abs() * E
                                + 0.05 * p.detach().norm()
                                * (40 + p.numel()) * E)).all()
        opts[1].load_state_dict(opts[0].state_dict())
    assert opts[1].state[next(gpu.parameters())]["step"] == 3


@pytest.mark.gpu
def test_optimizer_mixes_fused_and_single_parameters():
    """A bf16 and a sliced parameter beside fp32 ones: each is stepped."""
    torch.manual_seed(0)
    base = torch.randn(10, 8, device="cuda")
    params = [torch.nn.Parameter(torch.randn(33, device="cuda")),
              torch.nn.Parameter(torch.randn(12, device="cuda").bfloat16()),
              torch.nn.Parameter(base[:, ::2])]
    before = [p.detach().clone() for p in params]
    opt = LAMB(params, lr=0.1, max_grad_norm=10.0)
    for p in params:
        p.grad = torch.randn_like(p)
    opt.step()
    for p, b in zip(params, before):
        assert torch.isfinite(p).all() and not torch.equal(p, b)
        assert opt.state[p]["step"] == 1


@pytest.mark.gpu
def test_devices_do_not_mix():
    _, lists = make([64, 8], "cpu")
    before = [t.clone() for ts in lists for t in ts]
    for k in range(4):
        mixed = [[t.cuda() if i == k else t for t in ts]
                 for i, ts in enumerate(lists)]
        with pytest.raises(ValueError, match="expected"):
            ops.fused_lamb_step(*mixed, step=1, lr=0.1)
    assert all(torch.equal(t, b) for t, b in
               zip((t for ts in lists for t in ts), before))


@pytest.mark.gpu
def test_step_refuses_capture():
    _, lists = make([64], "cuda")
    before = lists[0][0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            ops.fused_lamb_step(*lists, step=1, lr=0.1)
        lists[1][0].mul_(1.0)
    torch.cuda.synchronize()
    assert torch.equal(lists[0][0], before)


@pytest.mark.gpu
def test_two_streams():
    made = [make([300_001, 50], "cuda", seed=s, gap=1)[1] for s in (1, 2)]
    before = [[[t.clone() for t in ts] for ts in lists] for lists in made]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    for lists, s in zip(made, streams):
        with torch.cuda.stream(s):
            ops.fused_lamb_step(*lists, step=5, lr=0.1, max_grad_norm=1.0)
    torch.cuda.synchronize()
    for lists, b in zip(made, before):
        norm = torch.cat([g.cpu().double() for g in b[1]]).norm().item()
        check(lists, b, 5, 0.1, 1e-6, [0.0, 0.0], 1.0 / (norm + 1e-6))


@pytest.mark.gpu
def test_thousands_of_tensors():
    _, lists = make([1 + i % 7 for i in range(3000)], "cuda", gap=1)
    before = [[t.clone() for t in ts] for ts in lists]
    ops.fused_lamb_step(*lists, step=2, lr=0.1)
    some = [[ts[i] for i in range(0, 3000, 59)] for ts in (*lists, *before)]
    check(some[:4], some[4:], 2, 0.1, 1e-6, [0.0] * len(some[0]))


@pytest.mark.gpu
def test_gradients_far_apart():
    """More than 2^32 elements between the gradients of two parameters."""
    sizes = [2000, 40_000, 7]
    _, lists = make(sizes, "cuda", torch.bfloat16, gap=1)
    arena = torch.empty(2 ** 32 + 100_000, dtype=torch.bfloat16,
                        device="cuda")
    for i, at in enumerate((5, 2 ** 32 + 50_000, 3000)):
        lists[1][i] = arena[at:at + sizes[i]].copy_(lists[1][i])
    before = [[t.clone() for t in ts] for ts in lists]
    ops.fused_lamb_step(*lists, step=2, lr=0.1)
    check(lists, before, 2, 0.1, 1e-6, [0.0] * 3)


@pytest.mark.gpu
def test_two_large_steps_at_once():
    """Steps that do not fit the chip together, on two streams: blocks that
    wait for ones that cannot start give up, and the values are the same."""
    sizes = [6_000_000, 70, 5_000_001, 300_000, 6_000_000]
    decay = [0.01] * len(sizes)
    made = [make(sizes, "cuda", seed=s)[1] for s in (1, 2, 1, 2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for step in range(1, 6):
        for lists, s in zip(made, streams):
            with torch.cuda.stream(s):
                ops.fused_lamb_step(*lists, step=step, lr=0.1,
                                    weight_decay=decay)
    torch.cuda.synchronize()
    for step in range(1, 6):
        for lists in made[2:]:
            ops.fused_lamb_step(*lists, step=step, lr=0.1, weight_decay=decay)
    torch.cuda.synchronize()
    for a, b in zip(made[:2], made[2:]):
        for x, y in zip(a, b):
            assert all(torch.equal(t, u) for t, u in zip(x, y))


def engine_args(tmp_path, device, *extra):
    import byol_amd.config as config
    args = config.parse_args([
        "--task", "synthetic_multi_augment_image_folder",
        "--arch", "resnet18", "--representation-size", "512",
        "--head-latent-size", "64", "--projection-size", "32",
        "--batch-size", "8", "--epochs", "1", "--num-replicas", "1",
        "--image-size-override", "32", "--synthetic-classes", "8",
        "--synthetic-train-samples", "32", "--synthetic-test-samples", "8",
        "--workers-per-replica", "0", "--model-dir", str(tmp_path / "m"),
        "--log-dir", str(tmp_path / "l"), *extra])
    args.cuda = device == "cuda"
    args.distributed_rank = 0
    return args


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("extra", [
    ("--optimizer", "lamb", "--lr", "0.001", "--clip-norm", "1.0"),
    ("--clip-norm", "1.0", "--clip", "0.5"),
    ("--clip-norm", "1.0", "--channels-last", "--hip-graph")])
def test_engine_epoch(device, extra, tmp_path):
    """Norm, clipping and step together, as the training engine runs them."""
    from byol_amd.engine import trainer
    from byol_amd.optim import build_optimizer
    args = engine_args(tmp_path, device, *extra)
    torch.manual_seed(0)
    loader, model, grapher = trainer.build_loader_model_grapher(args)
    opt, _ = build_optimizer(model, args)
    for group in opt.param_groups:
        group["lr"] = 0.001  # past the warmup's zero
    before = model.flat_space.flat_params.clone()
    trainer.train(1, model, opt, loader.train_loader, grapher, args)
    flat = model.flat_space.flat_params
    assert torch.isfinite(flat).all() and not torch.equal(flat, before)
    if "lamb" in extra:
        assert opt.max_grad_norm == 1.0
        assert {s["step"] for s in opt.state.values()} == {4}
        # the gradients live in the flat buffer still
        model.flat_space.flat_grads.fill_(2.0)
        assert all((p.grad == 2).all() for p in model.parameters())


@pytest.mark.parametrize("optimizer", ["lamb", "adam", "lars_momentum"])
def test_engine_keeps_gradients_where_they_are_reduced(optimizer, tmp_path):
    from byol_amd.engine import trainer
    from byol_amd.optim import build_optimizer
    from byol_amd.parallel.ddp import FlatDDP
    args = engine_args(tmp_path, "cpu", "--optimizer", optimizer,
                       "--clip-norm", "1.0")
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", "29571"
    dist.init_process_group("gloo", rank=0, world_size=1)
    try:
        loader, model, grapher = trainer.build_loader_model_grapher(args)
        ddp = FlatDDP(model)
        opt, _ = build_optimizer(ddp, args)
        trainer.train(1, ddp, opt, loader.train_loader, grapher, args)
    finally:
        dist.destroy_process_group()
    model.flat_space.flat_grads.fill_(2.0)
    assert all((p.grad == 2).all() for p in model.parameters())


def _replica(rank, port, out_dir, lamb):
    import types

    from byol_amd.models.byol import BYOL
    from byol_amd.optim import build_optimizer, clip_grad_norm_
    from byol_amd.parallel.ddp import FlatDDP
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=2)
    torch.manual_seed(rank)  # FlatDDP aligns the parameters
    model = BYOL(arch="resnet18", base_network_output_size=512,
                 projection_output_size=8, classifier_output_size=3,
                 total_training_steps=10, head_latent_size=16).finalize()
    ddp = FlatDDP(model)
    opt, _ = build_optimizer(ddp, types.SimpleNamespace(
        optimizer="lamb" if lamb else "lars_momentum", lr=0.01,
        weight_decay=1e-4, batch_size=4, num_replicas=2, clip_norm=0.5,
        lr_update_schedule="fixed", epochs=2, warmup=0))
    ddp.train()
    norms = []
    torch.manual_seed(100 + rank)
    for _ in range(3):
        out = ddp(torch.rand(4, 3, 32, 32), torch.rand(4, 3, 32, 32))
        loss = out["online_prediction1"].square().mean() \
            + out["linear_preds"].square().mean()
        opt.zero_grad()
        loss.backward()
        ddp.finish_grad_sync()
        if not lamb:
            norms.append(clip_grad_norm_(ddp.parameters(), 0.5))
            norms.append(ops.global_grad_norm([model.flat_space.flat_grads]))
        opt.step()
    torch.save({"params": model.flat_space.flat_params, "norms": norms},
               os.path.join(out_dir, f"{rank}.pt"))
    dist.destroy_process_group()


@pytest.mark.timeout(300)
@pytest.mark.parametrize("lamb", [True, False])
def test_replicas_stay_alike(lamb, tmp_path):
    """Two ranks on different data: the clipped steps follow the averaged
    gradients, the same on both."""
    mp.spawn(_replica, args=(29561 + lamb, str(tmp_path), lamb), nprocs=2,
             join=True)
    a, b = (torch.load(tmp_path / f"{r}.pt", weights_only=True)
            for r in (0, 1))
    assert torch.equal(a["params"], b["params"])
    for x, y in zip(a["norms"], b["norms"]):
        assert torch.equal(x, y)
    assert all(n <= 0.5 * (1 + 4 * E) for n in a["norms"][1::2])


class Branches(torch.nn.Module):
    """Two layers, of which forward uses the first and, if asked, the other."""

    def __init__(self):
        super().__init__()
        self.used = torch.nn.Linear(6, 5)
        self.unused = torch.nn.Linear(6, 5)
        self.frozen = torch.nn.Parameter(torch.ones(3), requires_grad=False)

    def forward(self, x, both=False):
        y = self.used(x)
        return (y + self.unused(x) if both else y).square().mean()


def flat_branches(device, **kw):
    from byol_amd.models.byol import FlatParamSpace
    torch.manual_seed(0)
    net = Branches().to(device)
    space = FlatParamSpace(net)
    space.flatten()
    opt = LAMB(net.parameters(), lr=0.01, weight_decay=1e-4, **kw)
    opt.attach_flat_space(space)
    return net, space, opt


@pytest.mark.parametrize("device", DEVICES)
def test_flat_space_skips_parameters_without_a_gradient(device):
    net, space, opt = flat_branches(device, max_grad_norm=1.0)
    x = torch.randn(8, 6, device=device)
    idle = (net.unused.weight, net.unused.bias, net.frozen)
    before = [p.detach().clone() for p in idle]
    moved = net.used.weight.detach().clone()
    for _ in range(5):
        opt.zero_grad()
        assert all(p.grad is None for p in net.parameters())
        net(x).backward()
        opt.step()
    for p, b in zip(idle, before):
        assert torch.equal(p, b) and p.grad is None and p not in opt.state
    assert not torch.equal(net.used.weight, moved)
    # then it is used, and its gradient is where the others are
    opt.zero_grad()
    net(x, both=True).backward()
    net(x, both=True).backward()  # and accumulates there
    want = torch.autograd.grad(net(x, both=True), list(net.used.parameters())
                               + list(net.unused.parameters()))
    for p, g in zip([*net.used.parameters(), *net.unused.parameters()], want):
        assert torch.allclose(p.grad, 2 * g)
    space.flat_grads.fill_(2.0)
    assert all((p.grad == 2).all() for p in net.parameters()
               if p.requires_grad)
    opt.step()
    assert not torch.equal(net.unused.weight, before[0])
    assert opt.state[net.unused.weight]["step"] == 1
    assert torch.equal(net.frozen, before[2])


def test_flat_space_clears_in_place_if_asked():
    net, space, opt = flat_branches("cpu")
    net(torch.randn(8, 6)).backward()
    opt.zero_grad(set_to_none=False)
    assert all((p.grad == 0).all() for p in net.parameters())
    space.flat_grads.fill_(2.0)
    assert all((p.grad == 2).all() for p in net.parameters())


def test_reduced_flat_space_keeps_all_gradients():
    """FlatDDP fills in gradients from other ranks: none is dropped, also if
    it wraps the model after an optimizer dropped them."""
    from byol_amd.parallel.ddp import FlatDDP
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", "29573"
    dist.init_process_group("gloo", rank=0, world_size=1)
    try:
        net, space, opt = flat_branches("cpu")
        net.frozen.requires_grad_(True)
        net.flat_space, net.target_network = space, None
        opt.zero_grad()
        ddp = FlatDDP(net)
        for _ in range(2):
            ddp(torch.randn(8, 6)).backward()
            ddp.finish_grad_sync()
            assert all(p.grad is not None for p in net.parameters())
            opt.step()
            opt.zero_grad()
        space.flat_grads.fill_(2.0)
        assert all((p.grad == 2).all() for p in net.parameters())
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,value,bound", [
    # factors 2.64e-10 and 0.0317
    (torch.float16, 6e4, 1e-2), (torch.float16, 0.5, 10.0),
    (torch.bfloat16, 6e4, 1e-2), (torch.bfloat16, 0.5, 10.0)])
def test_half_precision_parameters_clip_in_fp32(device, dtype, value, bound):
    """b1 = b2 = 0 puts the clipped gradient and its square in the moments, as
    they are but for roundings: 3e on g' in fp32 (see above), one to the
    moment's type and, on the way, one of the product with 1 - b1 = 1; for
    the square 7e and the same.  Below the type's normal numbers the rounding
    to it is half of its smallest subnormal instead."""
    p = torch.nn.Parameter(torch.full((400, 1000), 0.01, dtype=dtype,
                                      device=device))
    opt = LAMB([p], lr=0.1, betas=(0.0, 0.0), max_grad_norm=bound)
    p.grad = torch.full_like(p, value)
    g = p.grad[0, 0].double().item()
    want = g * min(1.0, bound / (g * math.sqrt(p.numel()) + 1e-6))
    opt.step()
    half = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).tiny * half
    state = opt.state[p]
    for name, value, terms in (("exp_avg", want, 4), ("exp_avg_sq", want ** 2,
                                                      8)):
        got = state[name].double()
        off = 1.01 * value * (terms * E + half) + least
        assert ((got - value).abs() <= off).all(), (name, got[0, 0], value)
    assert state["exp_avg"].dtype == dtype and p.isfinite().all()


@pytest.mark.gpu
def test_optimizer_steps_parameters_past_31_bits():
    """A parameter of 2^31 elements is too long for the fused step; beside
    one that is not.  With b1 = b2 = eps = 0 and g = 1, u = 1 without a
    rounding, and r = |p| / |u| = 0.5: sums of powers of two are exact up to
    2^24 of them, and joining those takes up to 31 roundings."""
    n = 2 ** 31
    params = [torch.nn.Parameter(torch.full((k,), 0.5, device="cuda"))
              for k in (n, 7)]
    for p in params:
        p.grad = torch.ones_like(p)
    opt = LAMB(params, lr=0.5, betas=(0.0, 0.0), eps=0.0)
    opt.step()
    for p in params:
        assert opt.state[p]["step"] == 1
        low, high = p.detach().aminmax()
        for got in (low, high):
            assert abs(got.item() - 0.25) <= 0.25 * 32 * E
    del params, p, opt
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_optimizer_lays_moments_out_like_their_parameter():
    """A checkpoint of another memory format, and moments of another type."""
    gen = torch.Generator().manual_seed(2)
    w = torch.randn(8, 6, 3, 3, generator=gen)
    g = torch.randn(8, 6, 3, 3, generator=gen)
    results = []
    for spoil in (False, True):
        p = torch.nn.Parameter(w.cuda().to(memory_format=torch.channels_last))
        opt = LAMB([p], lr=0.1)
        for turn in range(2):
            p.grad = g.cuda()
            opt.step()
            if spoil:
                state = opt.state[p]
                state["exp_avg"] = state["exp_avg"].contiguous()
                state["exp_avg_sq"] = state["exp_avg_sq"].double()
        results.append(p)
    assert torch.equal(*results)


@pytest.mark.parametrize("device", DEVICES)
def test_optimizer_counts_only_steps_that_it_takes(device, monkeypatch):
    p = torch.nn.Parameter(torch.ones(6, device=device))
    opt = LAMB([p], lr=0.1)
    p.grad = torch.ones_like(p)
    opt.step()
    before = p.detach().clone()

    def refuse(*args, **kw):
        raise ValueError("refused")
    with monkeypatch.context() as patch:
        patch.setattr(ops, "fused_lamb_step", refuse)
        patch.setattr(LAMB, "_fit_one_step", staticmethod(lambda *a: True))
        with pytest.raises(ValueError, match="refused"):
            opt.step()
    assert opt.state[p]["step"] == 1 and torch.equal(p, before)
    opt.step()
    assert opt.state[p]["step"] == 2


@pytest.mark.gpu
def test_optimizer_refuses_capture_before_it_does_anything():
    half = torch.nn.Parameter(torch.ones(6, device="cuda").bfloat16())
    p = torch.nn.Parameter(torch.ones(6, device="cuda"))
    opt = LAMB([half, p], lr=0.1, max_grad_norm=1.0)
    for t in (half, p):
        t.grad = torch.ones_like(t)
    opt.step()
    before = [t.detach().clone() for t in (half, p)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
        p.grad.mul_(1.0)
    torch.cuda.synchronize()
    for t, b in zip((half, p), before):
        assert torch.equal(t, b) and opt.state[t]["step"] == 1


@pytest.mark.parametrize("device", DEVICES)
def test_optimizer_steps_parameters_that_share_memory(device, monkeypatch):
    """One after the other, in torch operations: the bits of a list that is
    taken so in any case."""
    from byol_amd.ops.grad_clip import SharedMemoryError

    def stepped(alone, decay=(0.01, 0.0)):
        gen = torch.Generator().manual_seed(5)
        base = torch.randn(50, generator=gen).to(device)
        params = [torch.nn.Parameter(t) for t in (base[:30], base[20:],
                                                  base[:7].clone())]
        opt = LAMB([{"params": params[:2], "weight_decay": decay[0]},
                    {"params": params[2:], "weight_decay": decay[1]}], lr=0.1,
                   max_grad_norm=0.5)
        with monkeypatch.context() as patch:
            if alone:
                patch.setattr(LAMB, "_fit_one_step",
                              staticmethod(lambda *a: False))
            elif device == "cpu":  # the route that lists on a GPU take
                def refuse(*args, **kw):
                    raise SharedMemoryError("two share memory")
                patch.setattr(ops, "fused_lamb_step", refuse)
                patch.setattr(LAMB, "_fit_one_step",
                              staticmethod(lambda *a: True))
            for _ in range(3):
                for p in params:
                    p.grad = torch.randn(p.shape, generator=gen).to(device)
                opt.step()
        assert [opt.state[p]["step"] for p in params] == [3, 3, 3]
        return base, params[2]

    for a, b in zip(stepped(False), stepped(True)):
        assert torch.equal(a, b) and a.isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
def test_sharing_is_refused_as_such(device):
    from byol_amd.ops.grad_clip import SharedMemoryError
    _, (p, g, m, v) = make([64, 8], device)
    with pytest.raises(SharedMemoryError, match="twice"):
        ops.fused_lamb_step(p, g, m, m, step=1, lr=0.1)


def clipped_alike(devices, dtypes):
    """Gradients of several types or devices are clipped by their common norm:
    as much as after clipping them by hand."""
    gen = torch.Generator().manual_seed(6)
    values = [torch.randn(40, 9, generator=gen) for _ in dtypes]
    want = math.sqrt(sum(v.to(t).double().square().sum().item()
                         for v, t in zip(values, dtypes)))
    results = []
    for inside in (True, False):
        params = [torch.nn.Parameter(torch.full((40, 9), 0.1, dtype=t,
                                                device=d))
                  for t, d in zip(dtypes, devices)]
        opt = LAMB(params, lr=0.1, betas=(0.5, 0.5),
                   max_grad_norm=0.25 if inside else 0.0)
        for p, v in zip(params, values):
            p.grad = v.to(p.device, p.dtype)
            if not inside:
                p.grad.mul_(0.25 / (want + 1e-6))
        opt.step()
        results.append([opt.state[p]["exp_avg"].double().cpu()
                        for p in params])
    for a, b, t in zip(*results, dtypes):
        # both: factor, product and moment; fp64's norm is summed in fp64
        e = 2.0 ** -52 if t is torch.float64 else max(
            E, torch.finfo(t).eps / 2)
        assert ((a - b).abs() <= 8 * e * b.abs()).all()


def test_optimizer_clips_fp64():
    clipped_alike(["cpu"] * 2, [torch.float64] * 2)


def test_optimizer_clips_fp64_beside_fp32():
    clipped_alike(["cpu"] * 2, [torch.float64, torch.float32])


@pytest.mark.gpu
def test_optimizer_clips_on_several_devices():
    clipped_alike(["cuda", "cpu", "cuda"],
                  [torch.float32, torch.float32, torch.float64])


@pytest.mark.parametrize("device", DEVICES)
def test_views_of_negated_memory(device):
    """Gradients that are lazily negated views count with their sign; such
    parameters are refused by the operator on a GPU and stepped by LAMB."""
    _, lists = make([300, 41], device)
    before = [[t.clone() for t in ts] for ts in lists]
    lists[1] = [torch._neg_view(-g) for g in lists[1]]
    ops.fused_lamb_step(*lists, step=3, lr=0.1, max_grad_norm=0.5)
    norm = torch.cat([g.cpu().double() for g in before[1]]).norm().item()
    check(lists, before, 3, 0.1, 1e-6, [0.0, 0.0], 0.5 / (norm + 1e-6),
          slack=device == "cpu")
    results = []
    for negated in (False, True):
        value = torch.arange(1.0, 9.0, device=device)
        p = torch.nn.Parameter(torch._neg_view(-value) if negated else value)
        opt = LAMB([p], lr=0.1)
        p.grad = torch.ones(8, device=device)
        opt.step()
        results.append(p.detach().clone())
    # the fused form and the one in torch operations: see the bounds above
    assert torch.allclose(*results, rtol=64 * E, atol=0)


@pytest.mark.gpu
def test_clipping_views_of_negated_memory():
    g = torch.randn(500, device="cuda")
    view, before = torch._neg_view(-g), g.clone()
    norm = before.cpu().double().norm().item()
    ops.clip_grads_by_norm_([view], norm / 2)
    want = before.cpu().double() * (norm / 2 / (norm + 1e-6))
    # the factor and the product are rounded
    assert ((view.cpu().double() - want).abs()
            <= 1.01 * 2 * E * want.abs()).all()
    ops.clip_grads_by_value_([view], 0.25)
    assert torch.equal(view.sign(), before.sign())
    assert view.abs().max() == 0.25


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_do_not_share_what_is_written(device):
    _, (p, g, m, v) = make([64, 8], device)
    before = [t.clone() for t in p + m + v]
    wide = torch.ones(80, device=device)
    for bad in ([p[0], g[1]], [g[0], m[1]], [m[0], g[1]], [g[0], v[0][3:11]],
                [g[0], p[0][::8]]):
        with pytest.raises(ValueError, match="memory"):
            ops.fused_lamb_step(p, bad, m, v, step=1, lr=0.1)
    for a, b in zip(p + m + v, before):
        assert torch.equal(a, b)
    # among each other they may: they are only read
    ops.fused_lamb_step(p, [wide[:64], wide[60:68]], m, v, step=1, lr=0.1)
    assert not torch.equal(p[1], before[1])


@pytest.mark.gpu
def test_engine_replays_a_captured_step_that_clips(tmp_path, monkeypatch,
                                                   capsys):
    """--hip-graph with --clip-norm: the step is captured, not continued
    eagerly, and each replay leaves gradients of the bound's norm."""
    from byol_amd.engine import graph_step, trainer
    from byol_amd.optim import build_optimizer
    args = engine_args(tmp_path, "cuda", "--clip-norm", "0.001",
                       "--channels-last", "--hip-graph")
    torch.manual_seed(0)
    loader, model, grapher = trainer.build_loader_model_grapher(args)
    opt, _ = build_optimizer(model, args)
    for group in opt.param_groups:
        group["lr"] = 0.001  # past the warmup's zero
    norms, replay = [], graph_step.GraphedTrainStep.replay

    def watched(self, *inputs):
        model.flat_space.flat_grads.fill_(9.0)  # not the last step's
        out = replay(self, *inputs)
        norms.append(ops.global_grad_norm([model.flat_space.flat_grads]))
        return out
    monkeypatch.setattr(graph_step.GraphedTrainStep, "replay", watched)
    trainer.train(1, model, opt, loader.train_loader, grapher, args)
    assert "capture failed" not in capsys.readouterr().out
    assert len(norms) == 2  # of four minibatches the last two
    # the norm and the factor are rounded, and each product
    for norm in norms:
        want = 0.001 / (1 + 1e-6 / 1e-3)  # at least, for norms above 0.001
        assert want * (1 - 8 * E) <= norm.item() <= 0.001 * (1 + 8 * E)
    assert torch.isfinite(model.flat_space.flat_params).all()


def test_flat_space_drops_the_gradients_that_it_made():
    """A parameter that the model gets later is none of the flat space's: it
    does not shift the others' views."""
    net, space, opt = flat_branches("cpu")
    net.first = torch.nn.Linear(6, 6)
    net._modules = {"first": net.first, **net._modules}  # comes first
    x = torch.randn(8, 6)
    for _ in range(2):
        opt.zero_grad()
        net(x).backward()
        want = torch.autograd.grad(net(x), list(net.used.parameters()))
        for p, g in zip(net.used.parameters(), want):
            assert torch.allclose(p.grad, g)
        opt.step()
    space.flat_grads.fill_(2.0)
    assert all((p.grad == 2).all() for p in net.used.parameters())
    assert net.first.weight.grad is None
    by_name = space.named_views(space.flat_grads)
    for name, p in net.named_parameters():
        if p.grad is not None:
            assert p.grad.data_ptr() == by_name[name].data_ptr(), name


def test_flat_space_does_not_bring_old_gradients_back():
    """Gradients that the model or another optimizer drops, which leaves their
    values in the buffer, and FlatDDP around a model with such a buffer."""
    net, space, opt = flat_branches("cpu")
    xs = torch.randn(4, 8, 6)
    opt.zero_grad()
    net(xs[0]).backward()
    opt.step()
    params = list(net.used.parameters())
    for x in xs[1:]:
        net.zero_grad()
        net(x).backward()
        for p, g in zip(params, torch.autograd.grad(net(x), params)):
            assert torch.allclose(p.grad, g)
    opt.step()
    opt.zero_grad()
    net(xs[0]).backward()  # back in the buffer
    space.flat_grads.fill_(2.0)
    assert all((p.grad == 2).all() for p in params)
    net.zero_grad()
    space.attach_grads()
    assert all((p.grad == 0).all() for p in net.parameters())
