"""Global gradient norm and clipping: against 64-bit values, refusals, streams
and graphs.

Tolerances, e = 2^-24 (half an fp32 step): the kernels sum in 64 bits (n * 2^-53
is below e / 100 for every n here) and round the norm once, to fp32: e.  The
clipping factor is rounded once (e), its product with a value once more to
fp32 (e), and the result to the gradient's type (half a step of it; for fp32
the product is the result).  Results below a type's smallest normal number are
off by up to half its smallest subnormal instead.  1.01 covers products of
these terms.
"""

import math

import pytest
import torch

from byol_amd import ops
from byol_amd.optim import clip_grad_norm_, clip_grad_value_

E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
#: half of the smallest subnormal number
SUBNORMAL = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134,
             torch.float16: 2.0 ** -25}
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def exact_norm(grads, norm_type):
    parts = [g.detach().cpu().double().reshape(-1) for g in grads]
    flat = torch.cat(parts) if parts else torch.zeros(0).double()
    if norm_type == math.inf:
        return flat.abs().max().item() if len(flat) else 0.0
    return flat.square().sum().sqrt().item()


def check_norm(got, want):
    assert got.dtype == torch.float32 and got.dim() == 0
    got = got.item()
    if math.isnan(want):
        assert math.isnan(got)
    elif math.isinf(want):
        assert got == want
    else:
        assert abs(got - want) <= 1.01 * E * want + SUBNORMAL[torch.float32]


def check_scaled(got, before, norm, bound):
    want = before.cpu().double() * min(1.0, bound / (norm + 1e-6))
    dtype = got.dtype
    rel = 2 * E + (0 if dtype == torch.float32 else half_step(dtype))
    off = (got.cpu().double() - want).abs()
    assert (off <= 1.01 * rel * want.abs() + SUBNORMAL[dtype]).all(), \
        off.max().item()


def make(sizes, dtype, device, seed=0, gap=0):
    """Tensors in one buffer of sevens, `gap` values between them."""
    gen = torch.Generator().manual_seed(seed)
    total = sum(sizes) + gap * (len(sizes) + 1)
    arena = torch.full((total,), 7.0, dtype=dtype)
    spans, at = [], gap
    for i, n in enumerate(sizes):
        arena[at:at + n] = (torch.randn(n, generator=gen)
                            * 10.0 ** (-(i % 4))).to(dtype)
        spans.append((at, n))
        at += n + gap
    arena = arena.to(device)
    return arena, [arena[a:a + n] for a, n in spans]


def outside(arena, views):
    used = torch.zeros(arena.numel(), dtype=torch.bool)
    base = arena.data_ptr()
    for v in views:
        a = (v.data_ptr() - base) // arena.element_size()
        used[a:a + v.numel()] = True
    return arena.cpu()[~used]


LISTS = {
    "one value": [1],
    "one bias": [257],
    "no values among some": [0, 5, 0, 64],
    "around a pack": [3, 4, 5, 7, 8, 9, 15, 16, 17],
    "around a block's share": [2047, 2048, 2049, 4095, 4096, 4097],
    "more tensors than a table": [1 + (i * 37) % 300 for i in range(500)],
    "large beside small": [3_000_001, 1, 70_000],
}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gap", [0, 1])
@pytest.mark.parametrize("sizes", LISTS.values(), ids=LISTS.keys())
def test_norm_and_clip(device, norm_type, dtype, gap, sizes):
    arena, grads = make(sizes, dtype, device, gap=gap)
    before = [g.clone() for g in grads]
    want = exact_norm(grads, norm_type)
    check_norm(ops.global_grad_norm(grads, norm_type), want)
    for bound in (want * 3, want / 3):
        got = ops.clip_grads_by_norm_(grads, bound, norm_type)
        check_norm(got, want)
        for g, b in zip(grads, before):
            check_scaled(g, b, want, bound)
            if bound > want:
                assert torch.equal(g, b)
    assert (outside(arena, grads) == 7).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", LISTS.values(), ids=LISTS.keys())
def test_clip_by_value(device, dtype, sizes):
    arena, grads = make(sizes, dtype, device, gap=1)
    grads[0][:1] = math.nan
    grads[-1][-1:] = -math.inf
    before = [g.clone() for g in grads]
    ops.clip_grads_by_value_(grads, 0.3)
    for g, b in zip(grads, before):
        # one rounding on both sides: the same bits
        want = b.float().clamp(-0.3, 0.3).to(dtype)
        assert torch.equal(g.nan_to_num(5.0), want.nan_to_num(5.0))
    assert (outside(arena, grads) == 7).all()


@pytest.mark.parametrize("device", DEVICES)
def test_types_in_one_list(device):
    grads = [make([n], t, device, seed=n)[1][0]
             for n, t in zip((5000, 33, 1, 4097, 8, 600), TYPES * 2)]
    before = [g.clone() for g in grads]
    want = exact_norm(grads, 2.0)
    check_norm(ops.clip_grads_by_norm_(grads, want / 7), want)
    for g, b in zip(grads, before):
        check_scaled(g, b, want, want / 7)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_strides(device, norm_type):
    def grads():
        _, (a, b, c, d) = make([4 * 6 * 5 * 3, 40 * 9, 30 * 7, 64],
                               torch.float32, device, seed=3)
        return [a.view(4, 6, 5, 3).to(memory_format=torch.channels_last),
                b.view(40, 9).t(), c.view(30, 7)[:, 1:6:2], d[5:]]
    gs, before = grads(), [g.clone() for g in grads()]
    assert not gs[2].is_contiguous()
    want = exact_norm(gs, norm_type)
    check_norm(ops.global_grad_norm(gs, norm_type), want)
    strides = [g.stride() for g in gs]
    ops.clip_grads_by_norm_(gs, want / 5, norm_type)
    for g, b, s in zip(gs, before, strides):
        assert g.stride() == s
        check_scaled(g, b, want, want / 5)
    gs = grads()
    ops.clip_grads_by_value_(gs, 0.1)
    for g, b in zip(gs, before):
        assert torch.equal(g, b.clamp(-0.1, 0.1))


@pytest.mark.parametrize("device", DEVICES)
def test_expanded_view_counts_each_element(device):
    one = torch.tensor([3.0], device=device)
    check_norm(ops.global_grad_norm([one.expand(16)]), 12.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("value,norm", [
    (1e30, 1e30 * 2 ** 0.5), (1e-30, 1e-30 * 2 ** 0.5), (0.0, 0.0),
    (math.inf, math.inf), (-math.inf, math.inf), (math.nan, math.nan)])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_extreme_values(device, value, norm, norm_type):
    grads = [torch.zeros(700, device=device), torch.zeros(3, device=device)]
    grads[0][600] = grads[1][2] = value
    want = exact_norm(grads, norm_type)
    check_norm(ops.global_grad_norm(grads, norm_type), want)
    got = ops.clip_grads_by_norm_(grads, 1.0, norm_type)
    check_norm(got, want)
    if math.isnan(norm):  # a NaN factor reaches every value
        assert all(g.isnan().all() for g in grads)
    elif math.isinf(norm):  # factor 0, and 0 * inf
        assert grads[0][600].isnan() and grads[1][2].isnan()
        assert grads[0][599] == 0 and grads[1][0] == 0
    else:
        assert abs(grads[0][600].item()
                   - value * min(1.0, 1.0 / (want + 1e-6))) \
            <= 1.01 * 2 * E * abs(value)


@pytest.mark.parametrize("device", DEVICES)
def test_infinity_beside_nan(device):
    g = torch.zeros(5000, device=device)
    g[10], g[4000] = math.inf, math.nan
    assert ops.global_grad_norm([g]).isnan()
    assert ops.global_grad_norm([g], math.inf).isnan()


@pytest.mark.parametrize("device", DEVICES)
def test_bounds_of_zero_and_infinity(device):
    g = torch.randn(100, device=device)
    before = g.clone()
    ops.clip_grads_by_norm_([g], math.inf)
    ops.clip_grads_by_value_([g], math.inf)
    assert torch.equal(g, before)
    ops.clip_grads_by_norm_([g], 0.0)
    assert (g == 0).all()
    ops.clip_grads_by_value_([before], 0.0)
    assert (before == 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_nothing_to_clip(device):
    assert ops.global_grad_norm([]).item() == 0
    assert ops.clip_grads_by_norm_([], 1.0).item() == 0
    ops.clip_grads_by_value_([], 1.0)
    empty = [torch.zeros(0, device=device), torch.zeros(0, 4, device=device)]
    assert ops.global_grad_norm(empty).item() == 0
    assert ops.global_grad_norm(empty, math.inf).item() == 0
    assert ops.clip_grads_by_norm_(empty, 1.0).item() == 0
    ops.clip_grads_by_value_(empty, 1.0)


@pytest.mark.parametrize("device", DEVICES)
def test_one_tensor_is_a_list_of_it(device):
    g = torch.full((4, 4), 2.0, device=device)
    check_norm(ops.global_grad_norm(g), 8.0)
    check_norm(ops.clip_grads_by_norm_(g, 4.0), 8.0)
    check_scaled(g, torch.full((4, 4), 2.0), 8.0, 4.0)
    ops.clip_grads_by_value_(g, 0.5)
    assert (g == 0.5).all()
    with pytest.raises(TypeError):
        ops.global_grad_norm([1.0, g])


@pytest.mark.parametrize("device", DEVICES)
def test_thousands_of_tensors_then_few(device):
    _, many = make([1 + i % 5 for i in range(9000)], torch.float32, device,
                   gap=1)
    few = [torch.tensor(3.0, device=device), torch.full((2, 2), 2.0,
                                                        device=device)]
    for _ in range(2):
        check_norm(ops.global_grad_norm(few), 5.0)
        check_norm(ops.global_grad_norm(many), exact_norm(many, 2.0))
    before = [g.clone() for g in many]
    want = exact_norm(many, 2.0)
    check_norm(ops.clip_grads_by_norm_(many, 1.0), want)
    for g, b in zip(many[::97], before[::97]):
        check_scaled(g, b, want, 1.0)
    check_norm(ops.clip_grads_by_norm_(few, 1.0), 5.0)
    assert few[0].dim() == 0 and abs(few[0].item() - 0.6) < 1e-6


@pytest.mark.gpu
def test_inside_inference_mode():
    with torch.inference_mode():
        g = torch.full((100,), 2.0, device="cuda")
        check_norm(ops.clip_grads_by_norm_([g], 5.0), 20.0)
        check_scaled(g, torch.full((100,), 2.0), 20.0, 5.0)
        ops.clip_grads_by_value_([g], 0.25)
        assert (g == 0.25).all()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    g = torch.ones(64, device=device)
    calls = [lambda t: ops.clip_grads_by_norm_(t, 0.1),
             lambda t: ops.clip_grads_by_value_(t, 0.1)]
    for call in calls:
        for bad in ([g, g], [g[:40], g[20:]], [g[::2], g[1::2]],
                    [g[:1].expand(8)], [g.view(8, 8), g.view(8, 8).t()]):
            with pytest.raises(ValueError, match="memory|twice"):
                call(bad)
        for bad in (g.double(), g.long(), g.to_sparse(), g.cfloat()):
            with pytest.raises(TypeError):
                call([bad])
            with pytest.raises(TypeError):
                ops.global_grad_norm([bad])
    for bound in (-1.0, math.nan):
        with pytest.raises(ValueError, match="must be >= 0"):
            ops.clip_grads_by_norm_([g], bound)
        with pytest.raises(ValueError, match="must be >= 0"):
            ops.clip_grads_by_value_([g], bound)
    for norm_type in (1.0, 0, -math.inf, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            ops.global_grad_norm([g], norm_type)
        with pytest.raises(ValueError, match="norm_type"):
            ops.clip_grads_by_norm_([g], 1.0, norm_type)
    assert (g == 1).all()


@pytest.mark.skipif(not ops.has_extension(), reason="extension not built")
def test_binding_refuses_before_any_launch():
    """The checks of the binding itself, on CPU tensors: it never launches
    for them."""
    ext = ops.extension()
    g = torch.ones(64)
    for bad, error in (([g], ValueError), ([g, g], ValueError),
                       ([g[:1].expand(8)], ValueError),
                       ([g.double()], TypeError), ([g.to_sparse()], TypeError),
                       (["no tensor"], TypeError)):
        with pytest.raises(error):
            ext.grad_clip_norm(bad, 1.0, False)
        with pytest.raises(error):
            ext.grad_clip_value(bad, 1.0)
    with pytest.raises(ValueError):
        ext.grad_norm([g], False)
    with pytest.raises(ValueError):
        ext.grad_clip_norm([g], -1.0, False)
    assert (g == 1).all()


@pytest.mark.gpu
def test_devices_do_not_mix():
    a, b = torch.ones(8), torch.ones(8, device="cuda")
    for grads in ([a, b], [b, a]):
        with pytest.raises(ValueError, match="expected"):
            ops.global_grad_norm(grads)
        with pytest.raises(ValueError, match="expected"):
            ops.clip_grads_by_norm_(grads, 0.1)
        with pytest.raises(ValueError, match="expected"):
            ops.clip_grads_by_value_(grads, 0.1)
    assert (a == 1).all() and (b == 1).all()


@pytest.mark.parametrize("device", DEVICES)
def test_parameters(device):
    """The wrappers over parameters agree with torch's own functions."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(30, 7), torch.nn.Linear(7, 2))
    model.to(device)
    model[1].bias.requires_grad_(False)  # a parameter without a gradient
    model(torch.randn(5, 30, device=device)).square().sum().backward()
    grads = [p.grad for p in model.parameters() if p.grad is not None]
    before = [g.clone() for g in grads]
    version = grads[0]._version
    norm = clip_grad_norm_(model.parameters(), 0.5)
    assert grads[0]._version > version
    want = exact_norm(before, 2.0)
    check_norm(norm, want)
    for g, b in zip(grads, before):
        check_scaled(g, b, want, 0.5)
    clip_grad_value_(model.parameters(), 0.01)
    assert max(g.abs().max().item() for g in grads) <= 0.01 * (1 + E)
    clip_grad_norm_(model[0].weight, 1e-3)  # one parameter, not a list
    check_norm(clip_grad_norm_([model[0].weight], 1.0),
               exact_norm([model[0].weight.grad], 2.0))
    grads[0][0, 0] = math.nan
    with pytest.raises(RuntimeError, match="nan"):
        clip_grad_norm_(model.parameters(), 1.0, error_if_nonfinite=True)


@pytest.mark.gpu
def test_same_bits_every_time():
    _, grads = make([100_003, 5, 64, 1_000_000], torch.float32, "cuda", gap=3)
    norms = {ops.global_grad_norm(grads).item() for _ in range(20)}
    assert len(norms) == 1


@pytest.mark.gpu
def test_tensors_past_32_bits():
    """More than 2^30 elements in a tensor, more than 2^32 bytes in a list."""
    n = 2 ** 30 + 2 ** 29 + 5
    g = torch.zeros(n, device="cuda")
    places = torch.tensor([0, 2 ** 29, 2 ** 30 - 1, 2 ** 30, n - 1],
                          device="cuda")
    g[places] = torch.tensor([3.0, -4.0, 12.0, -84.0, 132.0], device="cuda")
    want = math.sqrt(9 + 16 + 144 + 84 ** 2 + 132 ** 2)
    check_norm(ops.global_grad_norm([g]), want)
    assert ops.global_grad_norm([g], math.inf).item() == 132
    ops.clip_grads_by_value_([g], 10.0)
    assert g[places].tolist() == [3.0, -4.0, 10.0, -10.0, 10.0]
    norm = math.sqrt(9 + 16 + 300)
    check_norm(ops.clip_grads_by_norm_([g], 1.0), norm)
    check_scaled(g[places], torch.tensor([3.0, -4.0, 10.0, -10.0, 10.0]),
                 norm, 1.0)
    assert int((g != 0).sum()) == 5


@pytest.mark.gpu
def test_tensors_far_apart():
    """More than 2^32 elements between two tensors of a list."""
    arena = torch.empty(2 ** 32 + 4096, dtype=torch.bfloat16, device="cuda")
    far = [arena[3:2003], arena[-777:], arena[5000:5001]]
    for i, g in enumerate(far):
        g.copy_(torch.randn(g.shape) * (i + 1))
    before = [g.clone() for g in far]
    want = exact_norm(far, 2.0)
    check_norm(ops.clip_grads_by_norm_(far, want / 9), want)
    for g, b in zip(far, before):
        check_scaled(g, b, want, want / 9)
    ops.clip_grads_by_value_(far, 0.01)
    assert max(g.abs().max().item() for g in far) <= 0.01 * (1 + 2.0 ** -8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_every_alignment(dtype):
    """Each place in a cache line, lengths around it, and chunks that begin
    inside a tensor; nothing beside the tensors changes."""
    for n in (1, 2, 7, 8, 9, 63, 64, 65, 129, 4096, 9001):
        arena = torch.full((40 * (n + 71) + 200,), 7.0, dtype=dtype,
                           device="cuda")
        grads, at = [], 0
        for i in range(40):
            at += 1 + i % 3
            grads.append(arena[at:at + n])
            at += n + 2 * i
        for i, g in enumerate(grads):
            g.copy_((torch.randn(n) + 3) * (1 + i % 2))
        before = [g.clone() for g in grads]
        rest = outside(arena, grads)
        want = exact_norm(grads, 2.0)
        check_norm(ops.clip_grads_by_norm_(grads, want / 2), want)
        for g, b in zip(grads, before):
            check_scaled(g, b, want, want / 2)
        check_norm(ops.global_grad_norm(grads, math.inf),
                   exact_norm(grads, math.inf))
        ops.clip_grads_by_value_(grads, 0.25)
        assert all(g.abs().max().item() <= 0.25 for g in grads)
        assert torch.equal(outside(arena, grads), rest)


@pytest.mark.gpu
def test_two_streams():
    """Two calls at once, on streams of their own, share nothing."""
    lists = [make([500_001, 77, 3000], torch.float32, "cuda", seed=s, gap=1)[1]
             for s in (1, 2)]
    want = [exact_norm(g, 2.0) for g in lists]
    streams = [torch.cuda.Stream() for _ in lists]
    before = [[g.clone() for g in gs] for gs in lists]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for gs, s in zip(lists, streams):
            with torch.cuda.stream(s):
                got.append(ops.global_grad_norm(gs))
    norms = []
    for gs, s, w in zip(lists, streams, want):
        with torch.cuda.stream(s):
            norms.append(ops.clip_grads_by_norm_(gs, w / 2))
    torch.cuda.synchronize()
    for i, norm in enumerate(got):
        check_norm(norm, want[i % 2])
    for gs, bs, norm, w in zip(lists, before, norms, want):
        check_norm(norm, w)
        for g, b in zip(gs, bs):
            check_scaled(g, b, w, w / 2)


@pytest.mark.gpu
def test_captured_graphs():
    """Two graphs of both clippings, replayed in turn with eager calls and
    waits in between, give what eager calls give on the same values."""
    sizes = [40_000, 3, 129, 8192]
    _, grads = make(sizes, torch.float32, "cuda", gap=1)
    _, other = make(sizes, torch.bfloat16, "cuda", seed=5)

    def step(gs, bound):
        norm = ops.clip_grads_by_norm_(gs, bound)
        ops.clip_grads_by_value_(gs, bound / 50)
        return norm

    graphs, norms = [], []
    for gs in (grads, other):
        with torch.cuda.stream(torch.cuda.Stream()):
            step([g.clone() for g in gs], 2.0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(step(gs, 2.0))
        graphs.append(graph)
    for turn in range(4):
        for gs, graph, norm in zip((grads, other), graphs, norms):
            fresh = [torch.randn_like(g) * (turn + 1) for g in gs]
            for g, f in zip(gs, fresh):
                g.copy_(f)
            graph.replay()
            want = step(fresh, 2.0)
            torch.cuda.synchronize()
            assert torch.equal(norm, want)
            for g, f in zip(gs, fresh):
                assert torch.equal(g, f)


@pytest.mark.gpu
def test_refuses_to_wait_while_captured():
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    p.grad = torch.ones(8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
        clip_grad_norm_([p], 1.0)
    graph.replay()
    torch.cuda.synchronize()
    check_scaled(p.grad, torch.ones(8), math.sqrt(8), 1.0)


@pytest.mark.gpu
def test_captured_with_the_lars_step():
    """Clipping and the fused LARS step in one graph.  Every tensor is below
    the step's chunk of 65536, so that one block sums it and the bits are the
    eager ones on every replay."""
    from byol_amd import layers
    from byol_amd.models.byol import FlatParamSpace
    from byol_amd.optim.lars import LARS

    def build():
        torch.manual_seed(3)
        net = torch.nn.Sequential(*(torch.nn.Linear(61, 61)
                                    for _ in range(5))).cuda()
        space = FlatParamSpace(net)
        space.flatten()
        opt = LARS(torch.optim.SGD(layers.add_weight_decay(net, 1e-4), lr=0.05,
                                   momentum=0.9))
        opt.attach_flat_space(space)

        def step():
            norm = clip_grad_norm_(net.parameters(), 0.5)
            opt.step()
            return norm
        return space, opt, step

    (want, _, eager), (got, opt, captured) = build(), build()
    values = [torch.randn_like(want.flat_grads) * 10.0 ** (turn - 2)
              for turn in range(5)]
    for space, step in ((want, eager), (got, captured)):
        space.flat_grads.copy_(values[0])
        step()  # makes the momentum
    opt._fused.lr_dev.fill_(0.05)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = captured()
    for value in values[1:]:
        got.flat_grads.copy_(value)
        graph.replay()
        want.flat_grads.copy_(value)
        expect = eager()
        torch.cuda.synchronize()
        assert torch.equal(norm, expect)
        assert torch.equal(got.flat_params, want.flat_params)


@pytest.mark.gpu
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("sizes", [[1], [300_001, 5, 64], [7] * 500,
                                   [3_000_001, 1, 70_000]])
def test_norm_of_a_join_that_does_not_wait(norm_type, sizes):
    """The joining block computes what it would have to wait for: the same
    bits, and no sum of a late block is left for a later call, whose list is
    shorter or longer and has other values."""
    ext, inf = ops.extension(), norm_type == math.inf
    _, grads = make(sizes, torch.float32, "cuda", gap=1)
    _, other = make([n // 2 + 1 for n in sizes] + [9], torch.bfloat16, "cuda",
                    seed=4, gap=1)
    lists = [grads, other, [2 * g for g in grads], grads + other]
    want = [ops.global_grad_norm(gs, norm_type) for gs in lists]
    for gs, norm in zip(lists, want):
        check_norm(norm, exact_norm(gs, norm_type))
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        for turn in range(6):
            for i in (0, 1, 2, 1, 3, 0):
                ticks = (0, 1, 1000000)[(turn + i) % 3]
                assert torch.equal(ext.grad_norm(lists[i], inf, ticks),
                                   want[i]), (turn, i, ticks)


@pytest.mark.skipif(not ops.has_extension(), reason="extension not built")
def test_binding_refuses_waits_out_of_range():
    g = torch.ones(64)
    for ticks in (-1, 10 ** 9):
        with pytest.raises(ValueError, match="wait_ticks"):
            ops.extension().grad_norm([g], False, ticks)


@pytest.mark.parametrize("device", DEVICES)
def test_parameters_with_gradients_of_any_kind_by_value(device):
    """What the operator refuses is bounded one by one: fp64, views that
    interleave or are the same memory, and fp32 beside them."""
    gen = torch.Generator().manual_seed(8)
    base = torch.randn(40, generator=gen)
    plain, double = torch.randn(9, generator=gen), torch.randn(
        7, generator=gen).double()

    def grads():
        b = base.to(device)
        return [b[::2], b[1::2], b[4:9]], [plain.to(device),
                                           double.to(device)]

    for part in range(2):
        values = grads()[part]
        want = [g.clamp(-0.25, 0.25) for g in grads()[part]]
        params = [torch.nn.Parameter(torch.zeros_like(g)) for g in values]
        for p, g in zip(params, values):
            p.grad = g
        clip_grad_value_(params, 0.25)
        for p, w in zip(params, want):
            assert torch.equal(p.grad, w) and p.grad.dtype == w.dtype
        for bad in (-1.0, math.nan):
            with pytest.raises(ValueError, match="must be >= 0"):
                clip_grad_value_(params, bad)
        for p, w in zip(params, want):
            assert torch.equal(p.grad, w)


@pytest.mark.gpu
def test_parameters_on_several_devices_by_value():
    params = [torch.nn.Parameter(torch.zeros(5, device=d))
              for d in ("cpu", "cuda")]
    for p in params:
        p.grad = torch.full_like(p, 3.0)
    clip_grad_value_(params, 0.5)
    assert all((p.grad == 0.5).all() for p in params)


@pytest.mark.gpu
def test_missing_extension_is_an_error(monkeypatch):
    """No fallback hides that the kernels are not built."""
    def missing(what):
        raise RuntimeError("not built")
    monkeypatch.setattr("byol_amd.ops.grad_clip.require_extension", missing)
    p = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="not built"):
        clip_grad_value_([p], 0.5)


@pytest.mark.gpu
def test_places_are_kept_for_some_streams_only():
    """Over more streams than places are kept for, twice over: every norm is
    right, whether its stream's places are there, gone or in the way."""
    lists = [make([n, 30_000], torch.float32, "cuda", seed=n)[1]
             for n in (5, 200_000)]
    want = [exact_norm(gs, 2.0) for gs in lists]
    streams = [torch.cuda.Stream() for _ in range(30)]
    torch.cuda.synchronize()
    got = []
    for turn in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i + turn, ops.global_grad_norm(
                    lists[(i + turn) % 2])))
    torch.cuda.synchronize()
    for i, norm in got:
        check_norm(norm, want[i % 2])
    assert ops.extension().grad_norm_streams() <= 16
