"""AdamW over a program's whole life: parameters whose gradients come late, groups, memory that is
shared or moves, divisors at the ends of the range. CFG and the numpy step are those of
test_network_norm_adamw_gpu, which give every bit."""
import math

import numpy as np
import pytest

from test_network_norm_adamw_gpu import CFG, F, _np, _numpy_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_each_parameter_counts_its_own_steps(bits):
    """A parameter whose first gradient comes after 50 steps of others takes a fresh optimiser's first
    step, one without a gradient in between goes on with its own count, and so does an optimiser made
    from the state."""
    import torch
    from splatx_cuda.network import AdamW
    gen = torch.Generator().manual_seed(bits)
    t = lambda n: torch.randn(n, generator=gen).cuda()  # noqa: E731
    early, late, never = t(3000), t(700), t(5)
    new, kept = late.clone(), never.clone()
    opt = AdamW([early, late, never], state_bits=bits, **CFG)
    for _ in range(50):
        opt.step([t(3000), None, None])
    assert torch.equal(late, new) and opt.state()["step"] == [50, 0, 0]
    g = [t(700) for _ in range(3)]
    opt.step([t(3000), g[0], None])
    fresh = AdamW([new], state_bits=bits, **CFG)
    fresh.step([g[0]])
    assert torch.equal(late, new)
    if bits == 32:
        was = np.zeros(700, F)
        first = torch.zeros(700, device="cuda")
        AdamW([first], **CFG).step([g[0]])
        assert np.array_equal(_np(first), _numpy_step(was, _np(g[0]), was, was, 1)[0])
    opt.step([None, g[1], None])
    fresh.step([g[1]])
    assert torch.equal(late, new) and opt.state()["step"] == [51, 2, 0]
    opt.step([None, None, None])
    assert opt.state()["step"] == [51, 2, 0] and torch.equal(never, kept)
    state = {k: v if k == "step" else [x.clone() for x in v] for k, v in opt.state().items()}
    copy = [x.clone() for x in (early, late, never)]
    other = AdamW(copy, state_bits=bits, state=state, **CFG)
    ge = t(3000)
    opt.step([ge, g[2], None])
    other.step([ge, g[2], None])
    fresh.step([g[2]])
    assert torch.equal(late, new) and all(torch.equal(x, y) for x, y in zip((early, late, never), copy))
    assert other.state()["step"] == [52, 3, 0] and fresh.state()["step"] == 3


def test_counts_of_steps_are_checked():
    import torch
    from splatx_cuda.network import AdamW
    a, b = torch.zeros(8, device="cuda"), torch.zeros(4, device="cuda")
    moments = lambda: [torch.zeros(8, device="cuda"), torch.zeros(4, device="cuda")]  # noqa: E731
    for bad in ([1], [1, 2, 3], [1, -1], -1):
        with pytest.raises(ValueError):
            AdamW([a, b], state={"step": bad, "exp_avg": moments(), "exp_avg_sq": moments()})
    for good, shown in ((7, 7), ([7, 7], 7), ([7, 0], [7, 0])):
        opt = AdamW([a, b], state={"step": good, "exp_avg": moments(), "exp_avg_sq": moments()})
        assert opt.state()["step"] == shown


def test_a_bad_rate_stops_every_launch():
    import torch
    from splatx_cuda.network import AdamW
    a, b = torch.zeros(8, device="cuda"), torch.zeros(4, device="cuda")
    opt = AdamW([a, b], **CFG)
    opt.step([torch.ones_like(a), None])
    was = a.clone()
    for lr in ([1e-3, np.nan], [np.inf, 1e-3]):
        opt.set_lr(lr)
        with pytest.raises(ValueError):
            opt.step([torch.ones_like(a), torch.ones_like(b)])
    assert torch.equal(a, was) and not b.any() and opt.state()["step"] == [1, 0]


def test_a_step_shows_in_the_versions_of_what_it_updates():
    import torch
    from splatx_cuda.network import AdamW
    a, b = (torch.zeros(8, device="cuda") for _ in range(2))
    versions = a._version, b._version
    AdamW([a, b], **CFG).step([torch.ones_like(a), None])
    assert a._version > versions[0] and b._version == versions[1]


def test_refused_while_a_graph_is_captured():
    """A captured step would take the same step number, with the same bias corrections, in every
    replay."""
    import torch
    from splatx_cuda.network import AdamW
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    opt = AdamW([p], **CFG)
    opt.step([g])
    was = p.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p * 2
        with pytest.raises(RuntimeError, match="captured"):
            opt.step([g])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p, was) and opt.state()["step"] == 1
    opt.step([g])
    assert opt.state()["step"] == 2 and not torch.equal(p, was)


def test_groups_take_rate_and_decay_and_nothing_else():
    """betas and eps are one for all parameters: a group's own, or a name with a slip, is refused
    instead of dropped."""
    import torch
    from splatx_cuda.network import AdamW
    p, o = torch.zeros(8, device="cuda"), torch.zeros(4, device="cuda")
    AdamW([{"params": [p], "lr": 0.1, "weight_decay": 0.0}, {"params": iter([o])}, {"params": []}])
    for bad in ({"betas": (0.5, 0.9)}, {"eps": 1e-4}, {"weigth_decay": 0.0}):
        with pytest.raises(ValueError, match=next(iter(bad))):
            AdamW([{"params": [p], **bad}])
    for bad in ([{"lr": 0.1}], [{"params": [p]}, o], [o, {"params": [p]}], [{"params": p}], ["p"], p, {"params": [p]}):
        with pytest.raises(ValueError):
            AdamW(bad)


def test_memory_that_is_updated_twice_is_refused():
    """Parameters and moments whose bytes overlap, whatever their starts, when the optimiser is made and
    when a parameter is given other memory later: two CTAs would read and write them without order."""
    import torch
    from splatx_cuda.network import AdamW
    flat, m, v = (torch.zeros(1024, device="cuda") for _ in range(3))
    state = lambda m0, m1, v0, v1: {"step": 0, "exp_avg": [m0, m1], "exp_avg_sq": [v0, v1]}  # noqa: E731
    m0, m1, v0, v1 = m[:512], m[512:], v[:512], v[512:]
    AdamW([flat[:512], flat[512:]], state=state(m0, m1, v0, v1))
    for params, st in (([flat[:512], flat[256:768]], None), ([flat[256:768], flat[:512]], None),
                       ([flat, flat[1000:1001]], None), ([flat[:512], flat[512:]], state(m0, m0, v0, v1)),
                       ([flat[:512], flat[512:]], state(m0, m1, v0, m1)),
                       ([flat[:512], flat[512:]], state(m0, m1, v[:512], v[511:1023])),
                       ([flat[:512], flat[512:]], state(m0, m1, v0, flat[512:])),
                       ([flat[:512].bfloat16(), flat.view(torch.float16)[:1], flat], None)):
        with pytest.raises(ValueError, match="overlap|more than once"):
            AdamW(params, state=st)
    a, b = (torch.nn.Parameter(torch.randn(600, device="cuda")) for _ in range(2))
    g = torch.randn(600, device="cuda")
    opt = AdamW([a, b], **CFG)
    opt.step([g, g])
    own = b.data
    for tied in (a.data, opt.state()["exp_avg"][0]):
        b.data = tied
        was = a.detach().clone(), [t.clone() for t in opt.state()["exp_avg"]]
        with pytest.raises(ValueError, match="overlap"):
            opt.step([g, g])
        assert torch.equal(a, was[0]) and all(torch.equal(x, y) for x, y in zip(opt.state()["exp_avg"], was[1]))
    b.data = own
    opt.step([g, g])
    assert opt.state()["step"] == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_the_moments_stay_the_optimisers_own(bits):
    """What state() hands out, and what the constructor was given, may be replaced or given other memory
    without changing where the next step reads and writes its moments."""
    import torch
    from splatx_cuda.network import AdamW
    gen = torch.Generator().manual_seed(3)
    t = lambda: torch.randn(900, generator=gen).cuda()  # noqa: E731
    p, grads = t(), [t() for _ in range(4)]
    q = p.clone()
    want, opt = AdamW([q], state_bits=bits, **CFG), AdamW([p], state_bits=bits, **CFG)
    want.step([grads[0]])
    opt.step([grads[0]])
    given = opt.state()
    opt = AdamW([p], state_bits=bits, state=given, **CFG)
    for i, g in enumerate(grads[1:]):
        want.step([g])
        for shown in (given, opt.state()) if i else ():
            for key in shown:
                if key != "step":
                    shown[key][0].data = torch.empty_like(shown[key][0])  # as when moments are moved away
                    shown[key][0] = None
                    shown[key].clear()
        given = opt.state()
        opt.step([g])
        assert torch.equal(p, q), i
    for key, tensors in want.state().items():
        if key != "step":
            assert torch.equal(opt.state()[key][0].view(torch.uint8), tensors[0].view(torch.uint8))


def test_a_parameter_moved_off_the_device_is_refused():
    import torch
    from splatx_cuda.network import AdamW
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    opt = AdamW([p], **CFG)
    opt.step([torch.ones(8, device="cuda")])
    was, p.data = p.data, p.data.cpu()
    with pytest.raises(ValueError):
        opt.step([torch.ones(8)])
    with pytest.raises(ValueError):
        opt.step([torch.ones(8, device="cuda")])
    p.data = was
    opt.step([torch.ones(8, device="cuda")])
    assert opt.state()["step"] == 2


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [8192, 700])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-38, 1e-30, 1e30, 3e38])
def test_divisors_at_the_ends_of_the_range(eps, n, bits):
    """Values without a gradient beside others: m / (0 + eps) is 0 for every eps above zero, also for one
    that 32 bits hold below 2^-126, and not a number for none; a divisor near the largest value leaves
    the weights as they are. In chunks of the fast path and in tails."""
    import torch
    from splatx_cuda.network import AdamW
    rng = np.random.default_rng(n)
    g = rng.standard_normal(n).astype(F)
    g[::3] = 0
    was = rng.standard_normal(n).astype(F)
    p = torch.from_numpy(was).cuda()
    cfg = {**CFG, "eps": eps}
    AdamW([p], state_bits=bits, **cfg).step([torch.from_numpy(g).cuda()])
    with np.errstate(invalid="ignore"):
        b1, b2 = CFG["betas"]
        m, v = g * F(1 - b1), (g * g) * F(1 - b2)
        d = np.sqrt(v) * F(1 / math.sqrt(1 - b2)) + F(eps)
        want = was * F(1 - CFG["lr"] * CFG["weight_decay"]) - m / d * F(CFG["lr"] / (1 - b1))
    assert np.array_equal(_np(p), want, equal_nan=True)
    assert np.isnan(want).any() == (eps == 0.0)


def test_numbers_that_32_bits_do_not_hold_are_refused():
    import torch
    from splatx_cuda.network import AdamW
    p, g = torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda")
    for f in (lambda: AdamW([p], eps=1e39).step([g]), lambda: AdamW([p], lr=-1e39).step([g]),
              lambda: AdamW([p], weight_decay=1e39).step([g]), lambda: AdamW([p]).step([g], grad_scale=1e39)):
        with pytest.raises(ValueError):
            f()
    assert not p.any()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [1 << 16, 1000])
def test_quotients_of_small_moments(n, bits):
    """Every bit from a moment of 2^-100 on; below that the quotient's last bit may be off, which moves
    the weight (zero before) by that much of itself, and a unit of the smallest numbers."""
    import torch
    from splatx_cuda.network import AdamW
    rng = np.random.default_rng(n)
    g = (rng.choice([-1, 1], n) * rng.uniform(1, 2, n) * 2.0 ** rng.uniform(-135, -60, n)).astype(F)
    p = torch.zeros(n, device="cuda")
    AdamW([p], state_bits=bits, **CFG).step([torch.from_numpy(g).cuda()])
    zero = np.zeros(n, F)
    want, m, _ = _numpy_step(zero, g, zero, zero, 1)
    exact = np.abs(m) >= 2.0 ** -100
    assert exact.any() and not exact.all() and np.array_equal(_np(p)[exact], want[exact])
    off = np.abs(_np(p).astype(np.float64) - want)
    assert np.all(off <= 2.0 ** -22 * np.abs(want.astype(np.float64)) + 2.0 ** -149)
