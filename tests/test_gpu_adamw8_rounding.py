"""Moments in 8 bits over many steps: rounded stochastically they follow their gradients, as moments in 32 bits do."""
import math

import numpy as np
import pytest
import torch

from comprex_amd import pygpi
from comprex_amd._lib import ComprexError
from comprex_amd.optimizer import ComprexAdamW

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
BLOCK = 256
KINDS = [(F32, F32, False, False), (BF16, BF16, False, False), (BF16, BF16, True, False), (F16, F32, True, False),
         (F16, F16, False, False), (F32, BF16, False, True), (BF16, BF16, False, True)]


class Small:
    """Tensors with 8-bit moments, back to zero before a step where that is asked for."""

    def __init__(self, sizes, param=F32, master=False):
        from comprex_amd import device as D
        self.p = [torch.zeros(n, dtype=param, device="cuda") for n in sizes]
        self.states = [D.AdamWSet.zeros8(p) for p in self.p]
        w = [p.float() for p in self.p] if master else None
        self.h = D.Handle()
        self.set = D.AdamWSet(self.h, self.p, *([s[k] for s in self.states] for k in (0, 1)), masters=w,
                              exp_avg_scales=[s[2] for s in self.states], exp_avg_sq_scales=[s[3] for s in self.states])
        self.moves = torch.zeros(sum(sizes), device="cuda")

    def zero(self):
        for s in self.states:
            for t in s:
                t.view(torch.uint8).zero_()

    def values(self):
        return self.h.adamw_states(self.set)


def neighbours(x, top, lowest_normal, step_below):
    """The step of the codes at x / top (a multiple of the smallest step; 3 fraction bits above the smallest normal)."""
    y = x / top
    e = torch.floor(torch.log2(torch.clamp(y, min=lowest_normal)))
    return torch.where(y < lowest_normal, step_below, 2.0 ** (e - 3)) * top


@pytest.mark.parametrize("param,grad,master,moves", KINDS, ids=str)
def test_codes_are_neighbours_of_their_values_and_right_on_average(param, grad, master, moves):
    """One step from zero moments, 400 times with other seeds.  A stored value is one of its value's two neighbours, at
    most one code step away (with the roundings that lead to it, below 8 u of it).  Its mean over T seeds differs from it by
    more than t steps with a probability of at most 2 exp(-2 T t^2) (Hoeffding; T = 400, t = 0.17: 2e-10 for each of 2 * 3306
    values); 16 random bits give the probability to 2^-16."""
    T, t = 400, 0.17
    sizes = [1, 255, 257, 2049, 744]
    S = Small(sizes, param, master)
    gen = torch.Generator(device="cuda").manual_seed(1)
    g = torch.empty(sum(sizes), device="cuda").normal_(generator=gen).exp() * torch.empty(sum(sizes), device="cuda").normal_(generator=gen)
    g = g.to(grad)
    grads = list(g.split(sizes))
    m, v = 0.1 * g.double(), 0.001 * g.double() ** 2
    mean_m, mean_v = torch.zeros_like(m), torch.zeros_like(v)
    sizes_of_blocks = [min(BLOCK, n - b) for n in sizes for b in range(0, n, BLOCK)]
    lengths = torch.tensor(sizes_of_blocks, device="cuda")
    tops = [torch.segment_reduce(x.abs(), "max", lengths=lengths).repeat_interleave(lengths) for x in (m, v)]
    # e4m3: 448 the largest, 2^-6 the smallest normal; the other: 2^30 * 1.875 the largest, code 8 the smallest normal
    step_m = neighbours(m.abs(), tops[0] / 448.0, 2.0 ** -6, 2.0 ** -9)
    step_v = neighbours(v, tops[1] / (1.875 * 2.0 ** 30), 1.0, 0.125)
    kept = None
    for seed in range(1, T + 1):
        S.zero()
        S.h.adamw_step(S.set, grads, 1, 0.0, seed=seed, moves=S.moves if moves else None)
        got_m, got_v = (x.double() for x in S.values())
        assert ((got_m - m).abs() < step_m * (1 + 1e-6) + 8 * U * m.abs()).all()
        assert ((got_v - v).abs() < step_v * (1 + 1e-6) + 8 * U * v).all()
        assert (got_v[v > 0] > 0).all()
        mean_m += got_m / T
        mean_v += got_v / T
        if seed == 7:
            kept = got_m, got_v
    assert ((mean_m - m).abs() <= step_m * (t + 2.0 ** -16) + 8 * U * m.abs()).all()
    above = v >= 0.125 * tops[1] / (1.875 * 2.0 ** 30)   # (below the lowest code nothing becomes 0)
    assert ((mean_v - v).abs() <= step_v * (t + 2.0 ** -16) + 8 * U * v)[above].all()
    # the same seed gives the same bits, and so does a count on the device; another step gives others
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    for step in (1, count):
        S.zero()
        S.h.adamw_step(S.set, grads, step, 0.0, seed=7, moves=S.moves if moves else None)
        assert all(torch.equal(a.double(), b) for a, b in zip(S.values(), kept))
    S.zero()
    S.h.adamw_step(S.set, grads, 2, 0.0, seed=7)
    assert not any(torch.equal(a.double(), b) for a, b in zip(S.values(), kept))


def test_what_is_not_finite_and_what_lies_on_a_code():
    """An infinity or NaN: exp_avg NaN, exp_avg_sq the largest, the others as without it.  A gradient of one size: every
    moment is its block's largest, which has a code of its own whatever the noise, and stays on it."""
    S, T = Small([1000]), Small([1000])
    g = torch.full((1000,), 3.0, device="cuda")
    bad = g.clone()
    bad[5], bad[300], bad[999] = math.inf, math.nan, -math.inf
    fine = torch.isfinite(bad)
    for step in range(1, 60):
        S.h.adamw_step(S.set, [bad], step, 0.0, seed=step)
        T.h.adamw_step(T.set, [g], step, 0.0, seed=step)
    m, v = S.values()
    assert torch.isnan(m[~fine]).all() and (S.states[0][1][~fine] == 255).all()
    want = 3.0 * (1 - 0.9 ** 59), 9.0 * (1 - 0.999 ** 59)
    for x, y, w in ((m, T.values()[0], want[0]), (v, T.values()[1], want[1])):
        assert torch.equal(x[fine], y[fine])
        # 59 steps, each with at most 8 roundings of a sum that only grows
        assert ((x[fine].double() - w).abs() <= 59 * 8 * U * w).all()


def steady(gen, n, step):
    return torch.empty(n, device="cuda").normal_(generator=gen)


def dropped(gen, n, step):
    """Every other gradient becomes ten times smaller."""
    g = steady(gen, n, step)
    if step > 1500:
        g[::2] *= 0.1
    return g


def spiked(gen, n, step):
    """One element of every block sees one large gradient."""
    g = steady(gen, n, step)
    if step == 1500:
        g[::BLOCK] = 100.0
    return g


def stopped(gen, n, step):
    """Every other gradient ends."""
    g = steady(gen, n, step)
    if step > 1500:
        g[::2] = 0.0
    return g


# What noise may do.  With X = v8 - v32: X' = beta2 X + xi, xi of mean 0 and of variance (code step) * |way from the code|.  A
# code step is at most v/8; the way is at most 0.001 (|g^2 / v - 1| + |the same of the block's largest|) v, on average
# at most 0.001 * 2 sqrt(2) v for normal gradients.  So a variance of at most 3.6e-4 v^2 a step.  Steady: 3.6e-4 / (1 - beta2^2) =
# 0.18 v^2.  While v falls by 0.1 % a step the noise of before stays as large beside it: 3.6e-4 v^2 for each step of the fall,
# 5000 * 3.6e-4 = 1.8 v^2 at most.  The noises of N elements are uncorrelated (up to 0.02 for neighbours): their mean is off by 6 sqrt(var / N) with a
# probability below 1e-8 (and a sample of squares by a third: N = 4096).
@pytest.mark.parametrize("gradients,steps,var", [(steady, 3000, 0.18), (dropped, 6500, 1.8), (spiked, 4500, 0.18)])
@pytest.mark.parametrize("param", [F32, BF16], ids=str)
def test_second_moments_follow_their_gradients(param, gradients, steps, var):
    n = 8192
    S = Small([n], param)
    gen = torch.Generator(device="cuda").manual_seed(2)
    v32 = torch.zeros(n, device="cuda")
    for step in range(1, steps + 1):
        g = gradients(gen, n, step)
        S.h.adamw_step(S.set, [g], step, 0.0, seed=11)
        v32.mul_(0.999).addcmul_(g, g, value=0.001)
    ratio = S.values()[1].double() / v32.double()
    for part in (ratio[::2], ratio[1::2]):
        assert abs(float(part.mean()) - 1) <= 6 * math.sqrt(var / part.numel()), float(part.mean())
        assert float(((part - 1) ** 2).mean()) <= var * 4 / 3, float(((part - 1) ** 2).mean())


def test_first_moments_end_with_their_gradients():
    """1500 steps without a gradient: 0.9^1500 of it is left in expectation, nothing of any element."""
    n = 8192
    S = Small([n])
    gen = torch.Generator(device="cuda").manual_seed(3)
    for step in range(1, 3001):
        S.h.adamw_step(S.set, [stopped(gen, n, step)], step, 0.0, seed=5)
    m, v = S.values()
    assert m[::2].count_nonzero() == 0 and m[1::2].count_nonzero() > 0 and (v > 0).all()


def test_the_optimizer_rounds_its_moments_so():
    """ComprexAdamW, one large gradient: 2500 steps later the other elements' second moments are those of a run in 32 bits,
    on average over N = 8160 of them (bounds as above), and its weights have not run away from that run's."""
    n = 8192
    env = pygpi.GaspiEnvironment()
    runs = [torch.nn.Parameter(torch.zeros(n, device="cuda")) for _ in range(2)]
    opts = [ComprexAdamW([p], env, learning_rate=1e-3, weight_decay=0.0, state_bits=b) for p, b in zip(runs, (32, 8))]
    gen = torch.Generator(device="cuda").manual_seed(4)
    for step in range(1, 4001):
        g = spiked(gen, n, step)
        for p, opt in zip(runs, opts):
            p.grad = g.clone()
            opt.step()
    part = opts[1]._parts[0]
    v8, v32 = opts[1].handle.adamw_states(part.set)[1].double(), opts[0].state[runs[0]]["exp_avg_sq"].double()
    others = torch.arange(n, device="cuda") % BLOCK != 0
    ratio = (v8 / v32)[others]
    assert abs(float(ratio.mean()) - 1) <= 6 * math.sqrt(0.18 / ratio.numel())
    assert float(((ratio - 1) ** 2).mean()) <= 0.24


def test_seeds_that_are_none():
    S = Small([300])
    g = [torch.ones(300, device="cuda")]
    for seed in (0, -1, 1 << 64):
        with pytest.raises(ComprexError):
            S.h.adamw_step(S.set, g, 1, 1e-3, seed=seed)
    S.h.adamw_step(S.set, g, 1, 1e-3, seed=(1 << 64) - 1)
    assert np.isfinite(S.values()[0].cpu().numpy()).all()


@pytest.mark.parametrize("seed", [None, 3])
@pytest.mark.parametrize("dtype,bits", [(F32, 0x7fc00000), (F32, 0xffc00000), (F32, 0x7fffffff), (F32, 0xffffffff), (F32, 0xff800001),
                                        (BF16, 0xffff), (BF16, 0x7fff), (F16, 0xffff), (F16, 0xfe00)], ids=str)
def test_every_nan_is_stored_as_the_blocks_largest(dtype, bits, seed):
    """Whatever its sign and payload: exp_avg NaN, exp_avg_sq code 255, and the others as they are without it."""
    S, T = Small([600]), Small([600])
    g = torch.ones(600, dtype=dtype, device="cuda")
    g[1::2] = 0.25
    bad = g.clone()
    word = torch.int32 if dtype == F32 else torch.int16
    width = 8 * dtype.itemsize
    bad.view(word)[5] = bits - (1 << width) if bits >> (width - 1) else bits
    assert torch.isnan(bad[5])
    S.h.adamw_step(S.set, [bad], 1, 0.0, seed=seed)
    T.h.adamw_step(T.set, [g], 1, 0.0, seed=seed)
    (m, v), (m0, v0) = S.values(), T.values()
    assert torch.isnan(m[5]) and S.states[0][1][5] == 255
    m[5], v[5] = m0[5], v0[5]
    assert torch.equal(m, m0) and torch.equal(v, v0)


@pytest.mark.parametrize("moves", [False, True])
def test_a_captured_step_rounds_with_each_replays_count(moves):
    """A step with its count on the device, captured and replayed, has the bits of the eager steps 1, 2, ..."""
    from comprex_amd import device as D
    sizes = [3000, 5, 513]
    A, B = Small(sizes, BF16, True), Small(sizes, BF16, True)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        B.h = D.Handle(side)
        fixed = [torch.zeros(n, dtype=BF16, device="cuda") for n in sizes]
        count = torch.zeros(1, dtype=torch.int32, device="cuda")

    def step(S, grads, at):
        S.h.adamw_step(S.set, grads, at, 1e-3, seed=9, moves=S.moves if moves else None)
        if moves:
            S.h.adamw_apply(S.set, S.moves, 1e-3)

    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(B, fixed, count)
    torch.cuda.synchronize()
    gen = torch.Generator(device="cuda").manual_seed(6)
    for k in range(1, 7):
        grads = [torch.empty(n, device="cuda").normal_(generator=gen).to(BF16) for n in sizes]
        step(A, grads, k)
        for f, g in zip(fixed, grads):
            f.copy_(g)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert count.item() == k
        assert all(torch.equal(p, q) for p, q in zip(A.p, B.p))
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for s, t in zip(A.states, B.states) for x, y in zip(s, t))
