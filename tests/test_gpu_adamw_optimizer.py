"""ComprexAdamW: clip, step and exchange as they are used together, against the formulas in 64 bits and itself
before and after a checkpoint."""
import copy
import math
import threading

import numpy as np
import pytest
import torch

from comprex_amd import pygpi
from comprex_amd.optimizer import ComprexAdamW

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16 = torch.bfloat16


def f64(t):
    return t.detach().double().cpu().numpy()


def parameter(values, dtype=torch.float32):
    return torch.nn.Parameter(torch.as_tensor(values).to(dtype).cuda())


class Formula:
    """AdamW of one tensor in 64 bits."""

    def __init__(self, w):
        self.w, self.m, self.v, self.t = w.copy(), np.zeros_like(w), np.zeros_like(w), 0

    def step(self, g, lr, wd, b1=0.9, b2=0.999, eps=1e-8):
        self.t += 1
        self.m = b1 * self.m + (1 - b1) * g
        self.v = b2 * self.v + (1 - b2) * g * g
        self.w = self.w - lr * wd * self.w - lr / (1 - b1 ** self.t) * self.m / (
            np.sqrt(self.v / (1 - b2 ** self.t)) + eps)


def within(p, want, steps, lr):
    """After n steps from zero moments: a moment's error is at most 10 u a step of the largest |g| so far (8 roundings
    a step, and the clip's 3), and the root of the corrected second moment is at least max|g| * sqrt(b2^n / n)
    (n <= 10: above max|g| / 3.2), so a step's move is wrong by at most lr * (3.2 * 10 u n + its own 20 u * 3.2), and a
    weight by 2 u of itself a step on top."""
    tol = steps * (lr * 3.2 * (10 * steps + 20) * U + 2 * U * np.abs(want)) + 1e-12
    assert (np.abs(f64(p) - want) <= tol).all(), np.abs(f64(p) - want).max()


def test_one_rank_follows_the_formula():
    """Two groups, a clip that bites, and a parameter that goes without a gradient for two steps: its own count."""
    env = pygpi.GaspiEnvironment()
    rng = np.random.default_rng(1)
    shapes = [(70, 33), (1,), (5000,), (257,)]
    start = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    params = [parameter(x) for x in start]
    opt = ComprexAdamW([{"params": params[:2], "weight_decay": 0.1}, {"params": params[2:], "lr": 3e-3}], env,
                       learning_rate=1e-2, weight_decay=0.0, clip_norm=1.0)
    want = [Formula(f64(p)) for p in params]
    for step in range(6):
        grads = [rng.standard_normal(s).astype(np.float32) * (0.001 if step == 3 else 1) for s in shapes]
        missing = step in (1, 2)
        for k, (p, g) in enumerate(zip(params, grads)):
            p.grad = None if missing and k == 3 else torch.from_numpy(g).cuda()
        live = [k for k in range(4) if not (missing and k == 3)]
        norm = math.sqrt(sum(float((grads[k].astype(np.float64) ** 2).sum()) for k in live))
        coef = min(1.0, 1.0 / norm)
        opt.step()
        for k in live:
            want[k].step(grads[k].astype(np.float64) * coef, (1e-2, 1e-2, 3e-3, 3e-3)[k], (0.1, 0.1, 0.0, 0.0)[k])
    assert [opt.state[p]["step"] for p in params] == [6, 6, 6, 4]
    for p, f, lr in zip(params, want, (1e-2, 1e-2, 3e-3, 3e-3)):
        within(p, f.w, 6, lr)


def test_gradients_of_other_layouts_and_frozen_parameters():
    env = pygpi.GaspiEnvironment()
    rng = np.random.default_rng(2)
    a, b = parameter(rng.standard_normal((40, 30)).astype(np.float32)), parameter(np.ones(10, np.float32))
    b.requires_grad_(False)
    opt = ComprexAdamW([a, b], env, learning_rate=1e-2, weight_decay=0.0)
    want = Formula(f64(a))
    for _ in range(3):
        g = rng.standard_normal((30, 40)).astype(np.float32)
        a.grad = torch.from_numpy(g).cuda().t()  # strided
        opt.step()
        want.step(g.T.astype(np.float64), 1e-2, 0.0)
    within(a, want.w, 3, 1e-2)
    assert (b == 1).all()
    a.grad = None
    before = a.detach().clone()
    opt.step()  # nobody has a gradient
    assert torch.equal(a, before)


@pytest.mark.parametrize("bits", [32, 8])
def test_masters_and_a_checkpoint(bits):
    """bf16 parameters with masters beside fp32 ones: the parameter is its master rounded, and a run that goes on
    from a saved state has the bits of one that was never interrupted."""
    env = pygpi.GaspiEnvironment()
    rng = np.random.default_rng(3)
    shapes = [(100, 300), (9,), (4096,), (5, 1001)]
    types = [BF16, BF16, torch.float32, torch.float32]
    start = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    grads = [[torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda().to(t) for s, t in zip(shapes, types)]
             for _ in range(6)]

    def make():
        params = [parameter(x, t) for x, t in zip(start, types)]
        return params, ComprexAdamW(params, env, learning_rate=1e-2, clip_norm=50.0, state_bits=bits)

    def run(params, opt, steps):
        for gs in steps:
            for p, g in zip(params, gs):
                p.grad = g.clone()
            opt.step()

    params, opt = make()
    run(params, opt, grads)
    for p in params:
        s = opt.state[p]
        assert ("master" in s) == (p.dtype == BF16) and ("exp_avg_scales" in s) == (bits == 8 and p.numel() >= 4096)
        if p.dtype == BF16:
            assert torch.equal(s["master"].to(BF16), p)
    again, first = make()
    run(again, first, grads[:3])
    saved = copy.deepcopy(first.state_dict())
    kept = [p.detach().clone() for p in again]
    run(again, first, grads[3:])  # goes on by itself: the saved state is not touched by it
    others = [torch.nn.Parameter(p) for p in kept]
    second = ComprexAdamW(others, env, learning_rate=1.0, clip_norm=50.0, state_bits=bits)
    second.load_state_dict(saved)
    run(others, second, grads[3:])
    for p, q, r in zip(params, again, others):
        assert torch.equal(p, q) and torch.equal(p, r)
        a, b = opt.state[p], second.state[r]
        assert a.keys() == b.keys() and a["step"] == b["step"] == 6
        for k in a:
            if k != "step":
                assert a[k].dtype == b[k].dtype and torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8))


def test_8bit_moments_stay_near_the_32bit_ones():
    """Each stored moment is within half a step of 3 fraction bits of its value, 2^-4, and what a step adds to it is
    exact: with decaying weights b^k of past roundings the first moment is within 2^-4 / (1 - 0.9) of the block's
    scale of rounding of the 32-bit run's."""
    env = pygpi.GaspiEnvironment()
    rng = np.random.default_rng(4)
    x = rng.standard_normal(8192).astype(np.float32)
    a, b = parameter(x), parameter(x)
    opts = [ComprexAdamW([p], env, learning_rate=1e-3, state_bits=bits) for p, bits in ((a, 32), (b, 8))]
    for _ in range(10):
        g = torch.from_numpy(rng.standard_normal(8192).astype(np.float32)).cuda()
        for p, opt in zip((a, b), opts):
            p.grad = g.clone()
            opt.step()
    part = opts[1]._parts[0]
    m, v = opts[1].handle.adamw_states(part.set)
    m32, v32 = opts[0].state[a]["exp_avg"], opts[0].state[a]["exp_avg_sq"]
    top = m32.abs().view(-1, 256).amax(1).repeat_interleave(256)
    # every past value lies below 1.2 times the largest of now times (1 / 0.9)^k; roundings decay with 0.9^k
    assert ((m - m32).abs() <= 2.0 ** -4 * 1.3 * 10 * top).all()
    # v only grows here (0.999^10 = 0.99): each of the 10 roundings is at most 2^-4 of what is there then
    assert (v <= v32 * (1 + 2.0 ** -4) ** 10).all() and (v >= v32 * (1 - 2.0 ** -4) ** 10).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_nonfinite_gradients_are_skipped(bits):
    env = pygpi.GaspiEnvironment()
    rng = np.random.default_rng(5)
    x = [rng.standard_normal(n).astype(np.float32) for n in (5000, 30)]
    runs = [[parameter(v) for v in x] for _ in range(2)]
    opts = [ComprexAdamW(p, env, learning_rate=1e-2, clip_norm=1.0, state_bits=bits, skip_nonfinite=True) for p in runs]
    for step in range(4):
        gs = [torch.from_numpy(rng.standard_normal(v.size).astype(np.float32)).cuda() for v in x]
        for ps, opt in zip(runs, opts):
            for p, g in zip(ps, gs):
                p.grad = g.clone()
        if step == 2:  # one of the runs sees a bad step before the good one
            runs[1][1].grad[7] = math.inf if bits == 8 else math.nan
            before = [p.detach().clone() for p in runs[1]]
            opts[1].step()
            assert all(torch.equal(p, q) for p, q in zip(runs[1], before))
            runs[1][1].grad.copy_(gs[1])
        for opt in opts:
            opt.step()
    for p, q in zip(*runs):
        assert torch.equal(p, q)
    steps = [[s["step"] for s in opt.state_dict()["state"].values()] for opt in opts]
    assert steps == [[4, 4], [4, 4]]
    # the count goes on from a saved state, and a group that joins does not reset it
    more = parameter(np.ones(5, np.float32))
    opts[0].add_param_group({"params": [more]})
    for p in runs[0] + [more]:
        p.grad = torch.ones_like(p)
    opts[0].step()
    assert [s["step"] for s in opts[0].state_dict()["state"].values()] == [5, 5, 1]


def run_ranks(R, program):
    """Each rank's program in a thread of its own."""
    env = pygpi.GaspiEnvironment()
    env.set_rank(0, R)
    env.set_blocking(True, 60.0)
    errors = []

    def rank_program(rank):
        try:
            env.set_rank(rank, R)
            program(env, rank)
            env.barrier()
        except Exception as e:  # noqa: BLE001
            errors.append((rank, repr(e)))

    threads = [threading.Thread(target=rank_program, args=(r,)) for r in range(R)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(180)
    assert not errors, errors


def flush_and_apply(opt, ranks):
    """What the exchange still holds back, applied like a step (without decay)."""
    opt.blob.zero_()
    opt.allreduce.flush(opt.blob)
    at = 0
    for part in opt._parts:
        opt.handle.adamw_apply(part.set, opt.blob[at:at + part.set.total], 0.0, 0.0, scale=1.0 / ranks)
        at += part.set.total


@pytest.mark.parametrize("side_stream", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("schedule", ["comprex_alltoone", "comprex_ring", "comprex_bigring"])
def test_ranks_end_with_the_sum_of_their_moves(schedule, bits, side_stream):
    """Three ranks as threads, each with gradients of its own: where the schedule delivers everything by the flush
    (the big ring on every rank, all-to-one on the chief) the weights are w0 less a third of the sum of all ranks' moves,
    each rank's from moments of its own gradients.  In 8 bits, whose moves no formula in 64 bits follows, the big ring's
    ranks agree."""
    R, steps, sizes, lr = 3, 4, [(70, 60), (5,), (300,)], 1e-2
    rng = np.random.default_rng(6)
    n = 70 * 60 + 5 + 300
    grads = rng.standard_normal((R, steps, n)).astype(np.float32)
    w0 = rng.standard_normal(n).astype(np.float32)
    got = {}

    def program(env, rank):
        stream = torch.cuda.Stream() if side_stream else torch.cuda.default_stream()
        with torch.cuda.stream(stream):
            params, at = [], 0
            for s in sizes:
                k = int(np.prod(s))
                params.append(parameter(w0[at:at + k].reshape(s)))
                at += k
            opt = ComprexAdamW(params, env, learning_rate=lr, weight_decay=0.0, state_bits=bits,
                               allreduce_type=schedule, compression_ratio=0.05, size_factor=3.0)
            for step in range(steps):
                env.barrier()
                at = 0
                for p in params:
                    p.grad = torch.from_numpy(grads[rank, step, at:at + p.numel()]).cuda().view_as(p)
                    at += p.numel()
                opt.step()
            env.barrier()
            flush_and_apply(opt, R)
            stream.synchronize()
            got[rank] = np.concatenate([f64(p).reshape(-1) for p in params])

    run_ranks(R, program)
    assert len(got) == R and all(np.isfinite(x).all() for x in got.values())
    moved = np.zeros(n)
    for rank in range(R):
        f = Formula(np.zeros(n))
        for step in range(steps):
            before = f.w
            f.step(grads[rank, step].astype(np.float64), lr, 0.0)
            moved += before - f.w
            f.w = np.zeros(n)
    want = w0.astype(np.float64) - moved / R
    # a move's error as in `within`; on their way at most steps * R additions of at most the sum of all moves, each
    # below 3.2 lr; steps + 1 subtractions from the weight, each with the product by 1 / R before it
    tol = (steps * lr * 3.2 * (10 * steps + 20) * U + U * (steps * R) ** 2 * 3.2 * lr / R
           + 2 * (steps + 2) * U * (np.abs(w0) + steps * 3.2 * lr))
    checked = {"comprex_bigring": range(R), "comprex_alltoone": [0], "comprex_ring": []}[schedule]
    for rank in checked:
        if bits == 32:
            assert (np.abs(got[rank] - want) <= tol).all(), (rank, np.abs(got[rank] - want).max())
        else:
            assert (np.abs(got[rank] - got[checked[0]]) <= 2 * tol).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_rank_with_a_nonfinite_gradient_adds_nothing(bits):
    """Two ranks, constant gradients: a first step moves every weight by lr whatever the gradient's size.  Rank 1's first
    one holds a NaN: it adds nothing then, and its second step is its first."""
    lr, got = 2.0 ** -7, {}

    def program(env, rank):
        p, q = parameter(np.zeros(5000, np.float32)), parameter(np.zeros(10, np.float32))
        opt = ComprexAdamW([p, q], env, learning_rate=lr, weight_decay=0.0, state_bits=bits, skip_nonfinite=True,
                           compression_ratio=0.5, size_factor=3.0)
        for step in range(2):
            env.barrier()
            p.grad = torch.full((5000,), float(rank + 1), device="cuda")
            q.grad = None if rank == 0 else torch.ones(10, device="cuda")
            if rank == 1 and step == 0:
                p.grad[3] = math.nan
            opt.step()
        env.barrier()
        flush_and_apply(opt, 2)
        torch.cuda.synchronize()
        got[rank] = f64(p), f64(q), opt.state_dict()["state"][0]["step"]

    run_ranks(2, program)
    for rank in range(2):
        p, q, count = got[rank]
        assert count == 2 - rank
        # m / sqrt(v) of a constant gradient is 1 up to 20 roundings (constants of beta and the rates among them), and
        # in 8 bits the largest of a block is stored within 2 u of itself; eps is 1e-8 of it
        assert (np.abs(p + lr * 3 / 2) <= lr * (60 * U + 4e-8)).all() and (np.abs(q + lr / 2) <= lr * (30 * U + 2e-8)).all()


def test_tensors_that_move_and_streams_that_change():
    """A parameter's storage or state replaced between steps, and steps on another stream: nothing stale."""
    env = pygpi.GaspiEnvironment()
    rng = np.random.default_rng(7)
    p = parameter(rng.standard_normal(5000).astype(np.float32))
    opt = ComprexAdamW([p], env, learning_rate=1e-2, weight_decay=0.0)
    want = Formula(f64(p))
    side = torch.cuda.Stream()
    for step in range(5):
        g = rng.standard_normal(5000).astype(np.float32)
        p.grad = torch.from_numpy(g).cuda()
        if step == 2:
            p.data = p.detach().clone()
        if step == 3:
            opt.state[p]["exp_avg"] = opt.state[p]["exp_avg"].clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(side if step % 2 else torch.cuda.default_stream()):
            opt.step()
        torch.cuda.synchronize()
        want.step(g.astype(np.float64), 1e-2, 0.0)
    within(p, want.w, 5, 1e-2)


def test_parameters_that_are_released_later():
    env = pygpi.GaspiEnvironment()
    a, b = parameter(np.ones(10, np.float32)), parameter(np.ones(10, np.float32))
    b.requires_grad_(False)
    opt = ComprexAdamW([a, b], env, learning_rate=0.5, weight_decay=0.0, skip_nonfinite=True)
    a.grad = torch.ones_like(a)
    opt.step()
    b.requires_grad_(True)
    b.grad = torch.ones_like(b)
    versions = a._version, b._version
    opt.step()
    assert (a.detach().cpu() - 0.0).abs().max() < 1e-5      # two moves of 0.5
    assert ((b.detach().cpu() - 0.5).abs() < 1e-5).all()    # one
    assert a._version > versions[0] and b._version > versions[1]   # autograd sees the weights change


def test_a_state_of_torchs_own_adamw_is_taken():
    """fp32 moments and counts of torch.optim.AdamW: the same formula goes on from them."""
    env = pygpi.GaspiEnvironment()
    rng = np.random.default_rng(9)
    x = rng.standard_normal(3000).astype(np.float32)
    p, q = parameter(x), parameter(x)
    theirs = torch.optim.AdamW([p], lr=1e-2, weight_decay=0.1)
    ours = ComprexAdamW([q], env, learning_rate=1e-2, weight_decay=0.1)
    want = Formula(f64(p))
    for step in range(6):
        g = rng.standard_normal(3000).astype(np.float32)
        if step == 3:
            with torch.no_grad():
                q.copy_(p)
            saved = theirs.state_dict()
            saved["param_groups"] = ours.state_dict()["param_groups"]
            ours.load_state_dict(saved)
        opt, w = (theirs, p) if step < 3 else (ours, q)
        w.grad = torch.from_numpy(g).cuda()
        opt.step()
        want.step(g.astype(np.float64), 1e-2, 0.1)
    assert ours.state[q]["step"] == 6
    within(q, want.w, 6, 1e-2)


def test_gradients_of_two_types_are_clipped_together():
    env = pygpi.GaspiEnvironment()
    rng = np.random.default_rng(8)
    x = [rng.standard_normal(n).astype(np.float32) for n in (5000, 300, 20)]
    types = [torch.float32, BF16, torch.float32]
    ps = [parameter(v, d) for v, d in zip(x, types)]
    opt = ComprexAdamW(ps, env, learning_rate=1e-2, weight_decay=0.0, clip_norm=1.0, skip_nonfinite=True)
    want = [Formula(f64(p)) for p in ps]
    for step in range(3):
        for p, v in zip(ps, x):
            p.grad = torch.from_numpy(rng.standard_normal(v.size).astype(np.float32)).cuda().to(p.dtype)
        gs = [f64(p.grad) for p in ps]
        coef = min(1.0, 1.0 / math.sqrt(sum(float((g * g).sum()) for g in gs)))
        opt.step()
        for f, g in zip(want, gs):
            f.step(g * coef, 1e-2, 0.0)
    for p, f in zip(ps, want):
        within(opt.state[p].get("master", p), f.w, 3, 1e-2)
    before = [p.detach().clone() for p in ps]
    ps[1].grad[4] = math.inf  # one type's, but all are skipped
    opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, before))


def test_another_layout_starts_another_exchange():
    """Two parameters of one size, one frozen and then the other: what was held back for the first is not the second's."""
    def program(env, rank):
        a, b = parameter(np.zeros(100, np.float32)), parameter(np.zeros(100, np.float32))
        b.requires_grad_(False)
        opt = ComprexAdamW([a, b], env, learning_rate=1.0, weight_decay=0.0, compression_ratio=0.05, size_factor=3.0)
        a.grad = torch.arange(1.0, 101.0, device="cuda")
        opt.step()
        a.requires_grad_(False)
        b.requires_grad_(True)
        env.barrier()
        b.grad = torch.zeros(100, device="cuda")
        opt.step()
        assert b.count_nonzero() == 0

    run_ranks(2, program)


def test_an_exchange_of_too_many_elements_is_refused(monkeypatch):
    from comprex_amd import optimizer
    monkeypatch.setattr(optimizer, "_MOST_EXCHANGED", 99)
    env = pygpi.GaspiEnvironment()
    env.set_rank(0, 2)
    p = parameter(np.ones(100, np.float32))
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError):
        ComprexAdamW([p], env).step()


def test_refusals():
    env = pygpi.GaspiEnvironment()
    p = parameter(np.ones(10, np.float32))
    for bad in (dict(allreduce_type="nope"), dict(state_bits=16), dict(clip_norm=0.0), dict(betas=(1.0, 0.9))):
        with pytest.raises(ValueError):
            ComprexAdamW([p], env, **bad)
    for q in (torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(6, 4, device="cuda").t()),
              torch.nn.Parameter(torch.zeros(3, dtype=torch.float64, device="cuda"))):
        with pytest.raises(ValueError):
            ComprexAdamW([q], env)
    opt = ComprexAdamW([p], env)
    p.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.tensor([1.0]), (10,)).cuda()
    with pytest.raises(RuntimeError):
        opt.step()


def recording(monkeypatch):
    """Every exchange keeps what it was given, by the thread and the exchange: {(thread, exchange): [vector, ...]}."""
    from comprex_amd import optimizer
    make, given = optimizer._make_allreduce, {}

    def made(*args):
        exchange = make(*args)
        apply = exchange.apply

        def recorded(vector):
            given.setdefault((threading.get_ident(), id(exchange)), []).append(vector.clone())
            return apply(vector)

        exchange.apply = recorded
        return exchange

    monkeypatch.setattr(optimizer, "_make_allreduce", made)
    return given


def check_sums(got, w0, vectors, where, steps, R):
    """Weights w0 less an R-th of the sum of all ranks' vectors.  With A the sum of their sizes: fewer than 2 steps R additions
    on the way, and for each of steps + 1 updates of a weight a product and a difference."""
    total = sum(f64(v) for v in vectors)
    size = sum(np.abs(f64(v)) for v in vectors)
    tol = (2 * steps * R * size / R + 2 * (steps + 2) * (np.abs(w0) + size / R)) * U
    off = np.abs(got - (w0.astype(np.float64) - total / R))
    assert (off <= tol)[where].all(), off[where].max()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("schedule", ["comprex_alltoone", "comprex_ring", "comprex_bigring"])
def test_what_ranks_put_into_the_exchange_arrives(schedule, bits, monkeypatch):
    """Two optimizers on streams of their own share an environment, three ranks.  After a flush the weights are w0 less a
    third of all that the ranks put in: with the big ring on every rank, with all-to-one on the chief, with the ring (whose
    broadcast drops what it does not send) on the rank where a segment's sum is made."""
    R, steps, sizes = 3, 4, [[(70, 60), (5,), (300,)], [(5000,), (33, 3)]]
    rng = np.random.default_rng(12)
    totals = [sum(int(np.prod(s)) for s in of) for of in sizes]
    w0 = [rng.standard_normal(n).astype(np.float32) for n in totals]
    grads = [rng.standard_normal((R, steps, n)).astype(np.float32) for n in totals]
    given, got, who = recording(monkeypatch), {}, {}

    def program(env, rank):
        who[threading.get_ident()] = rank
        runs = []
        for of, w in zip(sizes, w0):
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                params, at = [], 0
                for s in of:
                    k = int(np.prod(s))
                    params.append(parameter(w[at:at + k].reshape(s)))
                    at += k
                runs.append((stream, params, ComprexAdamW(params, env, learning_rate=1e-2, weight_decay=0.0, state_bits=bits,
                                                          allreduce_type=schedule, compression_ratio=0.05, size_factor=3.0)))
        for step in range(steps):
            for k, (stream, params, opt) in enumerate(runs):
                with torch.cuda.stream(stream):
                    at = 0
                    for p in params:
                        p.grad = torch.from_numpy(grads[k][rank, step, at:at + p.numel()]).cuda().view_as(p)
                        at += p.numel()
                    opt.step()
        for k, (stream, params, opt) in enumerate(runs):
            with torch.cuda.stream(stream):
                opt.flush()
            stream.synchronize()
            # in the vector's order: moments in 8 bits and in 32 lie apart
            order = [p for part in opt._parts for p in part.params]
            start = torch.cat([torch.from_numpy(w).cuda() for w in np.split(w0[k], np.cumsum([p.numel() for p in params])[:-1])])
            places = {id(p): x for p, x in zip(params, start.split([p.numel() for p in params]))}
            got[k, rank] = (np.concatenate([f64(p).reshape(-1) for p in order]),
                            np.concatenate([f64(places[id(p)]) for p in order]), id(opt.allreduce))
        env.barrier()
        for _, _, opt in runs:
            opt.allreduce.apply = None  # (the wrapper keeps its exchange alive)

    run_ranks(R, program)
    for k, n in enumerate(totals):
        vectors = [v for (thread, exchange), those in given.items() for v in those if exchange == got[k, who[thread]][2]]
        assert len(vectors) == R * steps
        segments = [n // R + (i < n % R) for i in range(R)]
        starts = np.cumsum([0] + segments)
        for rank in range(R):
            where = np.zeros(n, bool)
            if schedule == "comprex_bigring" or (schedule == "comprex_alltoone" and rank == 0):
                where[:] = True
            if schedule == "comprex_ring":
                mine = (rank + 1) % R
                where[starts[mine]:starts[mine + 1]] = True
            weights, start, _ = got[k, rank]
            check_sums(weights, start, vectors, where, steps, R)
            assert np.isfinite(weights).all()
