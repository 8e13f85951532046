"""ComprexAdamW's own bookkeeping, without a GPU: which stream an exchange is joined with, where a parameter's moves lie
in the exchanged vector, what a checkpoint restores.  The sets check their tensors as they do on a GPU; in place of
the kernels a step puts the (clipped) gradient itself into the moves, so that every weight shows whose moves it got.
Ranks are threads, and the exchange in between is a sum without compression, or a stand-in that a test describes."""
import contextlib
import threading

import pytest
import torch

from comprex_amd import optimizer
from comprex_amd.device import AdamWSet, TensorSet
from comprex_amd.optimizer import ComprexAdamW

CPU = torch.device("cpu")


class Stream:
    device = CPU

    def __init__(self, raw):
        self.cuda_stream = raw


class Here(threading.local):
    """What is current for a thread."""
    rank = 0
    stream = Stream(0)
    user_stream = None
    met = False


here = Here()


class HostSet(TensorSet):
    def _make(self, handle, sizes, state):
        self.handle, self.sizes, self.total = handle, sizes, sum(sizes)
        self._on(CPU)


class HostAdamWSet(AdamWSet):
    _make = HostSet._make


class HostHandle:
    device = CPU

    def __init__(self, stream):
        self.stream = stream

    def set_stream(self, stream):
        self.stream = stream

    def grad_norms(self, tensors, grads, max_norm=None):
        of = [g for g in grads.tensors if g is not None]
        norm = torch.cat([g.double().reshape(-1) for g in of]).norm()
        coef = 1.0 if max_norm is None else min(1.0, max_norm / float(norm))
        return (norm.float().reshape(1), torch.full((1,), coef),
                torch.full((1,), 0 if torch.isfinite(norm) else 1, dtype=torch.int32))

    def adamw_step(self, tensors, grads, step, lr, betas, eps, weight_decay, coefs, skip, moves, **how):
        grads = getattr(grads, "tensors", grads)
        skipped = skip is not None and bool(skip)
        if isinstance(step, torch.Tensor) and not skipped:
            step += 1
        at = 0
        for k, (g, n) in enumerate(zip(grads, tensors.sizes)):
            if moves is not None and g is not None:
                moves[at:at + n] = 0.0 if skipped else g.reshape(-1).float()
            if moves is None and g is not None and not skipped:
                tensors.kept[0][k].data.sub_(g)
            at += n

    def adamw_apply(self, tensors, moves, lr, weight_decay, scale=1.0):
        at = 0
        for p, n in zip(tensors.kept[0], tensors.sizes):
            p.data.sub_(moves[at:at + n].view_as(p) * scale)
            at += n


class Env:
    """R ranks, each in a thread of its own."""

    def __init__(self, ranks=1):
        self.ranks, self.meet = ranks, threading.Barrier(ranks, timeout=30)
        self.given = [None] * ranks

    def get_ranks(self):
        return self.ranks

    def barrier(self):
        self.meet.wait()

    def set_user_stream(self, stream):
        here.user_stream = stream


class Exchange:
    """Sums at once.  Joined with the thread's user stream, which has to be the one that the vector is written on."""
    made = []

    def __init__(self, kind, env, size, ratio, factor):
        self.env, self.size, self.resets, self.log = env, size, 0, []
        Exchange.made.append(self)

    def joined(self):
        assert here.user_stream is not None and here.user_stream.cuda_stream == here.stream.cuda_stream

    def apply(self, blob):
        self.joined()
        self.log.append(blob.clone())
        self.env.given[here.rank] = blob.clone()
        self.env.meet.wait()
        blob.copy_(sum(self.env.given))
        self.env.meet.wait()

    def reset(self):
        self.resets += 1


@pytest.fixture(autouse=True)
def on_the_host(monkeypatch):
    def gradients(self, grads):
        found = TensorSet.gradients(self, grads)
        if isinstance(grads, list):
            found.tensors = grads
        return found

    def part_of(self, grads, start):
        found = TensorSet.part_of(self, grads, start)
        found.tensors = grads.tensors[start:start + len(self.sizes)]
        return found

    for cls in (HostSet, HostAdamWSet):
        monkeypatch.setattr(cls, "gradients", gradients, raising=False)
        monkeypatch.setattr(cls, "part_of", part_of, raising=False)
    monkeypatch.setattr(optimizer, "TensorSet", HostSet)
    monkeypatch.setattr(optimizer, "AdamWSet", HostAdamWSet)
    monkeypatch.setattr(optimizer, "Handle", HostHandle)
    monkeypatch.setattr(optimizer, "_make_allreduce", Exchange)
    monkeypatch.setattr(ComprexAdamW, "_check", staticmethod(lambda p: None))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: here.stream)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", on_stream)
    Exchange.made = []
    here.__dict__.clear()


@contextlib.contextmanager
def on_stream(stream):
    before, here.stream = here.stream, stream
    try:
        yield
    finally:
        here.stream = before


def run_ranks(ranks, program):
    """program(env, rank) for every rank, each in a thread of its own."""
    env, errors = Env(ranks), []

    def rank_program(rank):
        here.rank = rank
        try:
            program(env, rank)
        except BaseException as e:  # noqa: BLE001
            env.meet.abort()
            errors.append((rank, e))

    threads = [threading.Thread(target=rank_program, args=(r,)) for r in range(ranks)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    for _, e in sorted(errors, key=lambda x: isinstance(x[1], threading.BrokenBarrierError)):
        raise e


def parameter(n, value=0.0, dtype=torch.float32):
    return torch.nn.Parameter(torch.full((n,), value, dtype=dtype))


def give(params, value):
    for p in params:
        p.grad = torch.full_like(p, value)


def test_the_exchange_is_joined_with_the_stream_of_each_step():
    """Two optimizers on streams of their own, the program's own use of the setting, another thread, and a first step
    on the null stream: every exchange is joined with the stream that its vector is written on."""
    def program(env, rank):
        a, b = [parameter(4)], [parameter(6)]
        opts = [ComprexAdamW(ps, env, weight_decay=0.0) for ps in (a, b)]
        streams = [Stream(1), Stream(2)]
        for step in range(3):
            for ps, opt, stream in zip((a, b), opts, streams):
                give(ps, 1.0)
                with on_stream(stream):
                    opt.step()
        env.set_user_stream(Stream(7))  # an exchange of the program's own
        give(a, 1.0)
        with on_stream(streams[0]):
            opts[0].step()
        assert torch.equal(a[0].detach(), torch.full((4,), -4.0)) and torch.equal(b[0].detach(), torch.full((6,), -3.0))
        env.set_user_stream(Stream(7))
        give(b, 1.0)
        first = ComprexAdamW(b, env, weight_decay=0.0)
        first.step()  # on the null stream

    run_ranks(2, program)


def test_a_step_from_another_thread_sets_that_threads_stream():
    def program(env, rank):
        ps = [parameter(4)]
        opt = ComprexAdamW(ps, env, weight_decay=0.0)
        errors = []

        def step():
            here.rank = rank
            give(ps, 1.0)
            try:
                with on_stream(Stream(3)):
                    opt.step()
            except BaseException as e:  # noqa: BLE001
                env.meet.abort()
                errors.append(e)

        for _ in range(2):
            t = threading.Thread(target=step)
            t.start()
            t.join(30)
        assert not errors, errors

    run_ranks(2, program)


def recorded(opt):
    """Where each parameter's moves lay in the last exchanged vector, by the values that were put there."""
    return opt.allreduce.log[-1].tolist()


@pytest.mark.parametrize("restore", [False, True])
def test_the_vectors_layout_does_not_depend_on_a_ranks_counts(restore):
    """Rank 1 skips a step (a NaN in its gradient) while the middle one of three parameters is frozen; then it is
    released, or a state saved before is loaded, which groups the parameters by their counts anew.  Every weight gets
    the average of its own moves."""
    def program(env, rank):
        ps = [parameter(n) for n in (3, 4, 5)]
        ps[1].requires_grad_(False)
        opt = ComprexAdamW(ps, env, weight_decay=0.0, skip_nonfinite=True)
        for k in (0, 2):
            give([ps[k]], float(k + 1))
        if rank == 1:
            ps[0].grad[1] = float("nan")
        opt.step()
        counts = [s["step"] for s in opt.state_dict()["state"].values()]
        assert counts == ([1, 1], [0, 0])[rank]
        ps[1].requires_grad_(True)
        want = [1.0] * 3 + [2.0] * 4 + [3.0] * 5
        for again in range(2):
            for k in range(3):
                give([ps[k]], float(k + 1))
            opt.step()
            assert recorded(opt) == want
            if restore:
                opt.load_state_dict(opt.state_dict())
        assert [s["step"] for s in opt.state_dict()["state"].values()] == ([3, 3, 2], [2, 2, 2])[rank]
        # the first step moved by half of rank 0's, the others by everything
        for k, first in ((0, 0.5), (1, 0.0), (2, 0.5)):
            assert torch.equal(ps[k].detach(), torch.full_like(ps[k], -(k + 1) * (2 + first)))

    run_ranks(2, program)


def test_the_vectors_layout_does_not_depend_on_what_a_rank_loaded():
    """Rank 1 goes on from a state in 32 bits, rank 0 starts anew in 8: parameters lie in the same places."""
    def program(env, rank):
        ps = [parameter(n) for n in (300, 20, 400)]
        opt = ComprexAdamW(ps, env, weight_decay=0.0, state_bits=8, min_8bit_size=100)
        if rank == 1:
            saved = ComprexAdamW(ps, Env(), weight_decay=0.0)
            give(ps, 0.0)
            saved.step()
            opt.load_state_dict(saved.state_dict())
        for k, p in enumerate(ps):
            give([p], float(k + 1))
        opt.step()
        assert ("exp_avg_scales" in opt.state[ps[0]]) == (rank == 0)
        for k, p in enumerate(ps):
            assert torch.equal(p.detach(), torch.full_like(p, -(k + 1.0)))

    run_ranks(2, program)


def test_counts_of_a_part_on_the_device():
    """One rank, counts on the device: parameters of different counts in one part each advance their own, those without
    a gradient none of their own count's go along."""
    env = Env()
    ps = [parameter(3) for _ in range(4)]
    for p in ps[2:]:
        p.requires_grad_(False)
    opt = ComprexAdamW(ps, env, weight_decay=0.0, skip_nonfinite=True)
    give(ps[:2], 1.0)
    opt.step()
    for p in ps[2:]:
        p.requires_grad_(True)
    give(ps, 1.0)
    ps[3].grad = None
    opt.step()
    ps[0].grad = ps[1].grad = None
    opt.step()
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [2, 2, 2, 2]
    assert [float(p[0]) for p in ps] == [-2, -2, -2, 0]


class Holding(Exchange):
    """Delivers a rank its own vector and holds back what the others sent until it is flushed."""

    def __init__(self, *args):
        super().__init__(*args)
        self.held = torch.zeros(self.size)

    def swap(self, blob):
        self.env.given[here.rank] = blob.clone()
        self.env.meet.wait()
        others = sum(self.env.given) - blob
        self.env.meet.wait()
        return others

    def apply(self, blob):
        self.joined()
        self.held += self.swap(blob)

    def flush(self, blob):
        self.joined()
        self.swap(blob)
        blob += self.held
        self.reset()

    def reset(self):
        super().reset()
        self.held.zero_()


def test_a_restored_state_gets_nothing_of_the_run_it_replaces(monkeypatch):
    monkeypatch.setattr(optimizer, "_make_allreduce", Holding)

    def program(env, rank):
        ps = [parameter(3), parameter(4)]
        opt = ComprexAdamW(ps, env, weight_decay=0.0)
        opt.flush()  # nothing to flush yet
        give(ps, 2.0 * (rank + 1))
        opt.step()
        assert float(ps[0][0]) == -(rank + 1)    # a half of its own; the other's is held back
        opt.flush()
        assert all((p == -3.0).all() for p in ps)
        saved, kept = opt.state_dict(), [p.detach().clone() for p in ps]
        give(ps, 64.0)
        opt.step()                             # of a run that is given up
        opt.load_state_dict(saved)
        with torch.no_grad():
            for p, k in zip(ps, kept):
                p.copy_(k)
        give(ps, 0.0)
        opt.step()
        opt.flush()
        assert all((p == -3.0).all() for p in ps)
        versions = [p._version for p in ps]
        opt.flush()
        assert all(p._version > v for p, v in zip(ps, versions)) and opt.blob.count_nonzero() == 0

    run_ranks(2, program)


def test_a_flush_by_one_rank_alone_changes_nothing():
    ps = [parameter(3, 1.0)]
    opt = ComprexAdamW(ps, Env(), weight_decay=0.5)
    give(ps, 0.0)
    opt.step()
    opt.flush()
    assert (ps[0] == 1.0).all() and opt.allreduce is None


class Growing(Exchange):
    """Its connections may replace the buffers of those before, so no rank may still be at an exchange."""

    def __init__(self, *args):
        super().__init__(*args)
        assert here.met, "made while another rank may still read what this one sent"

    def apply(self, blob):
        super().apply(blob)
        here.met = False


def test_ranks_meet_before_an_exchange_is_made(monkeypatch):
    """The messages of one exchange are read before the next one's connections are made: another layout, and another
    optimizer on the same environment."""
    monkeypatch.setattr(optimizer, "_make_allreduce", Growing)
    monkeypatch.setattr(Env, "barrier", lambda self: (self.meet.wait(), setattr(here, "met", True)))

    def program(env, rank):
        ps, more = [parameter(3), parameter(400)], [parameter(5000)]
        ps[1].requires_grad_(False)
        opt = ComprexAdamW(ps, env, weight_decay=0.0)
        give(ps, 1.0)
        opt.step()
        ps[1].requires_grad_(True)
        give(ps, 1.0)
        opt.step()
        give(more, 1.0)
        ComprexAdamW(more, env, weight_decay=0.0).step()
        met = here.met
        opt.step()
        assert met is here.met is False  # (only then)

    run_ranks(2, program)


class OnStream(torch.Tensor):
    """A tensor that is written on a stream: a look at its value waits for the one that is current."""

    def __int__(self):
        assert here.stream.cuda_stream == 5
        return super().__int__()


def test_counts_on_the_device_are_read_in_the_order_of_their_stream():
    """state_dict on another stream than the steps ran on: the counts are read behind them."""
    ps = [parameter(3)]
    opt = ComprexAdamW(ps, Env(), skip_nonfinite=True)
    with on_stream(Stream(5)):
        give(ps, 1.0)
        opt.step()
    for part in opt._parts:
        part.counts = [(count.as_subclass(OnStream), of) for count, of in part.counts]
    with on_stream(Stream(6)):
        assert opt.state_dict()["state"][0]["step"] == 1


def test_buffers_are_known_to_the_streams_that_use_them(monkeypatch):
    """The vector and the counts are allocated on one stream; steps on another tell the allocator, which would hand
    them out again as soon as they are let go of."""
    used = []
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, s: used.append((self.data_ptr(), s.cuda_stream)))

    def program(env, rank):
        ps = [parameter(3)]
        opt = ComprexAdamW(ps, env, skip_nonfinite=True)
        for raw in (5, 5, 6):
            with on_stream(Stream(raw)):
                give(ps, 1.0)
                opt.step()
        mine = {(t.data_ptr(), 6) for t in (opt.blob, opt._parts[0].counts[0][0])}
        env.barrier()
        assert mine <= set(used) and len(used) == 4

    run_ranks(2, program)


def at_the_same_place(t, dtype, shape=None):
    """Another tensor where `t` lies: what an allocation may get when the memory of `t` was let go of."""
    return t.detach().view(torch.uint8)[:t.numel() * torch.empty(0, dtype=dtype).element_size()].view(dtype)


def test_a_set_is_made_of_its_tensors_types_and_sizes_too():
    p, m, v = torch.zeros(12), torch.zeros(12), torch.zeros(12)
    s = HostAdamWSet(HostHandle(Stream(0)), [p], [m], [v])
    lists = lambda x=p: [[x], [m], [v], None, None, None]  # noqa: E731
    assert s.made_of(lists()) and s.made_of(lists(p.view(3, 4)))
    assert not s.made_of(lists(p.clone()))
    assert not s.made_of(lists(at_the_same_place(p, torch.bfloat16)))
    assert not s.made_of(lists(p[:11])) and not s.made_of(lists(p.view(3, 4).t()))
    assert not s.made_of([[p], [m], [v], [m], None, None]) and not s.made_of([[p], [m], [v[:11]], None, None, None])


def test_a_parameter_whose_type_changes_where_it_lies():
    """Halved and moved onto the memory it had: another type, another set."""
    ps = [parameter(300, 1.0), parameter(20)]
    opt = ComprexAdamW(ps, Env(), weight_decay=0.0)
    give(ps, 1.0)
    opt.step()
    was = opt._parts[0].set
    room = ps[0].data
    ps[0].data = at_the_same_place(room, torch.bfloat16)
    ps[0].data.fill_(3.0)
    assert ps[0].data_ptr() == room.data_ptr()
    give(ps, 1.0)
    opt.step()
    assert [part.set.kept[0][0].dtype for part in opt._parts] == [torch.bfloat16, torch.float32]
    assert was not in [part.set for part in opt._parts]
    assert (ps[0] == 2.0).all() and (ps[1] == -2.0).all()
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [2, 2]


@pytest.mark.parametrize("bad", [dict(amsgrad=True), dict(maximize=True), dict(decoupled_weight_decay=False, weight_decay=0.1)],
                         ids=str)
def test_groups_of_another_update_are_refused(bad):
    """What a state of torch's own optimizers may ask for and this step does not do; nothing is taken over then."""
    p = parameter(5, 1.0)
    opt = ComprexAdamW([p], Env(), learning_rate=0.5)
    give([p], 1.0)
    opt.step()
    saved = opt.state_dict()
    theirs = dict(saved, param_groups=[dict(saved["param_groups"][0], lr=0.25, **bad)])
    with pytest.raises(ValueError):
        opt.load_state_dict(theirs)
    assert opt.param_groups[0]["lr"] == 0.5
    fine = dict(saved, param_groups=[dict(saved["param_groups"][0], lr=0.25, amsgrad=False, maximize=False,
                                          decoupled_weight_decay=True, foreach=None)])
    opt.load_state_dict(fine)
    assert opt.param_groups[0]["lr"] == 0.25
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[parameter(3)], **bad))
    assert len(opt.param_groups) == 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_state_of_torchs_adamw_for_16_bit_parameters(dtype):
    """Its moments have the parameters' type and there are no masters: taken in 32 bits, and masters are made."""
    p = parameter(7, 1.5, dtype)
    theirs = torch.optim.AdamW([p], lr=1e-2)
    give([p], 0.5)
    theirs.step()
    q = parameter(7, 0.0, dtype)
    opt = ComprexAdamW([q], Env())
    opt.load_state_dict(theirs.state_dict())
    with torch.no_grad():
        q.copy_(p)   # a model is restored before or after its optimizer
    give([q], 0.5)
    opt.step()
    s = opt.state[q]
    assert s["step"] == 2 and s["exp_avg"].dtype == s["exp_avg_sq"].dtype == s["master"].dtype == torch.float32
    assert torch.equal(s["exp_avg"], theirs.state[p]["exp_avg"].float()) and torch.equal(s["master"], p.float())
    other = ComprexAdamW([q], Env(), master_weights=False)
    other.load_state_dict(theirs.state_dict())
    other.step()
    assert "master" not in other.state[q]


def test_what_the_step_would_refuse_is_refused_before_anything_counts():
    p, q = parameter(5), parameter(6)
    for bad in (dict(eps=0.0), dict(eps=1e-21), dict(eps=float("inf")), dict(weight_decay=-0.1), dict(learning_rate=-1.0),
                dict(betas=(0.9, 1.0)), dict(weight_decay=float("nan"))):
        with pytest.raises(ValueError):
            ComprexAdamW([p], Env(), **bad)
    with pytest.raises(ValueError):
        ComprexAdamW([dict(params=[p]), dict(params=[q], eps=0.0)], Env())
    opt = ComprexAdamW([dict(params=[p]), dict(params=[q])], Env(), learning_rate=torch.tensor(0.5))
    give([p, q], 1.0)
    opt.step()
    opt.param_groups[1]["eps"] = 0.0
    with pytest.raises(ValueError):
        opt.step()
    opt.param_groups[1]["eps"] = 1e-8
    assert (p == -1.0).all() and [s["step"] for s in opt.state_dict()["state"].values()] == [1, 1]


def test_a_step_that_is_refused_does_not_count(monkeypatch):
    p = parameter(5)
    opt = ComprexAdamW([p], Env())
    give([p], 1.0)

    def refuse(*args, **how):
        raise RuntimeError("refused")

    with monkeypatch.context() as m:
        m.setattr(HostHandle, "adamw_step", refuse)
        with pytest.raises(RuntimeError):
            opt.step()
    assert opt.state[p]["step"] == 0
    opt.step()
    assert opt.state[p]["step"] == 1


def test_ranks_meet_before_the_momentum_optimizer_makes_an_exchange(monkeypatch):
    monkeypatch.setattr(optimizer, "_make_allreduce", Growing)
    monkeypatch.setattr(Growing, "joined", lambda self: None)  # (it leaves the user stream to the program)
    monkeypatch.setattr(Env, "barrier", lambda self: (self.meet.wait(), setattr(here, "met", True)))

    def program(env, rank):
        ps = [parameter(3), parameter(400)]
        opt = optimizer.ComprexOptimizer(ps, env, learning_rate=1.0, momentum=0.0)
        give(ps[:1], 1.0)
        opt.step()
        give(ps, 0.125)
        opt.step()
        met = here.met
        opt.step()
        assert met is here.met is False
        assert (ps[0] == -1.25).all() and (ps[1] == -0.25).all()

    run_ranks(2, program)
