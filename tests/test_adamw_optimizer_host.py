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
