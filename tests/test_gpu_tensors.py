"""Clipping, packing and the AdamW step over many tensors (cx_grad_norms, cx_pack, cx_adamw_step,
cx_adamw_states, cx_adamw_set_states) against the formulas in 64 bits.

Tolerances count roundings: u = 2^-24 of a value for one rounding to fp32 (constants such as beta and
rates that were rounded on the host count as one), half a step of the type for the last rounding of a
16-bit parameter or an 8-bit state."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from comprex_amd import _lib
from comprex_amd._lib import ComprexError

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 2.0 ** -100
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
BLOCK = 256

SIZES = [[1], [3], [255], [256], [257], [1023, 1, 1025], [4096, 0, 3, 70001, 16384, 16385], [0], []]


def device_module():
    from comprex_amd import device
    return device


def spread(rng, n):
    """Values over several orders of magnitude, some of them zero."""
    x = rng.standard_normal(n) * 10.0 ** rng.uniform(-6, 0)
    x[rng.random(n) < 0.05] = 0.0
    return x


def odd(x, dtype, offset):
    """The values as a device tensor that starts `offset` elements behind an aligned address."""
    room = torch.zeros(len(x) + offset, dtype=dtype, device="cuda")
    room[offset:] = torch.as_tensor(np.asarray(x)).to(dtype)
    return room[offset:]


def f64(t):
    return t.double().cpu().numpy()


def half_step(dtype, x):
    """Half a step of a 16-bit type at |x|, subnormals included."""
    info = torch.finfo(dtype)
    return np.maximum(np.abs(x), info.tiny) * info.eps / 2


# ---- norms and packing -----------------------------------------------------------------------

@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("each", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", SIZES + [[262144], [262145], [1200003, 5, 70001]], ids=str)  # both sides of one launch
def test_norms_and_pack(sizes, dtype, each, offset):
    D = device_module()
    rng = np.random.default_rng(len(sizes) + offset)
    grads = [odd(spread(rng, n), dtype, offset) for n in sizes]
    g = [f64(x) for x in grads]
    scale, max_norm = -0.75, 0.3
    h = D.Handle()
    ts = D.TensorSet(h, sizes)
    norms, coefs, nonfinite = h.grad_norms(ts, grads, max_norm, each=each, scale=scale)
    want = np.array([abs(scale) * math.sqrt(float((x * x).sum())) for x in g])
    want = np.append(want, math.sqrt(float((want ** 2).sum())))
    # sums in 64 bits, one rounding to 32 at the end
    np.testing.assert_allclose(f64(norms), want, rtol=U * 1.001, atol=2.0 ** -149)
    which = want[:-1] if each else want[-1:]
    clip = np.array([max_norm / w if w > max_norm else 1.0 for w in which])
    np.testing.assert_allclose(f64(coefs), clip, rtol=U * 1.001)
    assert nonfinite.tolist() == [0]
    flat = h.pack(ts, grads, coefs=coefs, scale=scale)
    # coef, its product with the scale, the product with g: three roundings
    for k, (x, at) in enumerate(zip(g, np.cumsum([0] + sizes))):
        np.testing.assert_allclose(f64(flat[at:at + len(x)]), x * scale * clip[k if each else 0], rtol=3.01 * U,
                                   atol=2.0 ** -148)
    # the flat vector as the gradient gives the same norms, and may be packed onto itself
    again = h.grad_norms(ts, flat, None)[0]
    for k, x in enumerate(g):
        want_k = np.linalg.norm(x * scale * clip[k if each else 0])
        assert abs(float(again[k]) - want_k) <= 5 * U * want_k + 1e-40
    before = flat.clone()
    assert h.pack(ts, flat, out=flat, scale=0.5) is flat
    assert torch.equal(flat, before * 0.5)


def test_norms_without_some_gradients_and_beyond_one_launch():
    """1100 tensors: more than the addresses one launch carries; every third without a gradient."""
    D = device_module()
    rng = np.random.default_rng(1)
    sizes = [int(n) for n in rng.integers(0, 9, 1100)]
    grads = [None if k % 3 == 0 else odd(spread(rng, n), F32, 0) for k, n in enumerate(sizes)]
    h = D.Handle()
    ts = D.TensorSet(h, sizes)
    norms, coefs, _ = h.grad_norms(ts, grads, 1e-3, each=True)
    flat = h.pack(ts, grads, out=torch.full((sum(sizes),), 7.0, device="cuda"))
    at = 0
    for k, (n, g) in enumerate(zip(sizes, grads)):
        x = np.zeros(n) if g is None else f64(g)
        assert abs(float(norms[k]) - np.linalg.norm(x)) <= 1.01 * U * np.linalg.norm(x)
        assert np.array_equal(f64(flat[at:at + n]), x)
        at += n
    assert np.isclose(float(norms[-1]), np.linalg.norm(f64(flat)), rtol=2 * U)
    assert h.grad_norms(ts, [None] * 1100)[0].count_nonzero() == 0


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_nonfinite_gradients_are_found_and_skipped(dtype, bad):
    D = device_module()
    sizes = [5000, 3, 70000]
    rng = np.random.default_rng(2)
    h = D.Handle()
    ts = D.TensorSet(h, sizes)
    for where in (0, 4999, 5001, 74999):
        x = rng.standard_normal(sum(sizes))
        x[where] = bad
        flat = torch.as_tensor(x).to(dtype).cuda()
        grads = list(flat.split(sizes))
        norms, _, nonfinite = h.grad_norms(ts, grads, 1.0)
        assert nonfinite.item() == 1 and not math.isfinite(float(norms[-1]))
        assert [math.isfinite(float(v)) for v in norms[:-1]] == [bool(torch.isfinite(g).all()) for g in grads]
        out = torch.full((sum(sizes),), 3.0, device="cuda")
        assert h.pack(ts, grads, out=out, skip=nonfinite).count_nonzero() == 0
    # the largest finite values do not overflow the sum
    big = [torch.full((n,), torch.finfo(dtype).max, dtype=dtype, device="cuda") for n in sizes]
    norms, _, nonfinite = h.grad_norms(ts, big, scale=2.0 ** -20)
    assert nonfinite.item() == 0
    assert np.isclose(float(norms[-1]), torch.finfo(dtype).max * 2.0 ** -20 * math.sqrt(75003), rtol=2 * U)


def test_more_than_2_to_the_31_elements():
    D = device_module()
    sizes = [(1 << 31) + 5, 1000]
    flat = torch.zeros(sum(sizes), dtype=BF16, device="cuda")
    marks = {0: 1.0, (1 << 31) - 1: 2.0, 1 << 31: 4.0, (1 << 31) + 4: 8.0, (1 << 31) + 5: 16.0, sum(sizes) - 1: 32.0}
    for at, x in marks.items():
        flat[at] = x
    h = D.Handle()
    ts = D.TensorSet(h, sizes)
    norms = h.grad_norms(ts, [flat[:sizes[0]], flat[sizes[0]:]])[0]
    assert np.allclose(f64(norms), np.sqrt([85.0, 1280.0, 1365.0]), rtol=2 * U)
    out = h.pack(ts, flat, scale=3.0)
    assert int(out.count_nonzero()) == len(marks)
    assert all(float(out[at]) == 3 * x for at, x in marks.items())


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_on_more_than_2_to_the_31_elements(bits):
    D = device_module()
    sizes = [(1 << 31) + 5, 1000]
    total, marks = sum(sizes), [0, (1 << 31) - 1, 1 << 31, (1 << 31) + 4, (1 << 31) + 5, sum(SIZE for SIZE in sizes) - 1]
    g = torch.zeros(total, dtype=BF16, device="cuda")
    g[torch.tensor(marks, device="cuda")] = 2.0
    p = torch.zeros(total, dtype=BF16, device="cuda")
    h = D.Handle()
    split = lambda t: [t[:sizes[0]], t[sizes[0]:]]  # noqa: E731
    if bits == 32:
        m, v = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
        s = D.AdamWSet(h, split(p), split(m), split(v))
    else:
        small = [D.AdamWSet.zeros8(x) for x in split(p)]
        s = D.AdamWSet(h, split(p), *([x[k] for x in small] for k in (0, 1)), exp_avg_scales=[x[2] for x in small],
                       exp_avg_sq_scales=[x[3] for x in small])
    h.adamw_step(s, split(g), 1, 2.0 ** -7, weight_decay=0.0)   # a first step moves by lr
    h.adamw_step(s, g, 2, 2.0 ** -7, weight_decay=0.0)
    assert int(p.count_nonzero()) == len(marks)
    assert all(abs(float(p[at]) + 2.0 ** -6) <= 2.0 ** -6 * 2.0 ** -7 for at in marks)


# ---- AdamW -------------------------------------------------------------------------------------

E4M3 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
E5M3 = np.array([(1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 1) if c > 7 else c / 8 for c in range(256)])
E5M3 /= E5M3[255]


def rows(x):
    """A tensor's values in blocks, the last one filled with zeros."""
    return np.pad(x, (0, -len(x) % BLOCK)).reshape(-1, BLOCK)


def values8(codes, scales, table):
    c = codes.view(torch.uint8).cpu().numpy()
    return (table[rows(c)] * f64(scales)[:, None]).reshape(-1)[:len(c)]


class Params:
    """The tensors of an AdamW step with a history, and their values in 64 bits."""

    def __init__(self, seed, sizes, param, bits, master, offset):
        rng = np.random.default_rng(seed)
        D = device_module()
        self.sizes, self.param, self.bits = sizes, param, bits
        self.p, self.w, self.m, self.v, self.ms, self.vs = [], [] if master else None, [], [], [], []
        size = [10.0 ** rng.uniform(-5, -1) for _ in sizes]
        for n, s in zip(sizes, size):
            w = rng.standard_normal(n) * 0.02
            self.p.append(odd(w, param, offset))
            if master:
                self.w.append(odd(w, F32, offset))
            m = rng.standard_normal(n) * s * 0.3
            v = s * s * rng.random(n) * 2
            untouched = rng.random(n) < 0.05
            m[untouched] = v[untouched] = 0.0
            if bits == 32:
                self.m.append(odd(m, F32, offset))
                self.v.append(odd(v, F32, offset))
            else:  # any codes are a valid history: all of them but NaN occur
                c = rng.integers(0, 256, n).astype(np.uint8)
                c[(c & 127) == 127] = 0
                self.m.append(odd(c, torch.uint8, offset).view(torch.float8_e4m3fn))
                self.v.append(odd(rng.integers(0, 256, n).astype(np.uint8), torch.uint8, offset))
                blocks = -(-n // BLOCK)
                self.ms.append(odd(s * (0.1 + rng.random(blocks)) / 448, F32, offset))
                self.vs.append(odd(s * s * (0.1 + rng.random(blocks)), F32, offset))
        self.size, self.rng = size, rng
        self.h = D.Handle()
        self.set = D.AdamWSet(self.h, self.p, self.m, self.v, self.w, *((self.ms, self.vs) if bits == 8 else ()))

    def gradients(self, dtype, offset):
        """A gradient per tensor; in fp16 under a loss scale of 256."""
        up = 256.0 if dtype == F16 else 1.0
        out = []
        for n, s in zip(self.sizes, self.size):
            g = self.rng.standard_normal(n) * s * up
            g[self.rng.random(n) < 0.05] = 0.0
            out.append(odd(g, dtype, offset))
        return out, 1.0 / up

    def now(self):
        """Per tensor (w, m, v) in 64 bits."""
        got = []
        for k in range(len(self.sizes)):
            w = f64((self.w or self.p)[k])
            if self.bits == 32:
                got.append((w, f64(self.m[k]), f64(self.v[k])))
            else:
                got.append((w, values8(self.m[k], self.ms[k], E4M3), values8(self.v[k], self.vs[k], E5M3)))
        return got

    def snapshot(self):
        return [None if x is None else [t.clone() for t in x] for x in (self.p, self.w, self.m, self.v, self.ms, self.vs)]


def same(a, b):
    return all(x is y is None or all(torch.equal(s.view(torch.uint8) if s.dtype == torch.float8_e4m3fn else s,
                                                 t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t)
                                     for s, t in zip(x, y)) for x, y in zip(a, b))


def check_step(P, before, g, factor, step, lr, b1, b2, eps, wd, tensors=None):
    """P's tensors against one step from `before`, with gradients g (64 bits) times factor[k]."""
    now = P.now()
    for k in range(len(P.sizes)) if tensors is None else tensors:
        w, m, v = before[k]
        x = g[k] * factor[k]
        small = P.bits == 8
        # m: a code's value is a product (8 bits); beta, rest and factor are rounded, so are both products, g * factor
        # (factor itself coef * scale) and the sum
        m1 = b1 * m + (1 - b1) * x
        em = U * ((2 + small) * np.abs(b1 * m) + 6 * np.abs((1 - b1) * x) + 1.01 * np.abs(m1)) + 2.0 ** -147
        # v: a code's value has a rounded constant and two products
        v1 = b2 * v + (1 - b2) * x * x
        ev = U * ((2 + 3 * small) * b2 * v + 10 * (1 - b2) * x * x + 1.01 * v1) + 2.0 ** -147
        unit = 1 / math.sqrt(1 - b2 ** step)
        below = np.sqrt(v1) * unit + eps
        # sqrt of the range of v, the square root itself (one unit in the last place: 2 u), v_unit, the sum's rounding, eps
        eb = (np.sqrt(v1 + ev) - np.sqrt(np.maximum(v1 - ev, 0))) * unit + 5.01 * U * below
        rate = lr / (1 - b1 ** step)
        move = rate * m1 / below
        # the reciprocal (one unit in the last place: 2 u), its product with m, the rate, the product with it
        em_move = rate * em / below + np.abs(move) * (eb / (below - eb) + 5.01 * U)
        w1 = w - lr * wd * w - move
        ew = em_move + U * (3 * np.abs(lr * wd * w) + 2 * np.abs(move) + 1.01 * np.abs(w1))
        got_w, got_m, got_v = now[k]
        if P.w is not None:
            assert (np.abs(got_w - w1) <= ew).all(), (k, np.abs(got_w - w1).max())
        p = f64(P.p[k])
        last = 0.0 if P.param == F32 else half_step(P.param, np.abs(w1) + ew)
        assert (np.abs(p - w1) <= ew + last).all(), (k, np.abs(p - w1).max())
        if not small:
            assert (np.abs(got_m - m1) <= em).all() and (np.abs(got_v - v1) <= ev).all()
            continue
        check_codes(P, k, m1, em, v1, ev)


def check_codes(P, k, m1, em, v1, ev):
    """8-bit states of tensor k against the values they were rounded from (each known to em, ev)."""
    n = P.sizes[k]
    got_m, got_v = values8(P.m[k], P.ms[k], E4M3), values8(P.v[k], P.vs[k], E5M3)
    mt, vt = rows(np.abs(m1)).max(1, initial=0.0), rows(v1).max(1, initial=0.0)
    emt, evt = rows(em).max(1, initial=0.0), rows(ev).max(1, initial=0.0)
    ms, vs = f64(P.ms[k]), f64(P.vs[k])
    # the scale: the constant 1 / 448 and the product are rounded; a block near 2^-100 may go either way
    assert ((np.abs(ms - mt / 448) <= emt / 448 + 2.01 * U * mt) | ((ms == 0) & (mt - emt < TINY))).all()
    assert ((np.abs(vs - vt) <= evt) | ((vs == 0) & (vt - evt < TINY))).all()
    for got, want, err, top, scales, lowest, table in ((got_m, np.abs(m1), em, mt / 448, ms, 2.0 ** -9, E4M3),
                                                      (got_v, v1, ev, vt / 1.875 * 2.0 ** -30, vs, 2.0 ** -3, E5M3)):
        per = np.repeat(np.where(scales == 0, 0.0, top), BLOCK)[:n]
        keep = per > 0
        assert (got[~keep] == 0).all()
        # in units of the codes: what the value may be, with 5 more roundings (inverse, products, their constants), and
        # half a step of 3 fraction bits there; the codes' values themselves are read in 64 bits, scale within 2 u
        y = want[keep] / per[keep]
        slack = err[keep] / per[keep] + 5.01 * U * y + 2.0 ** -22 * lowest
        top_y = y + slack
        # binade of at least the smallest normal (lowest * 8)
        half = 2.0 ** np.floor(np.log2(np.maximum(top_y, lowest * 8))) / 16
        off = np.abs(np.abs(got[keep]) / per[keep] - y)
        ok = off <= half + slack + 3 * U * top_y + np.repeat(emt if lowest < 2.0 ** -8 else evt, BLOCK)[:n][keep] / np.maximum(
            np.repeat(mt if lowest < 2.0 ** -8 else vt, BLOCK)[:n][keep], 1e-300) * top_y
        if table is E5M3:  # above 0 is never stored as 0
            ok |= (np.abs(got[keep] / per[keep] - lowest) < 1e-5) & (y > 0) & (y < lowest)
            assert ((got[keep] > 0) == (v1[keep] > 0)).all()
        assert ok.all(), (k, off[~ok], y[~ok])
    signs = got_m != 0
    assert (np.sign(got_m[signs]) == np.sign(m1[signs])).all()


TYPES = [(F32, F32, False), (F32, BF16, False), (BF16, BF16, True), (BF16, BF16, False), (BF16, F32, False),
         (BF16, F16, True), (F16, F16, True), (F16, F16, False), (F16, F32, True), (F32, F16, False)]


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad,master", TYPES, ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_adamw_step(sizes, param, grad, master, bits, offset):
    if offset and len(sizes) not in (1, 3, 6):
        pytest.skip("alignment is tried on some of the sizes")
    P = Params(3, sizes, param, bits, master, offset)
    hyper = dict(lr=3e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.1)
    for step in (1, 2, 1000):
        before = P.now()
        grads, scale = P.gradients(grad, offset)
        n_coefs = (0, 1, len(sizes))[step % 3]
        coefs = torch.as_tensor(P.rng.uniform(0.2, 1.0, n_coefs), dtype=F32).cuda() if n_coefs else None
        P.h.adamw_step(P.set, grads, step, hyper["lr"], (hyper["b1"], hyper["b2"]), hyper["eps"], hyper["wd"],
                       coefs=coefs, scale=scale)
        c = [1.0] * len(sizes) if coefs is None else list(f64(coefs)) * (len(sizes) if n_coefs == 1 else 1)
        check_step(P, before, [f64(g) for g in grads], [x * scale for x in c], step, **hyper)


@pytest.mark.parametrize("param,grad,master", [(F32, F32, False), (BF16, BF16, True), (F16, F16, False)], ids=str)
@pytest.mark.parametrize("bits", [32, 8])
def test_nothing_beside_the_tensors_is_written(bits, param, grad, master):
    """Tensors between guards of a mark of their own: every kernel leaves them as they are."""
    D = device_module()
    sizes = [1, 2, 3, 5, 255, 257, 511, 513, 1023, 1025, 2047, 2049, 4100]
    blocks = [-(-n // BLOCK) for n in sizes]
    rooms = []

    def guarded(ns, dtype):
        """A buffer with 5 elements of guard before, between and behind parts of the given sizes."""
        room = torch.full((sum(ns) + 5 * (len(ns) + 1),), 77, dtype=dtype, device="cuda")
        inside = torch.zeros(room.numel(), dtype=torch.bool, device="cuda")
        parts, at = [], 5
        for n in ns:
            room[at:at + n] = 0
            inside[at:at + n] = True
            parts.append(room[at:at + n])
            at += n + 5
        rooms.append((room, inside))
        return parts

    p, w = guarded(sizes, param), guarded(sizes, F32) if master else None
    if bits == 32:
        m, v, scales = guarded(sizes, F32), guarded(sizes, F32), []
    else:
        m, v = [x.view(torch.float8_e4m3fn) for x in guarded(sizes, torch.uint8)], guarded(sizes, torch.uint8)
        scales = [guarded(blocks, F32), guarded(blocks, F32)]
    h = D.Handle()
    s = D.AdamWSet(h, p, m, v, w, *scales)
    grads = [torch.ones(n, dtype=grad, device="cuda") for n in sizes]
    flat, moves, norms, coefs = (guarded([n], F32)[0] for n in (sum(sizes), sum(sizes), len(sizes) + 1, len(sizes)))
    h.grad_norms(s, grads, 1.0, each=True, norms=norms, coefs=coefs)
    h.pack(s, grads, out=flat, coefs=coefs)
    h.adamw_step(s, grads, 1, 0.5)
    h.adamw_step(s, flat, 2, 0.5, moves=moves)
    h.adamw_apply(s, moves, 0.5)
    if bits == 8:
        a, b = (guarded([sum(sizes)], BF16)[0] for _ in range(2))
        c, d = (guarded([sum(sizes)], F32)[0] for _ in range(2))
        h.adamw_states(s, BF16, a, b)
        h.adamw_states(s, F32, c, d)
        h.adamw_set_states(s, c, d)
    h.synchronize()
    for room, inside in rooms:
        assert (room[~inside] == 77).all()
        assert (room[inside] != 0).all()  # (and everything inside was)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_flat_gradient_is_the_list(bits):
    """The flat vector, as the exchange leaves it, against the same gradients one by one: the same bits."""
    sizes = [7, 1000, 1, 70001, 256, 0, 513]
    A, B = (Params(4, sizes, F32, bits, False, 0) for _ in range(2))
    for step in (1, 2, 3):
        grads, _ = A.gradients(F32, 1)
        A.h.adamw_step(A.set, grads, step, 1e-3, scale=0.25)
        B.h.adamw_step(B.set, torch.cat(grads), step, 1e-3, scale=0.25)
        assert same(A.snapshot(), B.snapshot())


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_leaves_tensors_without_a_gradient(bits):
    sizes = [1000] * 500 + [4097]
    P = Params(5, sizes, BF16, bits, True, 0)
    grads, _ = P.gradients(BF16, 0)
    grads = [g if k % 2 else None for k, g in enumerate(grads)]
    was, before = P.snapshot(), P.now()
    P.h.adamw_step(P.set, grads, 7, 1e-2, weight_decay=0.3)
    now = P.snapshot()
    even = lambda s: [None if x is None else x[::2] for x in s]  # noqa: E731
    assert same(even(now), even(was))
    check_step(P, before, [None if g is None else f64(g) for g in grads], [1.0] * 501, 7, 1e-2, 0.9, 0.999, 1e-8, 0.3,
               tensors=range(1, 501, 20))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_coefficient_per_tensor_beyond_one_launch(bits):
    """A thousand tensors, three launches' addresses: each with the coefficient of its own, and packed with it too."""
    sizes = [1 + k % 300 for k in range(1000)]
    P = Params(12, sizes, F32, bits, False, 0)
    before = P.now()
    grads, _ = P.gradients(BF16, 0)
    coefs = torch.as_tensor(P.rng.uniform(0.2, 1.0, 1000), dtype=F32).cuda()
    flat = P.h.pack(P.set, grads, coefs=coefs)
    assert torch.equal(flat, torch.cat([g.float() * c for g, c in zip(grads, coefs)]))
    P.h.adamw_step(P.set, grads, 5, 1e-3, coefs=coefs)
    check_step(P, before, [f64(g) for g in grads], list(f64(coefs)), 5, 1e-3, 0.9, 0.999, 1e-8, 0.01)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_on_scalars_and_on_one_gradient_given_twice(bits):
    sizes = [1, 300, 300, 1]
    A, B = (Params(13, sizes, F32, bits, False, 0) for _ in range(2))
    g = torch.randn(300, device="cuda")
    x, y = torch.tensor(0.25, device="cuda"), torch.tensor([[-2.0]], device="cuda")
    A.h.adamw_step(A.set, [x, g, g, y], 1, 1e-3)
    B.h.adamw_step(B.set, [x.view(1).clone(), g.clone(), g.clone(), y.view(1).clone()], 1, 1e-3)
    assert same(A.snapshot(), B.snapshot())


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_host_count_with_a_flag_or_a_rate_on_the_device(bits):
    """Each of the device's values by itself: the flag with a host count, the rate with a host count."""
    sizes = [3000, 7]
    A, B = (Params(14, sizes, F32, bits, False, 0) for _ in range(2))
    rate = torch.full((1,), 2e-3, device="cuda")
    skip = torch.ones(1, dtype=torch.int32, device="cuda")
    for step in (1, 2, 30):
        grads, _ = A.gradients(F32, 0)
        was = B.snapshot()
        B.h.adamw_step(B.set, grads, step, 2e-3, skip=skip)
        assert same(was, B.snapshot())
        A.h.adamw_step(A.set, grads, step, float(rate))
        B.h.adamw_step(B.set, grads, step, rate, skip=torch.zeros_like(skip))
        assert same(A.snapshot(), B.snapshot())


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_count_and_rate_on_the_device(bits):
    """A device count and learning rate give the bits of the host's, skip leaves all as it is."""
    sizes = [5000, 300]
    A, B = (Params(6, sizes, F32, bits, False, 0) for _ in range(2))
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    rate = torch.zeros(1, device="cuda")
    skip = torch.zeros(1, dtype=torch.int32, device="cuda")
    for step in range(1, 6):
        grads, _ = A.gradients(F32, 0)
        rate.fill_(1e-3 * step)
        A.h.adamw_step(A.set, grads, step, float(rate), weight_decay=0.01)
        if step == 3:
            was = B.snapshot()
            skip.fill_(1)
            B.h.adamw_step(B.set, grads, count, rate, weight_decay=0.01, skip=skip)
            assert same(was, B.snapshot()) and count.item() == 2
            skip.zero_()
        B.h.adamw_step(B.set, grads, count, rate, weight_decay=0.01, skip=skip)
        assert count.item() == step
        assert same(A.snapshot(), B.snapshot())


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad,master", TYPES, ids=str)
def test_adamw_moves_and_apply_are_the_step(param, grad, master, bits, offset):
    """The step in two halves, moves and weights, has the bits of the step in one."""
    sizes = [1, 257, 70001, 0, 1024, 2048, 100]
    A, B = (Params(10, sizes, param, bits, master, offset) for _ in range(2))
    moves = odd(np.full(sum(sizes), 7.0), F32, offset)
    count, skip = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))
    coef = torch.full((1,), 0.3, device="cuda")
    for step in (1, 2, 3):
        grads, scale = A.gradients(grad, offset)
        if step == 2:  # nothing but zeros comes out of a step that is skipped
            was = B.snapshot()
            skip.fill_(1)
            B.h.adamw_step(B.set, grads, count, 1e-2, coefs=coef, scale=scale, skip=skip, moves=moves)
            assert moves.count_nonzero() == 0 and same(was, B.snapshot()) and count.item() == 1
            skip.zero_()
        A.h.adamw_step(A.set, grads, step, 1e-2, weight_decay=0.2, coefs=coef, scale=scale)
        w = [None if x is None else [t.clone() for t in x] for x in (B.p, B.w)]
        B.h.adamw_step(B.set, grads, count, 1e-2, weight_decay=0.2, coefs=coef, scale=scale, skip=skip, moves=moves)
        assert same(w, (B.p, B.w))  # the weights wait for the other half
        B.h.adamw_apply(B.set, moves, 1e-2, 0.2)
        assert same(A.snapshot(), B.snapshot())
    # in place of the flat gradient
    flat = torch.cat([g.float() for g in grads])
    C, E = (Params(10, sizes, param, bits, master, offset) for _ in range(2))
    C.h.adamw_step(C.set, flat, 1, 1e-2, scale=scale, moves=moves)
    E.h.adamw_step(E.set, flat, 1, 1e-2, scale=scale, moves=flat)
    assert torch.equal(moves, flat) and same(C.snapshot(), E.snapshot())
    # without a gradient: its part of the moves is left
    moves.fill_(5.0)
    grads[2] = None
    B.h.adamw_step(B.set, grads, 4, 1e-2, scale=scale, moves=moves)
    assert (moves[258:258 + 70001] == 5).all() and not (moves[258 + 70001:] == 5).any() and not (moves[:258] == 5).any()
    # a scale, and a rate on the device
    w = f64((B.w or B.p)[2])
    B.h.adamw_apply(B.set, moves, torch.full((1,), 0.5, device="cuda"), 0.25, scale=-0.5)
    want = w - 0.125 * w + 2.5
    last = 0.0 if param == F32 or master else half_step(param, want) * 1.01
    assert (np.abs(f64((B.w or B.p)[2]) - want) <= 3 * U * (np.abs(w) + 3) + last).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_packed_gradients_through_the_codec_and_into_a_step(dtype):
    """As one channel of the exchange uses them: clipped and packed, written with error feedback, added on the other
    side, taken by a step.  What a message does not carry stays in the residual, bit for bit."""
    D = device_module()
    sizes = [5000, 3, 70001, 256]
    P = Params(11, sizes, F32, 32, False, 0)
    total = sum(sizes)
    rests, flat, got = (torch.zeros(total, device="cuda") for _ in range(3))
    msg = torch.zeros(D.message_capacity(total, F32), dtype=torch.uint8, device="cuda")
    for step in (1, 2, 3):
        grads, _ = P.gradients(F32, 0)
        grads = [g.to(dtype) for g in grads]
        norms, coefs, flag = P.h.grad_norms(P.set, grads, 0.1)
        P.h.pack(P.set, grads, out=flat, coefs=coefs, skip=flag)
        want = torch.cat([g.float() * coefs for g in grads])
        assert torch.equal(flat, want)
        owed = rests + flat
        P.h.write_step(msg, flat, rests, 0.05, sync=False)
        got.zero_()
        P.h.add(got, msg)
        assert torch.equal(got + rests, owed) and 0 < int(got.count_nonzero()) < total
        before = P.now()
        P.h.adamw_step(P.set, got, step, 1e-3, scale=0.5)
        check_step(P, before, [f64(g) for g in got.split(sizes)], [0.5] * 4, step, 1e-3, 0.9, 0.999, 1e-8, 0.01)
    P.h.synchronize()


@pytest.mark.parametrize("bits", [32, 8])
def test_nonfinite_elements_stay_alone(bits):
    """Without a skip an infinity or NaN ruins its own weight and nothing else."""
    n = 1000
    P, Q = (Params(7, [n], F32, bits, False, 0) for _ in range(2))
    g = P.gradients(F32, 0)[0][0]
    bad = g.clone()
    where = torch.tensor([0, 100, 300, 999], device="cuda")
    clean = g.clone()
    clean[where] = 0.0
    bad[where] = torch.tensor([math.inf, -math.inf, math.nan, math.inf], device="cuda")
    fine = torch.ones(n, dtype=torch.bool, device="cuda")
    fine[where] = False
    # the elements' own history is zero on both sides, so that they count in no block's maximum
    for X in (P, Q):
        X.m[0].view(torch.uint8 if bits == 8 else F32)[where] = 0
        X.v[0][where] = 0
    for step in (1, 2):
        P.h.adamw_step(P.set, [bad], step, 1e-3)
        Q.h.adamw_step(Q.set, [clean], step, 1e-3)
        assert torch.equal(P.p[0][fine], Q.p[0][fine])
        assert not torch.isfinite(P.p[0][where]).any()
        m, v = P.m[0].view(torch.uint8) if bits == 8 else P.m[0], P.v[0]
        assert torch.equal(m[fine], (Q.m[0].view(torch.uint8) if bits == 8 else Q.m[0])[fine])
        assert torch.equal(v[fine], Q.v[0][fine])


def test_8bit_second_moments_that_overflow_stay_the_largest():
    """(1e20)^2 overflows fp32 though the gradient is finite: stored as the block's largest, not as something small."""
    D = device_module()
    p = torch.zeros(300, device="cuda")
    state = D.AdamWSet.zeros8(p)
    h = D.Handle()
    s = D.AdamWSet(h, [p], [state[0]], [state[1]], exp_avg_scales=[state[2]], exp_avg_sq_scales=[state[3]])
    g = torch.ones(300, device="cuda")
    g[7] = 1e20
    h.adamw_step(s, [g], 1, 1e-3)
    m, v = h.adamw_states(s)
    assert state[1][7] == 255 and float(v[7]) == float(state[3][0]) and torch.isfinite(v).all()
    assert torch.equal(v[:7], v[8:15]) and torch.isfinite(p).all()


def test_8bit_blocks_below_2_to_the_minus_100_are_zero():
    D = device_module()
    n = 3 * BLOCK + 5
    p = torch.ones(n, device="cuda")
    state = D.AdamWSet.zeros8(p)
    h = D.Handle()
    s = D.AdamWSet(h, [p], [state[0]], [state[1]], exp_avg_scales=[state[2]], exp_avg_sq_scales=[state[3]])
    g = torch.zeros(n, device="cuda")
    g[:BLOCK] = 2.0 ** -110          # both moments below
    g[BLOCK:2 * BLOCK] = 2.0 ** -60  # the second one
    g[2 * BLOCK] = 1.0               # one large value among tiny ones: they are kept, if coarsely
    g[2 * BLOCK + 1:3 * BLOCK] = 2.0 ** -40
    h.adamw_step(s, [g], 1, 0.0)
    m, v = h.adamw_states(s)
    assert torch.isfinite(p).all()
    assert state[2].tolist()[0] == 0 and state[2].tolist()[1] > 0 and state[3].tolist()[:2] == [0, 0]
    assert m[:BLOCK].count_nonzero() == 0 and v[:2 * BLOCK].count_nonzero() == 0
    assert (v[2 * BLOCK:3 * BLOCK] > 0).all()       # never 0
    assert state[2][3] == 0 and state[3][3] == 0    # no gradient: the last block stays zero


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", [[1], [255, 257], [4096, 0, 3, 70001], []], ids=str)
def test_8bit_states_to_values_and_back(sizes, dtype):
    P = Params(8, sizes, F32, 8, False, 1)
    was = P.snapshot()
    m, v = P.h.adamw_states(P.set, dtype)
    want_m = np.concatenate([values8(c, s, E4M3) for c, s in zip(P.m, P.ms)] + [np.zeros(0)])
    want_v = np.concatenate([values8(c, s, E5M3) for c, s in zip(P.v, P.vs)] + [np.zeros(0)])
    last = (lambda x: 0.0) if dtype == F32 else (lambda x: half_step(dtype, x))
    assert (np.abs(f64(m) - want_m) <= 1.01 * U * np.abs(want_m) + last(want_m) * 1.0001).all()
    assert (np.abs(f64(v) - want_v) <= 3.01 * U * want_v + last(want_v) * 1.0001).all()
    assert same(was, P.snapshot())
    if dtype != F32:
        return
    # back: within half a step of the values; once more: the same codes
    P.h.adamw_set_states(P.set, m, v)
    mv = [(a, b) for a, b in zip(np.split(f64(m), np.cumsum(sizes)[:-1]), np.split(f64(v), np.cumsum(sizes)[:-1]))] if sizes else []
    for k, (a, b) in enumerate(mv):
        check_codes(P, k, a, 0 * a, b, 0 * b)
    first = P.snapshot()
    P.h.adamw_set_states(P.set, *P.h.adamw_states(P.set))
    for k in range(len(sizes)):
        assert torch.equal(P.m[k].view(torch.uint8), first[2][k].view(torch.uint8))


# ---- a step as it is used ------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [32, 8])
def test_clip_pack_and_step_captured_and_replayed(bits):
    """norms -> pack -> step on a stream of its own, captured in a graph and replayed, against the eager calls:
    every replay gives the eager bits, with eager work in between."""
    D = device_module()
    sizes = [1000, 70001, 3, 256]
    A, B = (Params(9, sizes, BF16, bits, True, 0) for _ in range(2))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        B.h = D.Handle(side)
        fixed = [torch.zeros(n, dtype=BF16, device="cuda") for n in sizes]
        flat = torch.zeros(sum(sizes), device="cuda")
        norms, coefs = torch.zeros(len(sizes) + 1, device="cuda"), torch.zeros(1, device="cuda")
        nonfinite, count = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))

    def step(P, grads, step_arg):
        P.h.grad_norms(P.set, grads, 0.5, norms=norms, coefs=coefs, nonfinite=nonfinite)
        P.h.pack(P.set, grads, out=flat, coefs=coefs, skip=nonfinite)
        P.h.adamw_step(P.set, flat, step_arg, 1e-3, scale=0.5, skip=nonfinite)

    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(B, fixed, count)
    torch.cuda.synchronize()
    for k in range(1, 6):
        grads, _ = A.gradients(BF16, 0)
        step(A, grads, k)
        torch.cuda.synchronize()
        kept = flat.clone(), norms.clone(), coefs.clone()
        for f, g in zip(fixed, grads):
            f.copy_(g)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert count.item() == k
        assert all(torch.equal(a, b) for a, b in zip(kept, (flat, norms, coefs)))
        assert same(A.snapshot(), B.snapshot())


def test_from_plain_c():
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "bin", "tensors_test")
    assert os.path.exists(exe), "build tests/cpp first (make -C tests/cpp, or __graft_entry__.build())"
    print("running", exe, file=sys.stderr, flush=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    sys.stderr.write(r.stdout[-3000:] + r.stderr[-2000:])
    assert r.returncode == 0 and "+++ PASSED +++" in r.stdout, r.stdout[-2000:]


def test_outputs_are_of_the_handles_stream():
    """A handle on a stream of its own while another is current: what its calls allocate is that stream's memory."""
    D = device_module()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        h = D.Handle()
    s = D.TensorSet(h, [70001])
    g = torch.ones(70001, device="cuda")
    torch.cuda.synchronize()
    for _ in range(20):
        busy = torch.ones(70001, device="cuda")
        for _ in range(20):
            busy.mul_(1.0)
        del busy  # its memory may be the current stream's next, while the stream is still at it
        flat = h.pack(s, [g], scale=3.0)
        norms = h.grad_norms(s, flat)[0]
        side.synchronize()
        assert (flat == 3).all() and abs(float(norms[0]) - 3 * math.sqrt(70001)) < 1e-3


def test_lists_out_of_the_ordinary():
    """What the native look at a list leaves to Python: taken where it is sound, refused by name where it is not."""
    D = device_module()
    h = D.Handle()
    s = D.TensorSet(h, [6, 4])
    a, b = torch.arange(6.0, device="cuda"), torch.ones(4, device="cuda")
    want = torch.cat([a, b])
    assert torch.equal(h.pack(s, [a, b]), want)
    assert torch.equal(h.pack(s, (a, b)), want)
    assert torch.equal(h.pack(s, [a.view(2, 3), torch.nn.Parameter(b)]), want)
    half = h.pack(s, [a.half(), None])
    assert torch.equal(half, torch.cat([a, torch.zeros(4, device="cuda")]))
    for code, grads in ((_lib.CX_ERR_SIZE_MISMATCH, [a]), (_lib.CX_ERR_SIZE_MISMATCH, [b, a]),
                        (_lib.CX_ERR_INVALID, [a, b.cpu()]), (_lib.CX_ERR_INVALID, [a, b.double()]),
                        (_lib.CX_ERR_INVALID, [a, b.half()]), (_lib.CX_ERR_INVALID, [a.double(), b.double()]),
                        (_lib.CX_ERR_INVALID, [a, torch.ones(8, device="cuda")[::2]]),
                        (_lib.CX_ERR_INVALID, [a, torch.ones(4, device="meta")])):
        with pytest.raises(ComprexError) as e:
            h.pack(s, grads)
        assert e.value.code == code


def test_refusals_on_the_device():
    D = device_module()
    h = D.Handle()
    p = torch.zeros(10, device="cuda")
    z = lambda: torch.zeros(10, device="cuda")  # noqa: E731
    s = D.AdamWSet(h, [p], [z()], [z()])
    plain = D.TensorSet(h, [10])
    g = z()

    def refused(code, f, *args, **kw):
        with pytest.raises(ComprexError) as e:
            f(*args, **kw)
        assert e.value.code == code, e.value

    bad, size = _lib.CX_ERR_INVALID, _lib.CX_ERR_SIZE_MISMATCH
    refused(bad, h.adamw_step, plain, [g], 1, 1e-3)                 # no state
    refused(bad, h.adamw_states, s)                                 # not in 8 bits
    refused(bad, h.adamw_set_states, s, z(), z())
    refused(bad, h.adamw_step, s, [g], 0, 1e-3)                     # steps count from 1
    refused(bad, h.adamw_step, s, [g], 1, -1e-3)
    refused(bad, h.adamw_step, s, [g], 1, math.nan)
    refused(bad, h.adamw_step, s, [g], 1, 1e-3, betas=(1.0, 0.9))
    refused(bad, h.adamw_step, s, [g], 1, 1e-3, betas=(0.9, -0.1))
    refused(bad, h.adamw_step, s, [g], 1, 1e-3, eps=0.0)
    refused(bad, h.adamw_step, s, [g], 1, 1e-3, weight_decay=-1.0)
    refused(bad, h.adamw_step, s, [g], 1, 1e-3, scale=math.inf)
    refused(bad, h.adamw_step, s, [g], 1, 1e-3, scale=1e39)         # not in fp32
    refused(bad, h.adamw_step, s, [g], 1, 1e39)
    refused(bad, h.pack, s, [g], scale=1e39)
    refused(size, h.adamw_step, s, [g], 1, 1e-3, coefs=torch.ones(2, device="cuda"))
    refused(bad, h.adamw_step, s, [g], 1, 1e-3, moves=torch.zeros(10, dtype=BF16, device="cuda"))
    refused(size, h.adamw_step, s, [g], 1, 1e-3, moves=torch.zeros(11, device="cuda"))
    refused(bad, h.adamw_apply, s, None, 1e-3)
    refused(bad, h.adamw_apply, plain, z(), 1e-3)
    refused(bad, h.adamw_apply, s, z(), -1.0)
    refused(bad, h.adamw_apply, s, z(), 1e-3, weight_decay=math.nan)
    refused(bad, h.adamw_apply, s, z(), 1e-3, scale=math.inf)
    refused(bad, h.grad_norms, s, [g], 0.0)
    refused(bad, h.grad_norms, s, [g], math.nan)
    # the output across the gradients, in a place that is not their own
    room = torch.zeros(15, device="cuda")
    refused(bad, h.pack, plain, [room[5:]], out=room[:10])
    refused(bad, h.pack, plain, room[5:], out=room[:10])
    half = torch.zeros(20, dtype=BF16, device="cuda")
    refused(bad, h.pack, plain, [half[:10]], out=half.view(torch.float32))
    refused(bad, h.adamw_step, s, [room[5:]], 1, 1e-3, moves=room[:10])
    # a tensor twice, and buffers that overlap
    refused(bad, D.AdamWSet, h, [p, p], [z(), z()], [z(), z()])
    m = z()
    refused(bad, D.AdamWSet, h, [p], [m], [m])
    refused(bad, D.AdamWSet, h, [p], [None], [z()])
    refused(bad, D.AdamWSet, h, [p], [z().cpu()], [z()])
    refused(bad, D.AdamWSet, h, [p], [z().double()], [z()])
    refused(bad, D.AdamWSet, h, [p], [torch.zeros(20, device="cuda")[::2]], [z()])
    refused(size, D.AdamWSet, h, [p], [torch.zeros(11, device="cuda")], [z()])
    small = D.AdamWSet.zeros8(p)
    refused(bad, D.AdamWSet, h, [p], [small[0]], [small[0]], None, [small[2]], [small[3]])   # codes of the wrong kind
    refused(bad, D.AdamWSet, h, [p], [small[1]], [small[1].clone()], None, [small[2]], [small[3]])
    both = torch.zeros(15, device="cuda")
    refused(bad, D.AdamWSet, h, [p, z()], [both[:10], both[5:]], [z(), z()])
    before = p.clone()
    h.synchronize()
    assert torch.equal(p, before)


def test_second_moments_below_the_normal_range_count_under_the_root():
    """g = 2^-60: v = 0.001 g^2 lies below 2^-126, and with an eps of 1e-20 the root of it is nearly all that the move is
    divided by.  v is rounded to a multiple of 2^-149 (2^-20 of it, 2^-21 of its root); a dozen other roundings."""
    D = device_module()
    p, m, v = (torch.zeros(1030, device="cuda") for _ in range(3))
    h = D.Handle()
    s = D.AdamWSet(h, [p], [m], [v])
    g = 2.0 ** -60
    h.adamw_step(s, [torch.full((1030,), g, device="cuda")], 1, 1.0, eps=1e-20, weight_decay=0.0)
    want = g / (g + 1e-20)
    assert (np.abs(f64(p) + want) <= want * (2.0 ** -21 + 14 * U)).all()


def test_8bit_states_from_second_moments_that_are_not_above_zero():
    """-0, and what another format's rounding left below 0, are 0: not the block's largest."""
    D = device_module()
    n = 2 * BLOCK + 7
    p = torch.zeros(n, device="cuda")
    state = D.AdamWSet.zeros8(p)
    h = D.Handle()
    s = D.AdamWSet(h, [p], [state[0]], [state[1]], exp_avg_scales=[state[2]], exp_avg_sq_scales=[state[3]])
    v = torch.ones(n, device="cuda")
    v[3:n:5], v[4:n:5], v[0] = -0.0, -2.0, math.nan
    h.adamw_set_states(s, torch.ones(n, device="cuda"), v)
    got = h.adamw_states(s)[1]
    fine = v > 0
    # 1 is its block's largest: exact but for the three roundings of a code's value
    assert (got[fine] - 1).abs().max() <= 3.01 * U and got[1:][~fine[1:]].count_nonzero() == 0
    assert state[1][0] == 255 and (state[3] == 1).all()
    h.adamw_set_states(s, torch.ones(n, device="cuda"), -v.nan_to_num(1.0).abs())
    assert h.adamw_states(s)[1].count_nonzero() == 0 and state[3].count_nonzero() == 0
