"""What the operators over many tensors refuse before anything reaches a device: the checks of the Python
front end on host tensors, and those of the C entry point that makes a set."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from comprex_amd import _lib
from comprex_amd._lib import ComprexError
from comprex_amd.device import AdamWSet, Handle, TensorSet

F32 = torch.float32


def host_set(sizes, cls=TensorSet):
    """A set whose checks run on host tensors; it has no device part."""
    s = cls.__new__(cls)
    s.sizes, s.total = sizes, sum(sizes)
    s._on(torch.device("cpu"))
    return s


def refused(code, f, *args, **kw):
    with pytest.raises(ComprexError) as e:
        f(*args, **kw)
    assert e.value.code == code


def test_gradients_are_checked():
    s = host_set([3, 0, 5])
    good = [torch.zeros(3), torch.zeros(0), torch.zeros(1, 5)]
    assert s.gradients(good).type == _lib.CX_F32
    assert s.gradients([None, None, torch.zeros(5, dtype=torch.bfloat16)]).type == _lib.CX_BF16
    assert s.gradients([None] * 3).type == _lib.CX_F32
    assert s.gradients(torch.zeros(8, dtype=torch.float16)).type == _lib.CX_F16
    bad, size = _lib.CX_ERR_INVALID, _lib.CX_ERR_SIZE_MISMATCH
    ready = s.gradients(good)
    assert s.gradients(ready) is ready
    refused(bad, host_set([3, 0, 5]).gradients, ready)                                    # made for another set
    refused(bad, host_set([8]).gradients, s.gradients(torch.zeros(8)))
    refused(size, s.gradients, good[:2])
    refused(size, s.gradients, [torch.zeros(4), good[1], good[2]])
    refused(size, s.gradients, torch.zeros(7))
    refused(size, s.gradients, torch.zeros(2, 4))
    refused(bad, s.gradients, [torch.zeros(3, dtype=torch.bfloat16), None, torch.zeros(5)])   # two types
    refused(bad, s.gradients, [torch.zeros(3, dtype=torch.float64), None, None])
    refused(bad, s.gradients, torch.zeros(8, dtype=torch.int32))
    refused(bad, s.gradients, [torch.zeros(6)[::2], None, None])                             # strided
    refused(bad, s.gradients, [None, None, torch.zeros(5, device="meta")])
    refused(bad, s.gradients, torch.zeros(16)[::2])


def test_a_part_of_the_gradients_is_the_list_from_there_on():
    s, part = host_set([3, 0, 5, 5]), host_set([0, 5])
    grads = [torch.zeros(3), torch.zeros(0), None, torch.ones(5)]
    whole = s.gradients(grads)
    own = part.part_of(whole, 1)
    assert own.of is part and list((C.c_void_p * 2).from_address(own.each)) == [None, None]
    assert part.gradients(own) is own
    assert list((C.c_void_p * 1).from_address(host_set([5]).part_of(whole, 3).each)) == [grads[3].data_ptr()]
    for n, start in (([0, 5], 0), ([0, 5], 2), ([5, 5, 5], 2), ([5], 4), ([5], -1)):
        refused(_lib.CX_ERR_SIZE_MISMATCH, host_set(n).part_of, whole, start)
    refused(_lib.CX_ERR_SIZE_MISMATCH, host_set([8]).part_of, host_set([8]).gradients(torch.zeros(8)), 0)  # a flat one


def test_the_native_look_at_lists_answers_the_ordinary_case_only():
    """Host tensors, things that are no tensors and lists of another length are left to the checks in Python."""
    L = _lib.tensor_lists()
    sizes, out = (C.c_longlong * 2)(3, 4), (C.c_uint64 * 2)(7, 7)
    look = lambda x, n=2: L.addresses(x, n, C.addressof(sizes), C.addressof(out), 0)  # noqa: E731
    assert look([None, None]) == _lib.CX_F32 and list(out) == [0, 0]
    for x in ([torch.zeros(3), None], [None, 5], [None], [None] * 3, (None, None), "ab", [None, torch.zeros(4, device="meta")],
              [torch.zeros(3).to_sparse(), None]):
        assert look(x) == -1
    with pytest.raises(TypeError):
        L.addresses([], 0)
    with pytest.raises(TypeError):
        L.unmoved([], 0)
    with pytest.raises((TypeError, OverflowError)):
        L.addresses([], 0, -1, 0, 0)
    a, b = torch.zeros(3), torch.zeros(4)
    at = (C.c_uint64 * 2)(a.data_ptr(), b.data_ptr())
    assert L.unmoved([a, b], 2, C.addressof(at))
    for x in ([b, a], [a, b.clone()], [a], [a, None], (a, b), [a, 5]):
        assert not L.unmoved(x, 2, C.addressof(at))


def test_vectors_coefficients_and_single_values_are_checked():
    s = host_set([3, 5])
    bad, size = _lib.CX_ERR_INVALID, _lib.CX_ERR_SIZE_MISMATCH
    v = torch.zeros(8)
    assert s._vector(v, F32, "x") is v
    refused(size, s._vector, torch.zeros(9), F32, "x")
    refused(bad, s._vector, torch.zeros(8, dtype=torch.float64), F32, "x")
    refused(bad, s._vector, torch.zeros(16)[::2], F32, "x")
    refused(bad, s._vector, torch.zeros(2, 4), F32, "x")
    assert s._coefs(None) == (None, 0) and s._coefs(torch.ones(2))[1] == 2
    refused(bad, s._coefs, torch.ones(2, dtype=torch.float64))
    refused(bad, s._coefs, torch.ones(4)[::2])
    assert s._one(None, torch.int32, "x") is None
    refused(bad, s._one, torch.zeros(1), torch.int32, "x")
    refused(bad, s._one, torch.zeros(2, dtype=torch.int32), torch.int32, "x")


class HostHandle:
    device = torch.device("cpu")
    lib = None
    _h = None


def test_adamw_lists_are_checked():
    bad, size = _lib.CX_ERR_INVALID, _lib.CX_ERR_SIZE_MISMATCH
    z = lambda n=300, dt=F32: torch.zeros(n, dtype=dt)  # noqa: E731
    half, codes, bytes_ = z(dt=torch.bfloat16), z(dt=torch.uint8).view(torch.float8_e4m3fn), z(dt=torch.uint8)
    h = HostHandle()
    refused(bad, AdamWSet, h, [z(dt=torch.float64)], [z()], [z()])
    refused(size, AdamWSet, h, [z()], [z(), z()], [z()])
    refused(size, AdamWSet, h, [z()], [z(299)], [z()])
    refused(bad, AdamWSet, h, [z(), half], [z(), z()], [z(), z()])           # two types of parameters
    refused(bad, AdamWSet, h, [z()], [z()], [z()], [z()])                    # masters of fp32 parameters
    refused(bad, AdamWSet, h, [half], [z()], [z()], [half])                  # masters in 16 bits
    refused(bad, AdamWSet, h, [half], [half], [half])                        # moments in 16 bits
    refused(bad, AdamWSet, h, [z()], [codes], [bytes_])                      # 8 bits without scales
    refused(bad, AdamWSet, h, [z()], [codes], [bytes_], None, [z(2)])        # ... without one of them
    refused(size, AdamWSet, h, [z()], [codes], [bytes_], None, [z(1)], [z(2)])
    refused(bad, AdamWSet, h, [z()], [z()], [bytes_], None, [z(2)], [z(2)])
    refused(bad, AdamWSet, h, [z(600)[::2]], [z()], [z()])
    m, v, ms, vs = AdamWSet.zeros8(z(257))
    assert m.dtype == torch.float8_e4m3fn and v.dtype == torch.uint8 and ms.numel() == vs.numel() == 2


def test_c_entry_point_checks_before_it_touches_a_device():
    """The handle's memory is not looked at before the arguments are sound: zeros stand for one."""
    L = _lib.lib()
    fake = C.create_string_buffer(1 << 14)
    out = C.c_void_p(1)
    longs = lambda *x: (C.c_longlong * len(x))(*x)  # noqa: E731

    def create(count, sizes, state=None, handle=fake):
        rc = L.cx_tensors_create(C.byref(out), handle, count, sizes, state)
        assert not out.value
        return rc

    bad = _lib.CX_ERR_INVALID
    assert L.cx_tensors_create(None, fake, 0, None, None) == bad
    assert create(1, longs(4), handle=None) == bad
    assert create(-1, longs(4)) == bad
    assert create(1, None) == bad
    assert create(1, longs(-4)) == bad
    assert create(1, longs(1 << 41)) == bad
    assert create(2, longs(1 << 40, 1 << 40)) == bad
    assert create(2, longs(1 << 33, 1)) == bad
    assert create((1 << 20) + 1, longs(1)) == bad

    def state(**kw):
        a = (C.c_float * 64)()
        base = C.addressof(a)
        got = dict(param_type=_lib.CX_F32, state_bits=32, params=[base], masters=None, exp_avg=[base + 64],
                   exp_avg_sq=[base + 128], exp_avg_scales=None, exp_avg_sq_scales=None)
        got.update({k: [x and base + x for x in v] if isinstance(v, list) else v for k, v in kw.items()})
        keep = {k: (C.c_void_p * len(v))(*v) if isinstance(v, list) else v for k, v in got.items()}
        s = _lib.AdamwState(**{k: C.cast(v, C.c_void_p) if isinstance(v, C.Array) else v for k, v in keep.items()})
        s.kept = a, keep
        return s

    one = longs(16)
    assert create(1, one, state(param_type=_lib.CX_F64)) == bad
    assert create(1, one, state(state_bits=16)) == bad
    assert create(1, one, state(masters=[192])) == bad                              # fp32 has none
    assert create(1, one, state(exp_avg=None)) == bad
    assert create(1, one, state(exp_avg_scales=[192])) == bad                       # scales in 32 bits
    assert create(1, one, state(state_bits=8, exp_avg_scales=[192])) == bad         # one of two scales
    assert create(1, one, state(exp_avg=[66])) == bad                               # misaligned
    assert create(1, one, state(exp_avg_sq=[124])) == bad                           # overlaps exp_avg
    assert create(1, one, state(exp_avg_sq=[64])) == bad                            # the same
    assert create(2, longs(16, 16), state(params=[4, 8], exp_avg=[64, 64], exp_avg_sq=[128, 128])) == bad
    assert L.cx_tensors_destroy(None) == 0
    for rc in (L.cx_grad_norms(None, None, None, 1.0, 1.0, 0, None, None, None),
               L.cx_pack(None, None, None, None, 0, 1.0, None, None), L.cx_adamw_step(None, None, None, None),
               L.cx_adamw_apply(None, None, None, 1.0, 1.0, None, 0.0), L.cx_adamw_states(None, None, 0, None, None), L.cx_adamw_set_states(None, None, None, None)):
        assert rc == bad
    if _lib.lib().cx_device_count() == 0:
        assert create(1, one, state()) == _lib.CX_ERR_HIP                           # sound, but there is no device


def test_set_states_needs_both_vectors():
    h = Handle.__new__(Handle)
    h.lib, h._h = None, None
    refused(_lib.CX_ERR_INVALID, h.adamw_set_states, host_set([4]), None, torch.zeros(4))
    refused(_lib.CX_ERR_INVALID, h.adamw_set_states, host_set([4]), torch.zeros(4), None)


def test_the_library_is_built_without_torch():
    """A program in C or C++ needs the library alone; where torch is, its module is built too."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comprex_amd", "csrc")
    for python, lists in (("false", False), ("python3", True), ("python3 -S", False)):
        r = subprocess.run(["make", "-n", "-B", "-C", csrc, "PYTHON=" + python, "all"], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stderr
        assert "libcomprex_gfx950.so" in r.stdout and ("_tensor_lists.so" in r.stdout) == lists
