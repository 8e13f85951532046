"""Thin torch-tensor front end of the cx_* C ABI (include/comprex_gfx950.h).

PyTorch only supplies device memory and the current HIP stream; every operation
below is one call into libcomprex_gfx950.so.  Messages are uint8/int32 CUDA tensors
in the reference's IndexPairs layout (src/compressor.hxx:559-565).
"""
import array
import ctypes as C

import numpy as np
import torch

from . import _lib
from ._lib import CX_BF16, CX_F16, CX_F32, CX_F64, CX_I32, ComprexError, check  # noqa: F401

_DT = {torch.float32: CX_F32, torch.float64: CX_F64, torch.int32: CX_I32}
# parameters and gradients of the operators over many tensors
_NUM = {torch.float32: CX_F32, torch.bfloat16: CX_BF16, torch.float16: CX_F16}
_CT = {torch.float32: C.c_float, torch.float64: C.c_double, torch.int32: C.c_int}


def pair_bytes(dtype):
    return 4 + torch.empty((), dtype=dtype).element_size()


def message_capacity(n, dtype):
    """Bytes of the largest message a vector of n elements can produce."""
    return 8 + n * pair_bytes(dtype)


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _dt(t):
    assert t.is_cuda and t.is_contiguous() and t.dim() == 1, "need 1-D contiguous device tensors"
    return _DT[t.dtype]


def _invalid(text, *args, code=_lib.CX_ERR_INVALID):
    return ComprexError(code, text % args)


# what the native look at a list calls its tensors' types
_TYPE_CODES = {**_NUM, torch.float8_e4m3fn: 100, torch.uint8: 101}


class TensorSet:
    """The tensors of a training step (cx_tensors): how many elements each has, for `Handle.grad_norms`
    and `Handle.pack`.  Made once per model and kept; belongs to its handle, whose stream everything a call takes
    has to be ready on, and a graph captured with it needs it alive."""

    def __init__(self, handle, sizes):
        self._make(handle, [int(n) for n in sizes], None)

    def _make(self, handle, sizes, state):
        self.lib, self.handle, self.sizes = handle.lib, handle, sizes
        self._on(handle.device)
        self._sizes = (C.c_longlong * len(sizes))(*sizes)
        self._addresses = _lib.tensor_lists().addresses
        self.total = sum(sizes)
        self._t = C.c_void_p()
        if any(n < 0 or n >= 1 << 62 for n in sizes):
            raise _invalid("a tensor cannot have %d elements", min(sizes) if min(sizes) < 0 else max(sizes))
        check(self.lib.cx_tensors_create(C.byref(self._t), handle._h, len(sizes), self._sizes, state))

    _addresses = None

    def _on(self, device):
        """Where its tensors live."""
        self.device, self._where = device, device.index

    def close(self):
        if getattr(self, "_t", None):
            self.lib.cx_tensors_destroy(self._t)
            self._t = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def gradients(self, grads):
        """A list of gradients (an entry per tensor, None: no gradient) or the flat vector of all of them, checked
        and ready for several calls in a row, each of which takes it in place of the list.  It holds addresses, not
        tensors."""
        if isinstance(grads, _lib.Grads):
            if grads.of is not self:
                raise _invalid("these gradients were checked for another set")
            return grads
        if isinstance(grads, torch.Tensor):
            if grads.dim() != 1 or grads.numel() != self.total:
                raise _invalid("a flat gradient has %d elements in one dimension, got %s", self.total,
                               tuple(grads.shape), code=_lib.CX_ERR_SIZE_MISMATCH)
            if grads.dtype not in _NUM or grads.device != self.device or not grads.is_contiguous():
                raise _invalid("a flat gradient is a contiguous fp32, bf16 or fp16 tensor on %s", self.device)
            found = _lib.Grads(_NUM[grads.dtype], None, grads.data_ptr())
            found.of = self
            return found
        if len(grads) != len(self.sizes):
            raise _invalid("%d gradients for %d tensors", len(grads), len(self.sizes), code=_lib.CX_ERR_SIZE_MISMATCH)
        n, each = len(grads), array.array("Q", bytes(8 * len(grads)))
        at = each.buffer_info()[0]
        code = self._addresses(grads, n, C.addressof(self._sizes), at, self._where) if self._addresses else -1
        if not 0 <= code <= CX_F16:  # something is out of the ordinary
            code = self._examine(grads, each)
        found = _lib.Grads(code, at, None)
        found.kept, found.of = each, self
        return found

    def _examine(self, grads, each):
        """The type of a list of gradients and their addresses, or what is wrong with it."""
        dtype = None
        for k, (g, n) in enumerate(zip(grads, self.sizes)):
            if g is None:
                each[k] = 0
                continue
            if dtype is None:
                dtype = g.dtype
            if g.numel() != n:
                raise _invalid("gradient of %d elements for a tensor of %d", g.numel(), n, code=_lib.CX_ERR_SIZE_MISMATCH)
            if g.dtype != dtype or g.device != self.device or not g.is_contiguous():
                raise _invalid("gradients are contiguous tensors of one type on %s", self.device)
            each[k] = g.data_ptr()
        if dtype is not None and dtype not in _NUM:
            raise _invalid("gradients are fp32, bf16 or fp16, not %s", dtype)
        return _NUM[dtype or torch.float32]

    def part_of(self, grads, start):
        """The gradients of this set out of those that were checked as a list for a larger one, from its tensor `start`
        on."""
        sizes = grads.of.sizes[start:start + len(self.sizes)]
        if grads.each is None or start < 0 or sizes != self.sizes or grads.of.device != self.device:
            raise _invalid("these are not the gradients of this set's tensors", code=_lib.CX_ERR_SIZE_MISMATCH)
        found = _lib.Grads(grads.type, grads.each + start * C.sizeof(C.c_void_p), None)
        found.kept, found.of = grads.kept, self
        return found

    def _new(self, n, dtype):
        """A vector for the handle's stream to write: of that stream's memory where another one is current."""
        # (torch.cuda.current_stream() makes an object each time: 2 us more)
        if torch._C._cuda_getCurrentRawStream(self._where) == self.handle.stream.cuda_stream:
            return torch.empty(n, dtype=dtype, device=self.device)
        with torch.cuda.stream(self.handle.stream):
            return torch.empty(n, dtype=dtype, device=self.device)

    def _coefs(self, coefs):
        if coefs is None:
            return None, 0
        if coefs.dtype != torch.float32 or coefs.device != self.device or not coefs.is_contiguous():
            raise _invalid("coefficients are a contiguous fp32 tensor on %s", self.device)
        return coefs.data_ptr(), coefs.numel()

    def _one(self, t, dtype, what):
        """Address of a one-element device tensor, None for None."""
        if t is None:
            return None
        if t.dtype != dtype or t.device != self.device or t.numel() != 1:
            raise _invalid("%s is one element of %s on %s", what, dtype, self.device)
        return t.data_ptr()

    def _vector(self, t, dtype, what):
        """A given vector of all elements, checked, or a new one."""
        if t is None:
            return self._new(self.total, dtype)
        if t.dtype != dtype or t.device != self.device or t.dim() != 1 or not t.is_contiguous():
            raise _invalid("%s is a contiguous vector of %s on %s", what, dtype, self.device)
        if t.numel() != self.total:
            raise _invalid("%s has %d elements, not %d", what, self.total, t.numel(), code=_lib.CX_ERR_SIZE_MISMATCH)
        return t


class AdamWSet(TensorSet):
    """A TensorSet with what `Handle.adamw_step` updates: lists with a tensor per parameter.  `params`: fp32, bf16
    or fp16; `masters`: None, or the fp32 weights that bf16 or fp16 parameters are rounded from.  Moments in 32 bits:
    `exp_avg` and `exp_avg_sq` fp32.  Moments in 8 bits: `exp_avg` float8_e4m3fn, `exp_avg_sq` uint8 codes
    (include/comprex_gfx950.h says what they stand for), and fp32 scales, one for every `BLOCK` elements of a
    tensor; `AdamWSet.zeros8` makes them.  The tensors are kept, and updated where they are: one that moves
    needs a new set."""

    BLOCK = 256

    def __init__(self, handle, params, exp_avg, exp_avg_sq, masters=None, exp_avg_scales=None, exp_avg_sq_scales=None):
        lists = [params, exp_avg, exp_avg_sq, masters, exp_avg_scales, exp_avg_sq_scales]
        lists = [None if x is None else list(x) for x in lists]
        params, exp_avg, exp_avg_sq, masters, exp_avg_scales, exp_avg_sq_scales = lists
        small = exp_avg_scales is not None
        if small != (exp_avg_sq_scales is not None):
            raise _invalid("8-bit moments need the scales of both")
        sizes = [p.numel() for p in params]
        if params and params[0].dtype not in _NUM:
            raise _invalid("parameters are fp32, bf16 or fp16, not %s", params[0].dtype)
        dtype = params[0].dtype if params else torch.float32
        if not params:
            lists[3] = None  # nothing to have masters of
        elif masters is not None and dtype == torch.float32:
            raise _invalid("fp32 parameters have no masters")
        blocks = [-(-n // self.BLOCK) for n in sizes]
        f32 = torch.float32
        wanted = [("params", dtype, sizes), ("exp_avg", torch.float8_e4m3fn if small else f32, sizes),
                  ("exp_avg_sq", torch.uint8 if small else f32, sizes), ("masters", f32, sizes),
                  ("exp_avg_scales", f32, blocks), ("exp_avg_sq_scales", f32, blocks)]
        self.kept, self._at, self._is = lists, [], []  # the lists; per list the addresses, the sizes and the type
        for got, (name, dt, ns) in zip(lists, wanted):
            if got is None:
                self._at.append(None)
                self._is.append(None)
                continue
            if len(got) != len(sizes):
                raise _invalid("%d %s for %d parameters", len(got), name, len(sizes), code=_lib.CX_ERR_SIZE_MISMATCH)
            at, counts = array.array("Q", bytes(8 * len(got))), array.array("q", ns)
            if _lib.tensor_lists().addresses(got, len(got), counts.buffer_info()[0], at.buffer_info()[0],
                                             -1 if handle.device.index is None else handle.device.index) != _TYPE_CODES[dt]:
                self._examine_list(got, ns, name, dt, handle.device, at)
            self._at.append(at)
            self._is.append((at.buffer_info()[0], counts, counts.buffer_info()[0], _TYPE_CODES[dt]))
        self.state_bits = 8 if small else 32
        at = [None if a is None else a.buffer_info()[0] for a in self._at]
        self._make(handle, sizes, C.byref(_lib.AdamwState(_NUM[dtype], self.state_bits, at[0], at[3], at[1], at[2], at[4],
                                                          at[5])))

    @staticmethod
    def _examine_list(tensors, sizes, name, dtype, device, at):
        """Raises what is wrong with a list, or takes its addresses."""
        for k, (t, n) in enumerate(zip(tensors, sizes)):
            if t.numel() != n:
                raise _invalid("%s has %d elements where %d belong", name, t.numel(), n, code=_lib.CX_ERR_SIZE_MISMATCH)
            if t.dtype != dtype or t.device != device or not t.is_contiguous():
                raise _invalid("%s are contiguous tensors of %s on %s", name, dtype, device)
            at[k] = t.data_ptr()

    def made_of(self, lists):
        """Whether the set was made of these tensors as and where they are now: lists in __init__'s order."""
        same = _lib.tensor_lists().unmoved
        return all(x is known is None or (x is not None and known is not None and
                                          same(x, len(self.sizes), known[0], known[2], known[3]))
                   for x, known in zip(lists, self._is))

    @classmethod
    def zeros8(cls, param):
        """(exp_avg, exp_avg_sq, exp_avg_scales, exp_avg_sq_scales) of a parameter at the start of training."""
        n = param.numel()
        return (torch.zeros(n, dtype=torch.uint8, device=param.device).view(torch.float8_e4m3fn),
                torch.zeros(n, dtype=torch.uint8, device=param.device),
                torch.zeros(-(-n // cls.BLOCK), device=param.device), torch.zeros(-(-n // cls.BLOCK), device=param.device))


class Handle:
    """One compressor clone's scratch + stream (cx_create / cx_destroy)."""

    def __init__(self, stream=None):
        self.lib = _lib.lib()
        self._h = C.c_void_p()
        if stream is None:
            stream = torch.cuda.current_stream()
        self.stream = stream
        self.device = torch.device("cuda", torch.cuda.current_device())
        check(self.lib.cx_create(C.byref(self._h), C.c_void_p(stream.cuda_stream)))

    def close(self):
        if self._h:
            self.lib.cx_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    RESERVE_COMPRESS, RESERVE_THRESHOLD, RESERVE_REDUCE, RESERVE_RLE, RESERVE_ALL = 1, 2, 4, 8, 15

    def reserve(self, n, dtype, paths=7):
        """Sizes the handle's scratch for vectors of up to n elements of `dtype` so that later calls
        on the named paths (an OR of the RESERVE_* bits; default: all but the run-length codec) never
        allocate (cx_reserve)."""
        check(self.lib.cx_reserve(self._h, _DT[dtype], int(n), int(paths)))

    def set_stream(self, stream):
        """Works on another stream from now on (waits for the one before, if it is another)."""
        if stream.cuda_stream != self.stream.cuda_stream:
            check(self.lib.cx_set_stream(self._h, C.c_void_p(stream.cuda_stream)))
        self.stream = stream

    def set_option(self, key, value):
        check(self.lib.cx_set_option(self._h, key.encode(), int(value)))

    def profile_read(self, max_out=1024):
        """Milliseconds of the streaming kernel of each compress since the last read
        (needs set_option("profile_stage", 1)); waits for the stream."""
        buf = (C.c_float * max_out)()
        n = C.c_int(0)
        check(self.lib.cx_profile_read(self._h, buf, max_out, C.byref(n)))
        return [buf[i] for i in range(n.value)]

    def synchronize(self):
        """Waits for the stream; raises the first device-side error recorded since the last call."""
        check(self.lib.cx_synchronize(self._h))

    # ---- thresholds ------------------------------------------------------
    def topk_threshold(self, vec, add_vec, topK, default_subsamples=1000, subsample_factor=10.0,
                       out=None, to_host=True):
        """ThresholdTopK.prepare_with (add_vec given) / prepare (add_vec None)."""
        dt = _dt(vec)
        host = _CT[vec.dtype]() if to_host else None
        check(self.lib.cx_topk_threshold(
            self._h, dt, _p(vec), _p(add_vec), vec.numel(), 0 if add_vec is None else add_vec.numel(),
            C.c_float(topK), int(default_subsamples), C.c_float(subsample_factor), _p(out),
            C.byref(host) if to_host else None))
        return host.value if to_host else None

    def topk_threshold_indexed(self, vec, add_vec, idx, topK, out=None, to_host=True):
        dt = _dt(vec)
        assert idx.dtype == torch.int32 and idx.is_cuda
        host = _CT[vec.dtype]() if to_host else None
        check(self.lib.cx_topk_threshold_indexed(
            self._h, dt, _p(vec), _p(add_vec), vec.numel(), _p(idx), idx.numel(), C.c_float(topK), _p(out),
            C.byref(host) if to_host else None))
        return host.value if to_host else None

    def threshold_slot(self):
        """Raw device address of the handle's own threshold slot."""
        return self.lib.cx_threshold_slot(self._h)

    # ---- codec -------------------------------------------------------------
    def compress(self, out_msg, data, update, thr=None, d_thr=None, size_prefix=None, sync=True):
        """compress / compress_update / compress_add_update by which of data/update is None.
        thr: host scalar; else d_thr: 1-element device tensor; else the handle's slot.
        Returns bytes written when sync, else None."""
        ref = data if data is not None else update
        dt = _DT[ref.dtype] if ref is not None else CX_F32
        n = ref.numel() if ref is not None else 0
        if data is not None and update is not None and data.numel() != update.numel():
            raise ComprexError(_lib.CX_ERR_SIZE_MISMATCH,
                               "Compressor: Update vector size (%d) is not equal data vector size (%d)!"
                               % (update.numel(), data.numel()))
        hthr = None
        if thr is not None:
            hthr = _CT[ref.dtype](thr)
        nbytes = C.c_int(0)
        check(self.lib.cx_ip_compress(
            self._h, dt, _p(out_msg), out_msg.numel() * out_msg.element_size(), _p(data), _p(update), n,
            C.byref(hthr) if hthr is not None else None, _p(d_thr), _p(size_prefix),
            C.byref(nbytes) if sync else None))
        return nbytes.value if sync else None

    def compress_topk(self, out_msg, data, update, topk, d_thr=None, size_prefix=None):
        """Whole-vector ThresholdTopK(topk) on update + data and compress_add_update in one call
        (a single pass over the vectors when they are large).  The threshold is left in d_thr
        (1-element device tensor) or the handle's slot.  Returns bytes written."""
        if data.numel() != update.numel():
            raise ComprexError(_lib.CX_ERR_SIZE_MISMATCH, "vector sizes must be the same!")
        nbytes = C.c_int(0)
        check(self.lib.cx_ip_compress_topk(
            self._h, _dt(update), _p(out_msg), out_msg.numel() * out_msg.element_size(), _p(data), _p(update),
            update.numel(), float(topk), _p(d_thr), _p(size_prefix), C.byref(nbytes)))
        return nbytes.value

    def write_step(self, out_msg, data, update, topk, default_subsamples=1000, subsample_factor=10.0, idx=None,
                   d_thr=None, size_prefix=None, sync=True):
        """ThresholdTopK(topk, default_subsamples, subsample_factor).prepare_with(update, data) and
        compress_add_update in one call (cx_ip_write_step); idx: int32 device tensor of sample
        positions instead of the strided rule.  Returns bytes written when sync."""
        if data.numel() != update.numel():
            raise ComprexError(_lib.CX_ERR_SIZE_MISMATCH, "vector sizes must be the same!")
        nbytes = C.c_int(0)
        check(self.lib.cx_ip_write_step(
            self._h, _dt(update), _p(out_msg), out_msg.numel() * out_msg.element_size(), _p(data), _p(update),
            update.numel(), float(topk), int(default_subsamples), float(subsample_factor), _p(idx),
            0 if idx is None else idx.numel(), _p(d_thr), _p(size_prefix), C.byref(nbytes) if sync else None))
        return nbytes.value if sync else None

    def get_option(self, key):
        v = C.c_int(0)
        check(self.lib.cx_get_option(self._h, key.encode(), C.byref(v)))
        return v.value

    # ---- run-length codec -------------------------------------------------
    def rle_compress(self, out_msg, data, update, thr=None, d_thr=None, size_prefix=None, sync=True):
        """CompressorRLE: as compress(), but |x| >= thr is sent and the message carries values
        and run lengths instead of (index, value) pairs.  Returns bytes written when sync."""
        ref = data if data is not None else update
        if ref is None:
            raise ComprexError(_lib.CX_ERR_INVALID, "Compression needs a valid input vector!")
        if data is not None and update is not None and data.numel() != update.numel():
            raise ComprexError(_lib.CX_ERR_SIZE_MISMATCH,
                               "Compressor: Update vector size (%d) is not equal data vector size (%d)!"
                               % (update.numel(), data.numel()))
        hthr = _CT[ref.dtype](thr) if thr is not None else None
        nbytes = C.c_int(0)
        check(self.lib.cx_rle_compress(
            self._h, _DT[ref.dtype], _p(out_msg), out_msg.numel() * out_msg.element_size(), _p(data), _p(update),
            ref.numel(), C.byref(hthr) if hthr is not None else None, _p(d_thr), _p(size_prefix),
            C.byref(nbytes) if sync else None))
        return nbytes.value if sync else None

    def rle_decompress(self, out, msg):
        """Returns the vector length the message carries (what the reference's decoder returns)."""
        n = C.c_int(0)
        check(self.lib.cx_rle_decompress(self._h, _dt(out), _p(out), out.numel(), _p(msg), C.byref(n)))
        return n.value

    def rle_add(self, out, msg):
        check(self.lib.cx_rle_add(self._h, _dt(out), _p(out), out.numel(), _p(msg)))

    def decompress(self, out, msg, sync=True):
        nbytes = C.c_int(0)
        check(self.lib.cx_ip_decompress(self._h, _dt(out), _p(out), out.numel(), _p(msg),
                                        C.byref(nbytes) if sync else None))
        return nbytes.value if sync else None

    def add(self, out, msg, check_header=True, any_order=False):
        """any_order: look at the indices first (one more wait) and apply a message that is not
        index-sorted pair after pair, as the reference's loop does (CX_ADD_ANY_ORDER)."""
        check(self.lib.cx_ip_add(self._h, _dt(out), _p(out), out.numel(), _p(msg),
                                 2 if any_order else (1 if check_header else 0)))

    def reduce(self, out, msgs, accumulate=False, mode=0, any_order=False):
        arr = (C.c_void_p * len(msgs))(*[m.data_ptr() for m in msgs])
        check(self.lib.cx_ip_reduce(self._h, _dt(out), _p(out), out.numel(), arr, len(msgs),
                                    1 if accumulate else 0, int(mode) | (4 if any_order else 0)))

    # ---- residual maintenance ---------------------------------------------
    def zero(self, v):
        check(self.lib.cx_zero(self._h, _dt(v), _p(v), v.numel()))

    def add_vec(self, data, rests):
        if data.numel() != rests.numel():
            raise ComprexError(_lib.CX_ERR_SIZE_MISMATCH, "Vector of size %d does not match Rests Vector of size %d!"
                               % (data.numel(), rests.numel()))
        check(self.lib.cx_add_vec(self._h, _dt(data), _p(data), _p(rests), data.numel()))

    def threshold_apply(self, vec, thr, split=False):
        high = torch.empty_like(vec)
        low = torch.empty_like(vec) if split else None
        hthr = _CT[vec.dtype](thr)
        check(self.lib.cx_threshold_apply(self._h, _dt(vec), _p(high), _p(low), _p(vec), vec.numel(),
                                          C.byref(hthr), None))
        return (high, low) if split else high


    # ---- many tensors ------------------------------------------------------
    def grad_norms(self, tensors, grads, max_norm=None, each=False, scale=1.0, norms=None, coefs=None, nonfinite=None):
        """Norms of `scale` times the gradients of a TensorSet and their clip coefficients: (norms, coefs,
        nonfinite), on the device.  norms[t] is tensor t's, norms[-1] that of all; coefs: one, from the norm of
        all, or with `each` one for every tensor from its own (max_norm None clips nothing); nonfinite: int32, 1
        where a gradient holds an infinity or NaN.  `grads`: a list (None: no gradient) or the flat vector."""
        count = len(tensors.sizes)
        g = tensors.gradients(grads)
        out = []
        for t, n, dt, what in ((norms, count + 1, torch.float32, "norms"), (coefs, count if each else 1, torch.float32, "coefs"),
                               (nonfinite, 1, torch.int32, "nonfinite")):
            if t is None:
                t = tensors._new(n, dt)
            elif t.dtype != dt or t.device != tensors.device or t.numel() != n or not t.is_contiguous():
                raise _invalid("%s: %d contiguous elements of %s on %s", what, n, dt, tensors.device)
            out.append(t)
        check(self.lib.cx_grad_norms(self._h, tensors._t, g, scale, float("inf") if max_norm is None else max_norm,
                                     1 if each else 0, out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr()))
        return tuple(out)

    def pack(self, tensors, grads, out=None, coefs=None, scale=1.0, skip=None):
        """The gradients of a TensorSet, times coefs (one, or one per tensor) and scale, back to back in a flat
        fp32 vector: what the compressor and the allreduce schedules take.  `skip` (int32, e.g. grad_norms'
        nonfinite) other than 0: all zeros."""
        g = tensors.gradients(grads)
        out = tensors._vector(out, torch.float32, "the flat vector")
        at, n = tensors._coefs(coefs)
        check(self.lib.cx_pack(self._h, tensors._t, g, at, n, scale, tensors._one(skip, torch.int32, "skip"),
                               out.data_ptr()))
        return out

    def adamw_step(self, tensors, grads, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, coefs=None, scale=1.0,
                   skip=None, moves=None, seed=None):
        """One AdamW step on an AdamWSet with the gradients times coefs and scale (cx_adamw_step).  `grads`: a
        list (None: leave this tensor alone) or the flat vector; `step`: which step this is, from 1, or an int32
        device tensor that the call advances; `lr`: a number or an fp32 device tensor; `skip` (int32) other than
        0: nothing changes.  With `moves`, a flat fp32 vector, the moments take the step and what the weights would
        lose goes there, for an exchange between ranks and `adamw_apply` (a tensor without a gradient: its part is
        left as it is; skipped: zeros).  `seed`, a number from 1 to 2^64 - 1: moments in 8 bits are rounded stochastically
        with noise from it, the step's count and an element's place, and follow their gradients over many steps, which
        moments rounded to nearest (None) do not."""
        if seed is not None and not 0 < seed < 1 << 64:
            raise _invalid("a seed is a number from 1 to 2^64 - 1, not %s", seed)
        g = tensors.gradients(grads)
        on_device = isinstance(step, torch.Tensor)
        d_lr = isinstance(lr, torch.Tensor)
        at, n = tensors._coefs(coefs)
        check(self.lib.cx_adamw_step_seeded(self._h, tensors._t, g, _lib.AdamwArgs(
            0.0 if d_lr else lr, betas[0], betas[1], eps, weight_decay, scale, 0 if on_device else step,
            tensors._one(step, torch.int32, "step") if on_device else None,
            tensors._one(lr, torch.float32, "lr") if d_lr else None, at, n, tensors._one(skip, torch.int32, "skip"),
            None if moves is None else tensors._vector(moves, torch.float32, "moves").data_ptr()), seed or 0))

    def adamw_apply(self, tensors, moves, lr, weight_decay=0.01, scale=1.0):
        """The weights of an AdamWSet after `scale` times the flat vector of moves (adamw_step) and the decay:
        w (1 - lr weight_decay) - scale moves."""
        if moves is None:
            raise _invalid("needs the moves")
        d_lr = isinstance(lr, torch.Tensor)
        check(self.lib.cx_adamw_apply(self._h, tensors._t, tensors._vector(moves, torch.float32, "moves").data_ptr(), scale,
                                      0.0 if d_lr else lr, tensors._one(lr, torch.float32, "lr") if d_lr else None,
                                      weight_decay))

    def adamw_states(self, tensors, dtype=torch.float32, exp_avg=None, exp_avg_sq=None):
        """What the 8-bit moments of an AdamWSet stand for: (exp_avg, exp_avg_sq), flat vectors of `dtype`."""
        if dtype not in _NUM:
            raise _invalid("values are fp32, bf16 or fp16, not %s", dtype)
        m, v = tensors._vector(exp_avg, dtype, "exp_avg"), tensors._vector(exp_avg_sq, dtype, "exp_avg_sq")
        check(self.lib.cx_adamw_states(self._h, tensors._t, _NUM[dtype], m.data_ptr(), v.data_ptr()))
        return m, v

    def adamw_set_states(self, tensors, exp_avg, exp_avg_sq):
        """Sets the 8-bit moments of an AdamWSet from flat fp32 vectors (an exp_avg_sq below 0 counts as 0)."""
        if exp_avg is None or exp_avg_sq is None:
            raise _invalid("needs the values of both moments")
        check(self.lib.cx_adamw_set_states(self._h, tensors._t, tensors._vector(exp_avg, torch.float32, "exp_avg").data_ptr(),
                                           tensors._vector(exp_avg_sq, torch.float32, "exp_avg_sq").data_ptr()))


def message_to_numpy(msg, nbytes):
    """First nbytes of a device message tensor as a uint8 numpy array."""
    raw = msg.view(torch.uint8) if msg.dtype != torch.uint8 else msg
    return raw[:nbytes].cpu().numpy()
