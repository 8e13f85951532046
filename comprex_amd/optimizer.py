"""Optimizers whose gradient exchange is one of the compressed allreduce schedules: `ComprexOptimizer` (momentum
SGD) and `ComprexAdamW`.

`ComprexOptimizer` is the PyTorch counterpart of the reference's Keras optimizer
(keras/comprex_optimizer.py:7-170):

Per step and rank (blob mode, keras/comprex_optimizer.py:97-133): every gradient is clipped to
`pre_clipnorm`, turned into a local momentum term `m = momentum * m + lr * g`, all terms are
concatenated into ONE flat device buffer, the allreduce works in place on that buffer (device
pointer handed straight to the C ABI), the result is divided by the number of ranks, and
`w = (1 - weight_decay) * w - avg_m`.  With a single rank nothing is exchanged and, as in the
reference (:134-141,155-163), the update is `m = momentum * m + g; w = (1 - wd) * w - m`.

`ComprexAdamW` has no counterpart in the reference and keeps its order: every rank's moments follow its own
gradients (clipped together), what its weights would lose to the step is exchanged, and every rank applies the
average.  The schedules deliver each rank another vector and make up for it later; sums bear that, moments of
such vectors would not and the ranks' weights would drift apart.  Clipping and the step run as a few launches
over all tensors (`Handle.grad_norms`, `adamw_step`, `adamw_apply`), and nothing waits for the device.
"""
import itertools
import operator

import torch

from . import pygpi
from ._lib import ComprexError
from .device import AdamWSet, Handle, TensorSet

_SCHEDULES = {
    "comprex_alltoone": pygpi.Comprex_AllToOneAllreduce,
    "comprex_ring": pygpi.Comprex_RingAllreduce,
    "comprex_bigring": pygpi.Comprex_BigRingAllreduce,
}


def _make_allreduce(kind, gaspi_env, size, compression_ratio, size_factor):
    ar = _SCHEDULES[kind](gaspi_env)
    if kind == "comprex_alltoone":
        ar.setup_connections(size, 1, 0, compression_ratio, size_factor)
    else:
        ar.setup_connections(size, 1, compression_ratio, size_factor)
    return ar


class ComprexOptimizer(torch.optim.Optimizer):
    def __init__(self, params, gaspi_env, learning_rate=0.01, momentum=0.9, compression_ratio=0.01,
                 allreduce_type="comprex_bigring", size_factor=1.0, pre_clipnorm=5.0, weight_decay=0.0):
        if not 0 <= momentum <= 1:
            raise ValueError("`momentum` must be between [0, 1].")
        if allreduce_type not in _SCHEDULES:
            raise ValueError("AllreduceOp with name %s is not known!" % allreduce_type)
        super().__init__(params, dict(lr=learning_rate, momentum=momentum, weight_decay=weight_decay))
        self.gaspi_env = gaspi_env
        self.compression_ratio = compression_ratio
        self.size_factor = size_factor
        self.allreduce_type = allreduce_type
        self.pre_clipnorm = pre_clipnorm
        self.allreduce = None
        self.blob = None

    def set_compression_ratio(self, compression_ratio):
        self.compression_ratio = compression_ratio
        if self.allreduce is not None:
            self.allreduce.set_compression_ratio(compression_ratio)

    def _create_allreduce(self, size):
        return _make_allreduce(self.allreduce_type, self.gaspi_env, size, self.compression_ratio, self.size_factor)

    @torch.no_grad()
    def step(self):
        ranks = self.gaspi_env.get_ranks()
        entries = []
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum" not in state:
                    state["momentum"] = torch.zeros_like(p)
                entries.append((p, group, state["momentum"]))
        if ranks == 1:
            for p, group, mom in entries:
                mom.mul_(group["momentum"]).add_(p.grad)
                p.mul_(1 - group["weight_decay"]).sub_(mom)
            return
        total = sum(p.numel() for p, _, _ in entries)
        if self.blob is None or self.blob.numel() != total:
            # a channel grows for a larger vector: what an exchange before this one sent has to be read by then
            self.gaspi_env.barrier()
            self.blob = torch.empty(total, dtype=torch.float32, device=entries[0][0].device)
            self.allreduce = self._create_allreduce(total)
        off = 0
        for p, group, mom in entries:
            g = p.grad
            norm = g.norm()
            if norm > self.pre_clipnorm:  # tf.clip_by_norm
                g = g * (self.pre_clipnorm / norm)
            mom.mul_(group["momentum"]).add_(g, alpha=group["lr"])
            self.blob[off:off + p.numel()].copy_(mom.reshape(-1))
            off += p.numel()
        self.allreduce.apply(self.blob)  # in place, on the device
        self.blob.div_(ranks)
        off = 0
        for p, group, _ in entries:
            p.mul_(1 - group["weight_decay"]).sub_(self.blob[off:off + p.numel()].view_as(p))
            off += p.numel()


#: the exchange counts in 32-bit integers
_MOST_EXCHANGED = (1 << 31) - 1
_LARGEST = torch.finfo(torch.float32).max
_STATE = ("exp_avg", "exp_avg_sq", "master", "exp_avg_scales", "exp_avg_sq_scales")  # an AdamWSet's lists


class _Part:
    """Parameters of one group that share a type and a width of the moments, and their AdamWSet.  `counts`: where the
    steps are counted on the device, a count for each number that the parameters begin with, and whose it is."""

    def __init__(self, group, params):
        self.group, self.params, self.states, self.dtype = group, params, [], params[0].dtype
        self.set, self.counts, self.seed = None, [], None

    def tensors(self, state):
        """params, exp_avg, exp_avg_sq, masters, scales of both: lists, or None."""
        self.states = list(map(state.__getitem__, self.params))
        return [self.params] + [list(map(operator.itemgetter(k), self.states)) if k in self.states[0] else None
                                for k in _STATE]

    def count_on(self, device):
        members = {}
        for k, s in enumerate(self.states):
            members.setdefault(s["step"], set()).add(k)
        self.counts = [(torch.full((1,), n, dtype=torch.int32, device=device), ks) for n, ks in members.items()]


class _Kind:
    """The parts whose gradients share a type, and the set of all their gradients."""

    def __init__(self, parts):
        self.parts, self.set = parts, None
        self.params = [p for part in parts for p in part.params]

    def gradients(self):
        """(the list, the same checked for the set); (list, None) where there is none at all."""
        grads = list(map(operator.attrgetter("grad"), self.params))
        try:
            return grads, self.set.gradients(grads) if any(g is not None for g in grads) else None
        except (ComprexError, RuntimeError):  # perhaps one of another layout
            if any(g is not None and g.is_sparse for g in grads):
                raise RuntimeError("ComprexAdamW takes dense gradients only") from None
            grads = [None if g is None else g.contiguous() for g in grads]
            return grads, self.set.gradients(grads)


class ComprexAdamW(torch.optim.Optimizer):
    """AdamW over the compressed allreduce.

    Per step and rank: the gradients are clipped together to the norm `clip_norm` (None: not at all) and the
    moments take them.  With one rank the weights follow at once.  With several, the moves of all weights go as one
    flat fp32 vector through the exchange and come back summed, and every weight takes a `1 / ranks` of its sum
    and its decay; one without a gradient here may have had one elsewhere.

    state_bits 8: the moments of parameters of at least `min_8bit_size` elements take one byte each, rounded
    stochastically, with the same noise in a run that is repeated or goes on from a saved state.
    master_weights: bf16 and fp16 parameters get fp32 weights of which they are the rounded values.
    skip_nonfinite: a gradient with an infinity or NaN anywhere leaves its rank's moments and count as they are,
    and its weights too or, with several ranks, its part of the sum zero; decided on the device, where the steps
    are counted then (a parameter without a gradient counts along with those it is stepped with).

    Parameters are contiguous and on one GPU.  The layout of the exchanged vector follows the parameters that require
    a gradient: one that is frozen or released starts a new exchange, without what the old one held back (`flush`
    delivers that before).  `load_state_dict`, which every rank calls, drops what is held back.  With several
    ranks a step leaves the stream it ran on as the environment's user stream of its thread: a program with exchanges of
    its own sets theirs before them.  A program that captures its steps in a graph calls `Handle.grad_norms` and
    `Handle.adamw_step` itself."""

    def __init__(self, params, gaspi_env, learning_rate=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
                 clip_norm=None, state_bits=32, min_8bit_size=4096, master_weights=True, skip_nonfinite=False,
                 compression_ratio=0.01, allreduce_type="comprex_bigring", size_factor=1.0):
        if allreduce_type not in _SCHEDULES:
            raise ValueError("AllreduceOp with name %s is not known!" % allreduce_type)
        if state_bits not in (8, 32):
            raise ValueError("`state_bits` must be 8 or 32.")
        if clip_norm is not None and not clip_norm > 0:
            raise ValueError("`clip_norm` must be above 0.")
        super().__init__(params, dict(lr=learning_rate, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        for group in self.param_groups:
            for p in group["params"]:
                self._check(p)
        self.gaspi_env = gaspi_env
        self.clip_norm, self.state_bits, self.min_8bit_size = clip_norm, state_bits, min_8bit_size
        self.master_weights, self.skip_nonfinite = master_weights, skip_nonfinite
        self.compression_ratio, self.allreduce_type, self.size_factor = compression_ratio, allreduce_type, size_factor
        self.handle = self.allreduce = self.blob = self._parts = None
        self._order = []

    @staticmethod
    def _check(p):
        if not p.is_cuda or not p.is_contiguous() or p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise ValueError("parameters are contiguous fp32, bf16 or fp16 tensors on a GPU")

    @staticmethod
    def _check_group(group):
        """Refuses what the step does not do (torch's own optimizers save such groups) or would refuse."""
        if group.get("amsgrad") or group.get("maximize"):
            raise ValueError("`amsgrad` and `maximize` are not supported.")
        if group["weight_decay"] and not group.get("decoupled_weight_decay", True):
            raise ValueError("the weight decay is AdamW's: it does not go through the moments.")
        if not all(0 <= b < 1 for b in group["betas"]):
            raise ValueError("`betas` must be in [0, 1).")
        if not 1e-20 <= group["eps"] <= _LARGEST:
            raise ValueError("`eps` must be finite and at least 1e-20.")
        if not 0 <= group["weight_decay"] <= _LARGEST:
            raise ValueError("`weight_decay` must be finite and not negative.")
        if not isinstance(group["lr"], torch.Tensor) and not 0 <= group["lr"] <= _LARGEST:
            raise ValueError("the learning rate must be finite and not negative.")

    def set_compression_ratio(self, compression_ratio):
        self.compression_ratio = compression_ratio
        if self.allreduce is not None:
            self.allreduce.set_compression_ratio(compression_ratio)

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            self._check_group(self.param_groups[-1])
        except ValueError:
            del self.param_groups[-1]
            raise
        self._sync_counts()
        self._parts = None

    def load_state_dict(self, state_dict):
        for group in state_dict["param_groups"]:
            self._check_group({**self.defaults, **group})
        super().load_state_dict(state_dict)
        # the base class casts a parameter's state to the parameter's type: taken once more as it was saved
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            if i in state_dict["state"]:
                self.state[p] = {k: v.to(p.device, copy=True) if isinstance(v, torch.Tensor) else v
                                 for k, v in state_dict["state"][i].items()}
                self.state[p]["step"] = int(self.state[p]["step"])  # (torch's own optimizers save a tensor)
                for k in ("exp_avg", "exp_avg_sq"):  # (and moments of the parameter's type)
                    if self.state[p][k].dtype in (torch.bfloat16, torch.float16):
                        self.state[p][k] = self.state[p][k].float()
        self._parts = None
        if self.allreduce is not None:
            self.allreduce.reset()  # what it held back are moves of the run that ends here

    def _small(self, p):
        """Whether a parameter's moments begin in 8 bits."""
        return self.state_bits == 8 and p.numel() >= self.min_8bit_size

    def _new_state(self, p):
        state = self.state[p]
        state["step"] = 0
        if self._small(p):
            (state["exp_avg"], state["exp_avg_sq"], state["exp_avg_scales"],
             state["exp_avg_sq_scales"]) = AdamWSet.zeros8(p)
        else:
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)

    def _training(self):
        return [p.requires_grad for group in self.param_groups for p in group["params"]]

    def _make_parts(self):
        """The parts, in the order of the exchanged vector.  That follows from the groups, the types and the optimizer's
        settings, which all ranks share; where a rank's states differ from them (another width was loaded, steps were
        skipped), a part is divided where it stands."""
        alike = {}
        for k, group in enumerate(self.param_groups):
            for p in group["params"]:
                if not p.requires_grad:
                    continue
                self._check(p)
                if "exp_avg" not in self.state[p]:
                    self._new_state(p)
                if p.dtype == torch.float32:
                    self.state[p].pop("master", None)  # (of a type that it had before)
                elif self.master_weights and "master" not in self.state[p]:
                    self.state[p]["master"] = p.detach().to(torch.float32)
                alike.setdefault((str(p.dtype), k, self._small(p)), []).append(p)

        def form(p):
            return "exp_avg_scales" in self.state[p], "master" in self.state[p]

        self._parts = [_Part(self.param_groups[k], list(params))
                       for (_, k, _), those in sorted(alike.items(), key=lambda x: x[0][0])  # a kind's follow one another
                       for _, params in itertools.groupby(those, form)]
        at = 0
        for part in self._parts:  # moments in 8 bits are rounded with noise of each parameter's place
            part.seed = 1 + at if form(part.params[0])[0] else None
            at += sum(p.numel() for p in part.params)
        by_type = {}
        for part in self._parts:
            by_type.setdefault(part.params[0].dtype, []).append(part)
        self._kinds = [_Kind(of_one) for of_one in by_type.values()]
        self._trained = self._training()
        order = [p for kind in self._kinds for p in kind.params]
        if len(order) != len(self._order) or not all(map(operator.is_, order, self._order)):
            self.blob = self.allreduce = None  # another layout: another exchange
        self._order = order

    def _sync_counts(self):
        """The steps' counts where they live on the device, into the state (a saved state holds numbers)."""
        for part in getattr(self, "_parts", None) or ():
            for count, members in part.counts:
                with torch.cuda.stream(self.handle.stream):  # behind the steps, whatever is current here
                    n = int(count)
                for k in members:
                    self.state[part.params[k]]["step"] = n

    def state_dict(self):
        self._sync_counts()
        return super().state_dict()

    def _ready(self):
        """The parts and their sets as the parameters are now; the current stream, or None if nothing is trained."""
        if self._parts is not None and self._trained != self._training():  # parameters were frozen or released
            self._sync_counts()
            self._parts = None
        if self._parts is None:
            self._make_parts()
        return self._make_sets() if self._parts else None

    def _make_sets(self):
        """The parts' sets, made anew where a tensor has moved (a state that was replaced, a model that was)."""
        stream = torch.cuda.current_stream(self._parts[0].params[0].device)
        if self.handle is None or self.handle.device != stream.device:
            with torch.cuda.device(stream.device):
                self.handle = Handle(stream)
            for x in self._parts + self._kinds:
                x.set = None
        if stream.cuda_stream != self.handle.stream.cuda_stream:  # what another stream's memory holds is used on this one
            for t in [count for part in self._parts for count, _ in part.counts] + [self.blob]:
                if t is not None:
                    t.record_stream(stream)
        self.handle.set_stream(stream)
        for kind in self._kinds:
            if kind.set is None:
                kind.set = TensorSet(self.handle, [p.numel() for p in kind.params])
        for part in self._parts:
            lists = part.tensors(self.state)
            if part.set is not None and not part.set.made_of(lists):
                if any(p.dtype != part.dtype for p in part.params):  # other parts then
                    self._sync_counts()
                    self._make_parts()
                    return self._make_sets()
                part.set = None
            if part.set is None:
                part.set = AdamWSet(self.handle, *lists)
                if self.skip_nonfinite and not part.counts:
                    part.count_on(stream.device)
        return stream

    def _clip(self, found):
        """(coefficient or None, non-finite flag or None) of all gradients together."""
        found = [(kind, checked) for kind, _, checked in found if checked is not None]
        if not found or (self.clip_norm is None and not self.skip_nonfinite):
            return None, None
        found = [self.handle.grad_norms(kind.set, checked, self.clip_norm if len(found) == 1 else None)
                 for kind, checked in found]
        if len(found) == 1:
            norms, coef, flag = found[0]
        else:
            norm = torch.linalg.vector_norm(torch.stack([f[0][-1] for f in found]).double())
            coef = None
            if self.clip_norm is not None:
                coef = torch.where(norm > self.clip_norm, self.clip_norm / norm, 1.0).float().reshape(1)
            flag = torch.stack([f[2] for f in found]).amax(0)
        return (coef if self.clip_norm is not None else None), (flag if self.skip_nonfinite else None)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            self._check_group(group)  # before a count or a moment changes
        ranks = self.gaspi_env.get_ranks()
        stream = self._ready()
        if stream is None:
            return loss
        found = [(kind, *kind.gradients()) for kind in self._kinds]
        coef, flag = self._clip(found)
        each = []  # (part, its gradients, the same checked or None)
        for kind, grads, checked in found:
            at = 0
            for part in kind.parts:
                own = grads[at:at + len(part.params)]
                some = any(g is not None for g in own)
                each.append((part, own, part.set.part_of(checked, at) if some else None))
                at += len(own)
        if ranks == 1:
            for part, own, checked in each:
                if checked is not None:
                    self._step_part(part, own, checked, coef, flag)
                    torch.autograd.graph.increment_version([p for p, x in zip(part.params, own) if x is not None])
            return loss
        total = sum(part.set.total for part in self._parts)
        if total > _MOST_EXCHANGED:
            raise ValueError("an exchange takes at most %d elements, not %d" % (_MOST_EXCHANGED, total))
        if total == 0:
            return loss
        if self.blob is None:
            self.gaspi_env.barrier()  # as in ComprexOptimizer.step
            self.blob = torch.empty(total, dtype=torch.float32, device=stream.device)
            self.allreduce = _make_allreduce(self.allreduce_type, self.gaspi_env, total, self.compression_ratio,
                                             self.size_factor)
        at = 0
        for part, own, checked in each:
            moves = self.blob[at:at + part.set.total]
            if any(g is None for g in own):
                moves.zero_()
            if checked is not None:
                self._step_part(part, own, checked, coef, flag, moves)
            at += part.set.total
        # the exchange orders itself with this stream; the setting belongs to the thread, and others change it too
        self.gaspi_env.set_user_stream(stream)
        self.allreduce.apply(self.blob)  # in place, on the device
        self._apply(ranks)
        return loss

    def _apply(self, ranks, decay=True):
        """What came back from the exchange, into the weights."""
        at = 0
        for part in self._parts:
            self.handle.adamw_apply(part.set, self.blob[at:at + part.set.total], part.group["lr"] if decay else 0.0,
                                    part.group["weight_decay"] if decay else 0.0, scale=1.0 / ranks)
            torch.autograd.graph.increment_version(part.params)
            at += part.set.total

    @torch.no_grad()
    def flush(self):
        """Takes the moves that the exchange still holds back into the weights, where and as far as its schedule's flush
        delivers them (the big ring: everywhere; all-to-one: on the chief).  They are in no saved state: every rank
        calls this before it saves one, and before its parameters are frozen or released."""
        stream = self._ready()
        if stream is None or self.allreduce is None:
            return
        self.blob.zero_()
        self.gaspi_env.set_user_stream(stream)
        self.allreduce.flush(self.blob)
        self._apply(self.gaspi_env.get_ranks(), decay=False)

    def _step_part(self, part, grads, checked, coef, flag, moves=None):
        """The step of a part's parameters that have a gradient (`checked`: the same, ready for the set)."""
        group = part.group
        how = dict(betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], coefs=coef, skip=flag,
                   moves=moves, seed=part.seed)
        for count, members in part.counts:
            these = checked
            if len(part.counts) > 1:
                these = [g if k in members else None for k, g in enumerate(grads)]
                if all(g is None for g in these):
                    continue
            self.handle.adamw_step(part.set, these, count, group["lr"], **how)
        if part.counts:
            return
        stepped = [s for s, g in zip(part.states, grads) if g is not None]
        counts = {s["step"] for s in stepped}  # one, unless some parameter went without a gradient before
        for n in sorted(counts, reverse=True):
            these = checked if len(counts) == 1 else [g if s["step"] == n else None for s, g in zip(part.states, grads)]
            self.handle.adamw_step(part.set, these, n + 1, group["lr"], **how)
            for s in stepped:
                if s["step"] == n:
                    s["step"] = n + 1
