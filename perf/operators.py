"""Work that the optimizer's operators are measured on: clipping and packing the gradients of many
tensors into the compressor's flat vector, and the AdamW step with states in 32 bits and in 8.

`own = False` computes an operator in its plain form (elementary torch operations in 32 bits, 64 for
long sums), `own = True` through this package's entry points.  The tensors of a case are views of one
buffer, so that whole buffers can be returned: either back to back (`packed`, as the compressor's flat
vector holds them) or each at a multiple of 256 elements.

States in 8 bits, a scale for each block of 256 elements of one tensor: the first moment as e4m3 codes
of m * 448 / M with M the block's largest |m|; the second as floats of 5 exponent and 3 mantissa bits
without a sign (code 8e + f), code 255 standing for the block's largest value V, and never 0 for a
value above 0.  A block whose M (or V) is below 2^-100 is stored as zeros with scale 0.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 256
TINY = 2.0 ** -100
V_UNIT = 1.875 * 2.0 ** -96   # a second moment of V lies here before its bits are cut to 8
V_BACK = 2.0 ** 96 / 1.875
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BETAS, EPS, DECAY = (0.9, 0.999), 1e-8, 0.1

#: LeNet-5's ten tensors
LENET5 = "150,6,2400,16,48000,120,10080,84,840,10"


def _case(op, total, tensors=1, sizes="", split=7, param="f32", grad="f32", master=False, packed=False,
          flat=False, clip="none", scale=1.0):
    return dict(op=op, total=total, tensors=tensors, sizes=sizes, split=split, param=param, grad=grad,
                master=master, packed=packed, flat=flat, clip=clip, scale=scale)


def listed():
    n50 = 25557032  # ResNet-50: 161 tensors
    return [
        # clip: gradients to the compressor's vector.  A step of the smallest network: all latency.
        dict(_case("clip", 61706, 10, LENET5, clip="each"), name="clip lenet5"),
        # every gradient clipped by its own norm, as the momentum optimizer does before its exchange
        dict(_case("clip", n50, 161, clip="each"), name="clip resnet50"),
        # a language model's bf16 gradients, clipped together, divided by the number of micro-batches
        dict(_case("clip", 100_000_000, 300, grad="bf16", clip="global", scale=0.25), name="clip 100M bf16"),
        # states in 32 bits: smallest network, again latency
        dict(_case("adamw", 61706, 10, LENET5), name="adamw lenet5"),
        # an ordinary fp32 model behind a clip over all gradients
        dict(_case("adamw", n50, 161, clip="global"), name="adamw resnet50"),
        # mixed precision: bf16 weights and gradients, fp32 masters
        dict(_case("adamw", 100_000_000, 300, param="bf16", grad="bf16", master=True, clip="global"),
             name="adamw 100M bf16 master"),
        # behind the compressed exchange over 8 ranks: the gradient is the flat vector, nothing is aligned
        dict(_case("adamw", 1 << 26, 120, packed=True, flat=True, scale=0.125), name="adamw 64M flat"),
        # states in 8 bits: smallest network
        dict(_case("adamw8", 61706, 10, LENET5), name="adamw8 lenet5"),
        # 2^20 half-precision weights with masters, one tensor
        dict(_case("adamw8", 1 << 20, 1, param="f16", grad="f16", master=True), name="adamw8 1M f16 master"),
        # fp32, every gradient with a coefficient of its own
        dict(_case("adamw8", n50, 161, clip="each"), name="adamw8 resnet50"),
        # everything small: bf16 weights without masters
        dict(_case("adamw8", 100_000_000, 300, param="bf16", grad="bf16", clip="global"),
             name="adamw8 100M bf16"),
    ]


def draw(rng):
    op = rng.choice(["clip", "adamw", "adamw8"])
    total = int(round(math.exp(rng.uniform(math.log(50), math.log(1e8)))))
    tensors = rng.randint(1, min(300, max(1, total // 4)))
    param = rng.choice(["f32", "bf16", "f16"])
    packed = op != "adamw8" and rng.random() < 0.5
    return _case(op, total, tensors, split=rng.randint(0, 1 << 30), param=param,
                 grad=rng.choice(["f32", param] if op != "clip" else list(TYPES)),
                 master=param != "f32" and rng.random() < 0.5, packed=packed,
                 flat=packed and op == "adamw" and rng.random() < 0.5,
                 clip=rng.choice(["each", "global"] if op == "clip" else ["none", "each", "global"]),
                 scale=rng.choice([1.0, 0.125, 1.0 / 3.0]))


def _sizes(case):
    if case["sizes"]:
        return [int(s) for s in case["sizes"].split(",")]
    total, k = case["total"], case["tensors"]
    w = np.random.Generator(np.random.PCG64(case["split"])).random(k) ** 3 + 1e-4
    sizes = np.maximum(1, np.floor(w / w.sum() * total)).astype(np.int64)
    while sizes.sum() > total:
        sizes[np.argmax(sizes)] -= 1
    sizes[np.argmax(sizes)] += total - sizes.sum()
    return [int(s) for s in sizes]


def _layout(case):
    """Sizes, first elements and the length of the buffer that holds all tensors."""
    sizes = _sizes(case)
    room = [n if case["packed"] else -(-n // BLOCK) * BLOCK for n in sizes]
    starts = [0] + [int(x) for x in np.cumsum(room)]
    return sizes, room, starts[:-1], starts[-1]


# ---- the 8-bit states in 32-bit torch operations -----------------------------------------

def _m_to_8(m):
    m = m.view(-1, BLOCK)
    top = m.abs().amax(1)
    kept = top >= TINY
    inverse = torch.where(kept, torch.full_like(top, 448.0) / top, 0.0)
    return (m * inverse[:, None]).to(torch.float8_e4m3fn).view(-1), torch.where(kept, top * (1.0 / 448.0), 0.0)


def _v_to_8(v):
    v = v.view(-1, BLOCK)
    top = v.amax(1)
    kept = top >= TINY
    inverse = torch.where(kept, torch.ones_like(top) / top, 0.0)
    bits = (v * inverse[:, None] * V_UNIT).view(torch.int32)
    code = ((bits + 0x80000) >> 20).clamp(max=255)
    code = torch.where(kept[:, None], torch.maximum(code, (v > 0).to(torch.int32)), 0)
    return code.to(torch.uint8).view(-1), torch.where(kept, top, 0.0)


def _m_of_8(code, scale):
    return (code.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _v_of_8(code, scale):
    return ((code.to(torch.int32) << 20).view(torch.float32).view(-1, BLOCK) * V_BACK * scale[:, None]).view(-1)


# ---- inputs ------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    sizes, room, starts, length = _layout(case)
    gen = torch.Generator(device=dev).manual_seed(seed)
    rooms = torch.tensor(room, device=dev)
    # gradients of different layers differ by orders of magnitude
    layer = torch.exp(torch.empty(len(sizes), device=dev).uniform_(math.log(1e-5), math.log(1e-1), generator=gen))
    size = layer.repeat_interleave(rooms, output_size=length)
    if not case["packed"]:  # nothing between the tensors
        behind = torch.arange(length, device=dev) - torch.tensor(starts, device=dev).repeat_interleave(rooms, output_size=length)
        size.masked_fill_(behind >= torch.tensor(sizes, device=dev).repeat_interleave(rooms, output_size=length), 0.0)
        del behind

    def normal():
        return torch.empty(length, device=dev).normal_(generator=gen)

    # some elements got no gradient this time, some never had one
    g = normal() * size * (torch.empty(length, device=dev).uniform_(generator=gen) >= 0.05)
    s = dict(case=dict(case), sizes=sizes, starts=starts, step=999,
             lr=10.0 ** float(torch.empty(1, device=dev).uniform_(-4, -2.5, generator=gen)))
    s["lengths"] = torch.tensor(sizes, device=dev)
    s["rooms"] = rooms
    s["index"] = None if case["packed"] else (
        torch.arange(case["total"], device=dev)
        + torch.tensor(np.array(starts) - np.concatenate([[0], np.cumsum(sizes)[:-1]]), device=dev)
        .repeat_interleave(s["lengths"], output_size=case["total"]))
    s["scale"] = case["scale"]
    if case["grad"] == "f16":  # under a loss scale
        g = g * 256.0
        s["scale"] /= 256.0
    s["g"] = g.to(TYPES[case["grad"]])
    del g
    if case["op"] == "clip":
        s["max_norm"] = 5.0 if case["clip"] == "each" else 1.0
    else:
        s["coefs"] = None
        if case["clip"] != "none":
            k = len(sizes) if case["clip"] == "each" else 1
            s["coefs"] = torch.empty(k, device=dev).uniform_(0.2, 1.0, generator=gen)
        w = normal() * 0.02 * (size > 0)
        touched = torch.empty(length, device=dev).uniform_(generator=gen) >= 0.02
        m = normal() * size * 0.3 * touched
        v = size.square() * (0.25 + normal().square()) * touched
        s["p"] = w.to(TYPES[case["param"]])
        s["w"] = w if case["master"] else None
        if case["op"] == "adamw":
            s["m"], s["v"] = m, v
        else:
            s["m"], s["ms"] = _m_to_8(m)
            s["v"], s["vs"] = _v_to_8(v)
    if own:
        _bind(s)
    return s


def _views(s, name, of=1):
    """The tensors' parts of a buffer; `of`: elements that one of the buffer's stands for."""
    t = s[name]
    return None if t is None else [t[a // of:a // of + -(-n // of)] for a, n in zip(s["starts"], s["sizes"])]


def _bind(s):
    """What a program that calls the framework keeps: the handle, its tensors, their set."""
    from comprex_amd.device import AdamWSet, Handle, TensorSet
    s["h"] = Handle()
    s["grads"] = s["g"] if s["case"]["flat"] else _views(s, "g")
    if s["case"]["op"] == "clip":
        s["set"] = TensorSet(s["h"], s["sizes"])
        return
    small = s["case"]["op"] == "adamw8"
    s["set"] = AdamWSet(s["h"], _views(s, "p"), _views(s, "m"), _views(s, "v"), masters=_views(s, "w"),
                        exp_avg_scales=_views(s, "ms", BLOCK) if small else None,
                        exp_avg_sq_scales=_views(s, "vs", BLOCK) if small else None)


# ---- one pass ----------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if case["op"] == "clip":
        return _run_clip(s)
    s["step"] += 1
    if own:
        s["h"].adamw_step(s["set"], s["grads"], s["step"], s["lr"], BETAS, EPS, DECAY, coefs=s["coefs"],
                          scale=s["scale"])
        values = s["h"].adamw_states(s["set"], torch.bfloat16) if case["op"] == "adamw8" else None
    elif case["op"] == "adamw":
        _adamw(s, s["m"], s["v"])
    else:
        m, v = _m_of_8(s["m"], s["ms"]), _v_of_8(s["v"], s["vs"])
        _adamw(s, m, v)
        for name, (code, scale) in (("m", _m_to_8(m)), ("v", _v_to_8(v))):
            s[name].copy_(code)
            s[name + "s"].copy_(scale)
        values = [_dense(s, x).bfloat16() for x in (_m_of_8(s["m"], s["ms"]), _v_of_8(s["v"], s["vs"]))]
    out = {"p": s["p"]}
    if s["w"] is not None:
        out["w"] = s["w"]
    if case["op"] == "adamw":
        return dict(out, m=s["m"], v=s["v"])
    return dict(out, ms=s["ms"], vs=s["vs"], m=values[0], v=values[1])


def _dense(s, x):
    """The tensors of a buffer back to back."""
    return x if s["index"] is None else x[s["index"]]


def _run_clip(s):
    case = s["case"]
    each = case["clip"] == "each"
    if own:
        norms, coefs, nonfinite = s["h"].grad_norms(s["set"], s["grads"], s["max_norm"], each=each, scale=s["scale"])
        flat = s["h"].pack(s["set"], s["grads"], coefs=coefs, scale=s["scale"])
        return {"norms": norms, "coefs": coefs, "nonfinite": nonfinite, "flat": flat}
    flat = _dense(s, s["g"]).float()
    squares = torch.segment_reduce(flat.double().square(), "sum", lengths=s["lengths"])
    squares = torch.cat([squares, squares.sum(0, keepdim=True)])
    norms = squares.sqrt() * s["scale"]
    which = norms[:-1] if each else norms[-1:]
    coefs = torch.where(which > s["max_norm"], s["max_norm"] / which, 1.0).float()
    factor = coefs * s["scale"]
    if each:
        factor = factor.repeat_interleave(s["lengths"], output_size=flat.numel())
    return {"norms": norms.float(), "coefs": coefs, "nonfinite": (~torch.isfinite(norms[-1:])).int(),
            "flat": flat * factor}


def _adamw(s, m, v):
    """The weights and, in place, the moments in 32 bits."""
    case, (b1, b2) = s["case"], BETAS
    g = s["g"].float()
    if s["coefs"] is None:
        g = g * s["scale"]
    else:
        factor = s["coefs"] * s["scale"]
        g = g * (factor if factor.numel() == 1 else factor.repeat_interleave(s["rooms"], output_size=g.numel()))
    m.mul_(b1).add_(g * (1 - b1))
    v.mul_(b2).add_(g * g * (1 - b2))
    w = s["p"].float() if s["w"] is None else s["w"]
    below = v.sqrt() * (1.0 / math.sqrt(1 - b2 ** s["step"])) + EPS
    new = w * (1 - s["lr"] * DECAY) - m / below * (s["lr"] / (1 - b1 ** s["step"]))
    if s["w"] is not None:
        s["w"].copy_(new)
    s["p"].copy_(new)


# ---- what it cannot do without -----------------------------------------------------------

def work(case):
    n = case["total"]
    g = 2 if case["grad"] != "f32" else 4
    if case["op"] == "clip":
        return {"bytes": n * (g + 4), "flops": 3 * n}
    p = 2 if case["param"] != "f32" else 4
    weights = p + 8 if case["master"] else 2 * p
    if case["op"] == "adamw":
        return {"bytes": n * (weights + g + 16), "flops": 15 * n}
    blocks = sum(-(-k // BLOCK) for k in _sizes(case))
    return {"bytes": n * (weights + g + 4 + 4) + blocks * 16, "flops": 25 * n}  # + 4: the states' values in bf16


# ---- the definition in 64 bits -----------------------------------------------------------

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    spans = [slice(a, a + n) for a, n in zip(s["starts"], s["sizes"])]
    g = s["g"].double()
    if case["op"] == "clip":
        norms = [s["scale"] * math.sqrt(float((g[p] * g[p]).sum())) for p in spans]
        total = math.sqrt(sum(x * x for x in norms))
        coefs = [s["max_norm"] / x if x > s["max_norm"] else 1.0 for x in (norms if case["clip"] == "each" else [total])]
        flat = torch.cat([g[p] * (coefs[k if len(coefs) > 1 else 0] * s["scale"]) for k, p in enumerate(spans)])
        f64 = dict(dtype=torch.float64, device=g.device)
        return {"norms": torch.tensor(norms + [total], **f64), "coefs": torch.tensor(coefs, **f64), "nonfinite": None,
                "flat": flat}
    g *= s["scale"]
    if s["coefs"] is not None:
        for k, p in enumerate(spans):
            g[p] *= float(s["coefs"][k if case["clip"] == "each" else 0])
    t, (b1, b2) = s["step"] + 1, BETAS
    if case["op"] == "adamw":
        m, v = s["m"].double(), s["v"].double()
    else:
        e4m3, e5m3 = _tables(g.device)
        blocks = torch.arange(g.numel(), device=g.device) // BLOCK
        m = e4m3[s["m"].view(torch.uint8).long()] * s["ms"].double()[blocks]
        v = e5m3[s["v"].long()] * s["vs"].double()[blocks]
    m = m + (1 - b1) * (g - m)
    v = v + (1 - b2) * (g ** 2 - v)
    w = (s["p"] if s["w"] is None else s["w"]).double()
    w = w - s["lr"] * (DECAY * w + (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + EPS))
    out = {"p": w}
    if s["w"] is not None:
        out["w"] = w
    if case["op"] == "adamw":
        return dict(out, m=m, v=v)
    tops = [x.abs().view(-1, BLOCK).max(1).values for x in (m, v)]
    tops = [torch.where(x < TINY, 0.0, x) for x in tops]
    got = []
    for x, top, values in ((m, tops[0] / 448.0, e4m3[:127]), (v, tops[1], e5m3)):
        unit = (x.abs() / top[blocks]).nan_to_num(0.0, 0.0)
        k = torch.bucketize(unit, (values[1:] + values[:-1]) / 2)
        if x is v:
            k = torch.maximum(k, (unit > 0).long())
        got.append(torch.cat([(values[k] * top[blocks] * x.sign())[p] for p in spans]))
    return dict(out, ms=tops[0] / 448.0, vs=tops[1], m=got[0], v=got[1])


def _tables(device):
    """What the codes stand for: e4m3, and 5 exponent and 3 mantissa bits with 255 as 1."""
    code = torch.arange(256, device=device)

    def floats(c, bias):
        e, f = (c >> 3).double(), (c & 7).double()
        return torch.where(e > 0, (1 + f / 8) * 2.0 ** (e - bias), f / 8 * 2.0 ** (1.0 - bias))

    signed = floats(code & 127, 7) * torch.where(code > 127, -1.0, 1.0)
    signed[127] = signed[255] = math.nan
    unsigned = floats(code, 0)
    return signed, unsigned / unsigned[255]
