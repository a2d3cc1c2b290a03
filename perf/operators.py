"""What the decode operators are measured on: norm and rotation of queries and keys, the 8-bit key/value
cache (filling it, a decode step through it, attention over it) and products with 4-bit weights.

`own` false: the operators in elementary torch operations; `own` true: the framework's calls.  A case is a
dict of plain values; `prepare` makes what a program has in hand before the call, `run` is one pass.
"""
import ctypes
import importlib
import math

import numpy as np
import torch

own = False

BLOCK = 64          # tokens of one head that share a scale in the cache
THETA = 10000.0
EPS = 1e-5
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # queries and keys of a whole prompt batch, grouped heads: pure memory traffic
        {"name": "norm-rope prompt", "kind": "norm_rope", "dtype": "f16", "batch": 8, "seq": 2048, "heads": 32,
         "kv_heads": 8, "dim": 128, "start": 0, "recorded": False},
        # the same for one new token of each of eight sequences: the smallest call, all latency
        {"name": "norm-rope one token", "kind": "norm_rope", "dtype": "bf16", "batch": 8, "seq": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "start": 2047, "recorded": True},
        # a prompt's second part in full precision: odd length, narrow heads
        {"name": "norm-rope odd f32", "kind": "norm_rope", "dtype": "f32", "batch": 3, "seq": 511, "heads": 12,
         "kv_heads": 4, "dim": 64, "start": 17, "recorded": False},
        # four prompts of different lengths put into an empty cache as one padded batch, and read back
        {"name": "cache fill ragged", "kind": "fill", "dtype": "bf16", "batch": 4, "seq": 2048, "kv_heads": 8,
         "dim": 128, "ragged": True},
        # one decode step of eight sequences: roll back the last draft, norm, rotate, append, attend
        {"name": "decode step", "kind": "step", "dtype": "f16", "batch": 8, "length": 2048, "heads": 32, "kv_heads": 8,
         "dim": 128, "new": 1, "ragged": True, "recorded": True},
        # one token against one very long context
        {"name": "attention long", "kind": "attention", "dtype": "bf16", "batch": 1, "length": 131071, "heads": 32,
         "kv_heads": 8, "dim": 128, "new": 1, "ragged": False, "recorded": True},
        # one token of each of 32 sequences of very different lengths
        {"name": "attention batch", "kind": "attention", "dtype": "f16", "batch": 32, "length": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "new": 1, "ragged": True, "recorded": False},
        # five drafted tokens checked at once in full precision, every head with keys of its own
        {"name": "attention drafts f32", "kind": "attention", "dtype": "f32", "batch": 4, "length": 3001, "heads": 16,
         "kv_heads": 16, "dim": 64, "new": 5, "ragged": True, "recorded": False},
        # one row through a gate projection
        {"name": "q4 one row", "kind": "q4", "dtype": "f16", "rows": 1, "n": 11008, "k": 4096, "group": 128,
         "recorded": True},
        # a small batch through a down projection
        {"name": "q4 seven rows", "kind": "q4", "dtype": "bf16", "rows": 7, "n": 4096, "k": 11008, "group": 64,
         "recorded": False},
        # odd sizes in full precision: a last group that is not full, rows that do not fill a tile
        {"name": "q4 odd f32", "kind": "q4", "dtype": "f32", "rows": 3, "n": 1003, "k": 4331, "group": 32,
         "recorded": False},
        # a prompt through the same 4-bit weights
        {"name": "q4 prompt", "kind": "q4", "dtype": "f16", "rows": 500, "n": 11008, "k": 4096, "group": 128,
         "recorded": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm_rope", "fill", "step", "attention", "attention", "q4", "q4"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    recorded = rng.random() < 0.5
    if kind == "q4":
        return {"kind": kind, "dtype": dtype, "rows": _log(rng, 1, 500), "n": _log(rng, 300, 11008),
                "k": _log(rng, 300, 11008 if dtype != "f32" else 4096), "group": rng.choice([32, 64, 128]),
                "recorded": recorded}
    dim = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 5, 8])
    heads = kv * rng.choice([1, 2, 4, 7])
    batch = _log(rng, 1, 8)
    if kind == "norm_rope":
        return {"kind": kind, "dtype": dtype, "batch": batch, "seq": _log(rng, 1, 1500), "heads": heads, "kv_heads": kv,
                "dim": dim, "start": rng.randrange(0, 2000), "recorded": recorded}
    if kind == "fill":
        return {"kind": kind, "dtype": dtype, "batch": batch, "seq": _log(rng, 1, 2000), "kv_heads": kv, "dim": dim,
                "ragged": rng.random() < 0.5}
    new = rng.choice([1, 1, 1, 2, 4, 6])
    if kind == "step":
        return {"kind": kind, "dtype": rng.choice(["f16", "bf16"]), "batch": batch, "length": _log(rng, 40, 6000),
                "heads": heads, "kv_heads": kv, "dim": dim, "new": new, "ragged": rng.random() < 0.5,
                "recorded": recorded}
    return {"kind": kind, "dtype": dtype, "batch": batch, "length": _log(rng, 20, 8000), "heads": heads,
            "kv_heads": kv, "dim": dim, "new": new, "ragged": rng.random() < 0.5, "recorded": recorded}


def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["kind"] == "q4":
        groups = -(-c["k"] // c["group"])
        # 4-bit codes and 16- or 32-bit scales, the rows in and out
        return {"bytes": c["n"] * c["k"] / 2 + c["n"] * groups * e + c["rows"] * (c["k"] + c["n"]) * e,
                "flops": 2.0 * c["rows"] * c["n"] * c["k"]}
    if c["kind"] == "norm_rope":
        rows = c["batch"] * c["seq"] * (c["heads"] + c["kv_heads"])
        return {"bytes": 2 * rows * c["dim"] * e + c["seq"] * c["dim"] * e + 2 * c["dim"] * e,
                "flops": 8.0 * rows * c["dim"]}
    if c["kind"] == "fill":
        tokens = sum(_lengths(c["batch"], c["seq"], c["ragged"])) * c["kv_heads"]
        longest = max(_lengths(c["batch"], c["seq"], c["ragged"])) * c["batch"] * c["kv_heads"]
        # keys and values in, codes out; the codes read back and the values they stand for written
        return {"bytes": 2 * tokens * c["dim"] * (e + 2) + 2 * longest * c["dim"] * e, "flops": 6.0 * tokens * c["dim"]}
    keys = sum(_lengths(c["batch"], c["length"], c["ragged"])) * c["kv_heads"]
    rows = c["batch"] * c["new"] * c["heads"]
    moved = 2 * keys * c["dim"] + 8 * keys / BLOCK + 2 * rows * c["dim"] * e
    flops = 4.0 * keys * c["heads"] / c["kv_heads"] * c["new"] * c["dim"]
    if c["kind"] == "step":
        moved += c["batch"] * c["new"] * c["kv_heads"] * c["dim"] * (2 * e + 2)
    return {"bytes": moved, "flops": flops}


def _lengths(batch, longest, ragged):
    """Ragged: spread from an eighth of the longest to all of it, in no order; a property of the case, not of its seed."""
    if not ragged:
        return [longest] * batch
    got = [max(1, longest - (i * 5 % batch) * (longest - longest // 8) // batch) for i in range(batch)]
    return got


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dt)

    c, kind = case, case["kind"]
    if kind == "q4":
        # a projection as it was initialised: N(0, 0.02), with a few channels that stand out
        w = torch.randn(c["n"], c["k"], generator=g, device="cuda") * 0.02
        w *= 1 + 4 * (torch.rand(c["k"], generator=g, device="cuda") < 0.01)
        return {"x": normal(c["rows"], c["k"]), "w": w.to(dt)}
    b, d = c["batch"], c["dim"]
    s = {}
    lengths = _lengths(b, c.get("length", c.get("seq")), c.get("ragged", False))
    t = c["seq"] if kind in ("norm_rope", "fill") else c["new"]
    if kind != "norm_rope":
        # some key channels are large, as they are in trained models
        big = 1 + 5 * (torch.rand(d, generator=g, device="cuda") < 0.03)
        total = t if kind == "fill" else c["length"]
        s["keys"] = (torch.randn(b, total, c["kv_heads"], d, generator=g, device="cuda") * big).to(dt)
        s["values"] = normal(b, total, c["kv_heads"], d)
        s["lengths"] = lengths
    if kind == "fill":
        return s
    s["q"] = normal(b, t, c["heads"], d)                     # projections as they come: heads side by side
    if kind in ("norm_rope", "step"):
        s["k"] = normal(b, t, c["kv_heads"], d, std=2.0)
        if kind == "step":
            s["v"] = normal(b, t, c["kv_heads"], d)
        s["wq"], s["wk"] = normal(d, std=0.1, mean=1.0), normal(d, std=0.1, mean=1.0)
        far = c["start"] + t if kind == "norm_rope" else c["length"] + t
        angle = torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * THETA ** (
            -torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        s["cos"], s["sin"] = torch.cos(angle).to(dt), torch.sin(angle).to(dt)
    return s


# ---------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------
def _norm_rope(x, w, cos, sin):
    """x [batch, heads, seq, dim]; cos, sin broadcast to [batch, 1, seq, dim / 2]: each head normed, then rotated."""
    x = x.float()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    lo, hi = y[..., : y.shape[-1] // 2], y[..., y.shape[-1] // 2:]
    c, s = cos.float(), sin.float()
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


def _blocks(x, lengths):
    """x [batch, kv_heads, tokens, dim] as blocks of tokens [batch, kv_heads, n, BLOCK, dim], zero behind each length."""
    b, h, t, d = x.shape
    n = -(-t // BLOCK)
    x = torch.where(torch.arange(t, device=x.device)[None, None, :, None] < lengths[:, None, None, None], x, torch.zeros_like(x))
    return torch.cat([x, x.new_zeros(b, h, n * BLOCK - t, d)], 2).reshape(b, h, n, BLOCK, d)


def _to_8_bits(x, lengths):
    """Codes in [-127, 127] and a scale for each block of tokens and head: code = round(127 x / max|x|)."""
    x = _blocks(x, lengths)
    top = x.abs().amax((-1, -2), keepdim=True)
    # 64 bits: values next to a border between two codes
    codes = torch.round(127.0 * x.double() / torch.clamp(top.double(), min=2.0 ** -100)).to(torch.int8)
    return codes, torch.clamp(top.float(), min=2.0 ** -100) / 127.0


def _values(codes, scales):
    x = codes.float() * scales
    b, h, n, t, d = x.shape
    return x.reshape(b, h, n * t, d)


def _attend(q, k, v, lengths, scale):
    """q [batch, heads, new, dim] at the last positions of each sequence, k and v [batch, kv_heads, tokens, dim]."""
    b, heads, new, d = q.shape
    kv, tokens = k.shape[1], k.shape[2]
    q = q.to(k.dtype).reshape(b, kv, heads // kv * new, d)
    scores = (q @ k.transpose(-1, -2) * scale).reshape(b, kv, heads // kv, new, tokens)
    last = lengths[:, None] - new + torch.arange(new, device=q.device)
    seen = (torch.arange(tokens, device=q.device) <= last[:, :, None])[:, None, None]
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    return (p.reshape(b, kv, -1, tokens) @ v).reshape(b, heads, new, d)


def _put(old, fresh, lengths):
    """old [batch, kv_heads, tokens, dim] with `fresh` [batch, kv_heads, new, dim] written behind each length."""
    new = fresh.shape[2]
    x = torch.cat([old, old.new_zeros(*old.shape[:2], new, old.shape[3])], 2)
    at = (lengths[:, None] + torch.arange(new, device=x.device))[:, None, :, None]
    return x.scatter(2, at.expand(-1, x.shape[1], -1, x.shape[3]), fresh)


def _to_4_bits(w, group):
    """Codes in [-7, 7] and a scale of w's type for each row and group of columns: code = round(w / scale)."""
    n, k = w.shape
    x = torch.cat([w, w.new_zeros(n, -k % group)], 1).reshape(n, -1, group)
    scales = (x.float().abs().amax(-1, keepdim=True) / 7.0).to(w.dtype)
    codes = torch.round(x.double() / torch.where(scales > 0, scales, torch.ones_like(scales)).double())
    return codes.clamp(-8, 7).to(torch.int8), scales


def _weight(codes, scales, k):
    return (codes.float() * scales.float()).reshape(codes.shape[0], -1)[:, :k]


# ---------------------------------------------------------------------------------------------------
# the framework's side: its tensors over torch's data
# ---------------------------------------------------------------------------------------------------
_loaded = None


def _framework():
    global _loaded
    if _loaded is None:
        wgf = importlib.import_module("wgpu-kernal-fusion_b200")
        dev = wgf.Device(0)
        dev.set_timing(False)
        _loaded = wgf, dev
    return _loaded


class _Array:
    """Device memory as torch.as_tensor takes it; holds on to the owner."""

    def __init__(self, ptr, shape, kind, strides=None, owner=None):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": shape, "strides": strides, "typestr": kind,
                                         "version": 2}


def _give(x):
    """A framework tensor with the values of a torch one (a copy on the device)."""
    wgf, dev = _framework()
    x = x.contiguous()
    lib, buf, ptr, size = wgf.lib(), ctypes.c_void_p(), ctypes.c_void_p(), x.numel() * x.element_size()
    wgf.check(lib.wgf_buffer_alloc(dev.h, ctypes.c_uint64(size), ctypes.c_int32(0), ctypes.byref(buf)))
    wgf.check(lib.wgf_buffer_device_ptr(buf, ctypes.byref(ptr), None))
    dev.sync()
    torch.as_tensor(_Array(ptr.value, (size,), "|u1"), device="cuda").copy_(x.reshape(-1).view(torch.uint8))
    torch.cuda.synchronize()
    desc = wgf.TensorDesc(buf=buf, dtype={torch.float32: wgf.F32, torch.float16: wgf.F16, torch.bfloat16: wgf.BF16}[x.dtype],
                          rank=x.dim(), offset=0)
    for i in range(x.dim()):
        desc.shape[i], desc.stride[i] = x.shape[i], x.stride(i)
    out = ctypes.c_void_p()
    wgf.check(lib.wgf_tensor_from_desc(dev.h, ctypes.byref(desc), ctypes.byref(out)))
    wgf.check(lib.wgf_buffer_release(buf))
    return wgf.Tensor(dev, out)


def _take(t):
    """A framework tensor's memory as a torch tensor; nothing is copied and nothing waits."""
    wgf, _ = _framework()
    d, ptr = t.desc(), ctypes.c_void_p()
    buf = ctypes.c_void_p(d.buf)
    wgf.check(wgf.lib().wgf_buffer_device_ptr(buf, ctypes.byref(ptr), None))
    wgf.lib().wgf_buffer_release(buf)
    e = 4 if d.dtype == wgf.F32 else 2
    shape = tuple(d.shape[: d.rank])
    a = _Array(ptr.value + d.offset * e, shape, {wgf.F32: "<f4", wgf.F16: "<f2", wgf.BF16: "<i2"}[d.dtype],
               tuple(s * e for s in d.stride[: d.rank]), t)
    x = torch.as_tensor(a, device="cuda")
    return x.view(torch.bfloat16) if d.dtype == wgf.BF16 else x


# ---------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------
def prepare(case, seed):
    s, c = _inputs(case, seed), case
    s["case"] = c
    if "lengths" in s:
        s["counts"] = s["lengths"] if c["ragged"] else None
        s["at"] = torch.tensor(s["lengths"], device="cuda")
    if not own:
        if c["kind"] == "q4":
            s["w"] = _to_4_bits(s["w"], c["group"])
        elif c["kind"] == "attention":
            k, v = s.pop("keys").transpose(1, 2), s.pop("values").transpose(1, 2)
            s["k8"], s["v8"] = _to_8_bits(k, s["at"]), _to_8_bits(v, s["at"])
        return s
    wgf, dev = _framework()
    s = {n: _give(x) if isinstance(x, torch.Tensor) and n != "at" else x for n, x in s.items()}
    if c["kind"] == "q4":
        s["w"] = s["w"].quantize_q4(c["group"])
    elif c["kind"] != "norm_rope":
        room = c["seq"] if c["kind"] == "fill" else c["length"] + c["new"]
        s["cache"] = dev.kv_cache(c["batch"], c["kv_heads"], c["dim"], room, s["values"].dtype)
        if c["kind"] != "fill":
            s["cache"].append(s.pop("keys").transpose(1, 2), s.pop("values").transpose(1, 2), s["counts"])
    dev.sync()
    if c.get("recorded"):
        _pass(s)                       # everything that a first call sets up happens outside the recording
        if c["kind"] == "step":
            s["cache"].truncate(s["lengths"])
        with dev.record() as s["schedule"]:
            s["out"] = _pass(s, rollback=False)
        s["taken"] = [_take(t) for t in s["out"]]
        dev.sync()
    return s


def _pass(s, rollback=True):
    """The framework's calls of one pass."""
    c = s["case"]
    if c["kind"] == "q4":
        return [s["x"].mat_mul_q4(s["w"]).materialize()]
    if c["kind"] == "norm_rope":
        q, k = s["q"].transpose(1, 2).qk_norm_rope(s["k"].transpose(1, 2), s["wq"], s["wk"], s["cos"], s["sin"], EPS, c["start"])
        return [q.materialize(), k.materialize()]
    cache = s["cache"]
    if c["kind"] == "fill":
        cache.truncate([0] * c["batch"])
        cache.append(s["keys"].transpose(1, 2), s["values"].transpose(1, 2), s["counts"])
        return list(cache.read())
    q = s["q"].transpose(1, 2)
    if c["kind"] == "step":
        if rollback:
            cache.truncate(s["lengths"])
        q = cache.append_qk(q, s["k"].transpose(1, 2), s["v"].transpose(1, 2), s["wq"], s["wk"], s["cos"], s["sin"], EPS)
        return [cache.attention(q), q]
    return [cache.attention(q)]


def run(s):
    c = s["case"]
    if own:
        if not c.get("recorded"):
            return [_take(t) for t in _pass(s)]
        if c["kind"] == "step":
            s["cache"].truncate(s["lengths"])
        s["schedule"].launch()
        return s["taken"]
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "q4":
        return [(s["x"].float() @ _weight(*s["w"], c["k"]).T).to(dt)]
    if c["kind"] == "norm_rope":
        cos, sin = (s[n][c["start"]: c["start"] + c["seq"]] for n in ("cos", "sin"))
        return [_norm_rope(s[x].transpose(1, 2), s[w], cos, sin).to(dt) for x, w in (("q", "wq"), ("k", "wk"))]
    if c["kind"] == "fill":
        longest = max(s["lengths"])
        return [_values(*_to_8_bits(s[n].transpose(1, 2), s["at"]))[:, :, :longest].to(dt) for n in ("keys", "values")]
    q, at = s["q"].transpose(1, 2), s["at"]
    if c["kind"] == "step":
        where = at[:, None] + torch.arange(c["new"], device="cuda")
        cos, sin = s["cos"][where][:, None], s["sin"][where][:, None]
        q = _norm_rope(q, s["wq"], cos, sin).to(dt)                # what goes into the attention comes back too
        k = _put(s["keys"].transpose(1, 2), _norm_rope(s["k"].transpose(1, 2), s["wk"], cos, sin).to(dt), at)
        v = _put(s["values"].transpose(1, 2), s["v"].transpose(1, 2), at)
        at = at + c["new"]
        s8 = _to_8_bits(k, at), _to_8_bits(v, at)
    else:
        s8 = s["k8"], s["v8"]
    out = _attend(q, _values(*s8[0]), _values(*s8[1]), at, c["dim"] ** -0.5).to(dt)
    return [out, q] if c["kind"] == "step" else [out]


# ---------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    s, c = _inputs(case, seed), case
    wide = {n: x.double() if isinstance(x, torch.Tensor) else x for n, x in s.items()}
    if c["kind"] == "q4":
        n, k, g = c["n"], c["k"], c["group"]
        w = torch.nn.functional.pad(wide["w"], (0, -k % g)).view(n, -1, g)
        # the scale is a number of the weights' type, so its rounding is part of the definition
        step = (w.abs().amax(2) / 7).float().to(s["w"].dtype).double()[:, :, None]
        w = torch.where(step > 0, torch.round(w / step).clamp(-8, 7) * step, 0 * w).reshape(n, -1)[:, :k]
        return [torch.einsum("mk,nk->mn", wide["x"], w)]
    d, half = c["dim"], c["dim"] // 2

    def rotate(x, w, first):
        """[batch, seq, heads, dim] as complex numbers turned by the angle of their position."""
        x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / d + EPS) * w
        at = first[:, None] + torch.arange(x.shape[1], device="cuda")
        turn = torch.complex(wide["cos"][at], wide["sin"][at])[:, :, None]
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1).transpose(1, 2)

    if c["kind"] == "norm_rope":
        first = torch.full((c["batch"],), c["start"], device="cuda")
        return [rotate(wide["q"], wide["wq"], first), rotate(wide["k"], wide["wk"], first)]

    lengths = np.array(s["lengths"])
    dt = DTYPES[c["dtype"]]

    def stands_for(x, n):
        """x [tokens, kv_heads, dim] of one sequence of n tokens: the values of its codes."""
        x = x[:n].double()
        t = -(-n // BLOCK) * BLOCK
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, t - n)).view(-1, BLOCK, x.shape[1], d)
        step = (x.abs().amax((1, 3), keepdim=True) / 127).clamp(min=2.0 ** -100 / 127)
        return (torch.round(x / step) * step).reshape(t, -1, d)[:n]

    if c["kind"] == "fill":
        out = []
        for name in ("keys", "values"):
            y = torch.zeros(c["batch"], c["kv_heads"], int(lengths.max()), d, device="cuda", dtype=torch.float64)
            for b, n in enumerate(lengths):
                y[b, :, :n] = stands_for(s[name][b], int(n)).transpose(0, 1)
            out.append(y)
        return out
    q, new = wide["q"].transpose(1, 2), c["new"]
    out = torch.zeros(c["batch"], c["heads"], new, d, device="cuda", dtype=torch.float64)
    if c["kind"] == "step":
        first = torch.tensor(lengths, device="cuda")
        # what is rounded to the type between two operators is rounded here too
        q = rotate(wide["q"], wide["wq"], first)
        turned = q
        q = q.to(dt).double()
        k_new = rotate(wide["k"], wide["wk"], first).to(dt).transpose(1, 2)
    for b, n in enumerate(lengths):
        n, keys, values = int(n), s["keys"][b], s["values"][b]
        if c["kind"] == "step":
            keys, values = torch.cat([keys[:n], k_new[b]]), torch.cat([values[:n], s["v"][b]])
            n += new
        k, v = (torch.repeat_interleave(stands_for(x, n), c["heads"] // c["kv_heads"], 1) for x in (keys, values))
        e = torch.einsum("htd,nhd->htn", q[b], k) / math.sqrt(d)
        later = torch.arange(n, device="cuda")[None, :] > (n - new + torch.arange(new, device="cuda"))[:, None]
        out[b] = torch.einsum("htn,nhd->htd", torch.softmax(e.masked_fill(later, -math.inf), -1).nan_to_num(0.0), v)
    return [out, turned] if c["kind"] == "step" else [out]
