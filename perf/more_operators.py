"""Performance cases of rotary positions and an 8-bit KV cache with block scales on one MI355X.

What a layer does around its attention when the paged cache is held in 8 bits with one scale
for each block of tokens and kv head, each operator reached as an engine reaches it:

* ``rotary``: queries and keys rotated by their positions (``apply_rotary``);
* ``append``: a window of new keys and values per sequence written into the paged cache, keys
  (and queries) rotated on the way (``append_kv``); pools of the rows' type, fp8 with a scale
  per vector, fp8 or int8 with a scale per block and head, whose earlier tokens are held over
  the new scale when a new token raises it;
* ``attend``: attention over a cache with block scales: single tokens, verify windows, prompts
  (the attention backend's per-row and packed calls);
* ``load``: the cached keys and values of whole sequences as numbers (``load_kv``).

``listed()`` gives the fixed cases, ``draw(rng)`` one more of the same ranges;
``prepare`` makes a case's inputs from a seed, ``run`` is the timed pass -- the plain torch
form, or with ``own`` the framework's call -- ``work`` what it cannot do without and
``exact`` the same outputs in float64 from the definition.
"""

import functools
import importlib.util
import math
import os
import sys
import zlib

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _package():
    """The framework: the directory vllm-rlt_amd, imported as ``vllm_rlt_amd``."""
    if "vllm_rlt_amd" not in sys.modules:
        path = os.path.join(_ROOT, "vllm-rlt_amd")
        spec = importlib.util.spec_from_file_location(
            "vllm_rlt_amd", os.path.join(path, "__init__.py"), submodule_search_locations=[path])
        module = importlib.util.module_from_spec(spec)
        sys.modules["vllm_rlt_amd"] = module
        spec.loader.exec_module(module)
    return sys.modules["vllm_rlt_amd"]


_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_FP8 = torch.float8_e4m3fn
_DEV = "cuda"
# 8-bit pools: code type and the largest value that a code stands for before its scale
_CODES = {"fp8_vector": (_FP8, 448.0), "fp8_block": (_FP8, 448.0), "int8_block": (torch.int8, 127.0)}
_TINY = torch.finfo(torch.float32).tiny


# ------------------------------------------------------------------------------- cases

def _rotary(name, rows, far, heads, dim, rotary, scaling="none", interleaved=False, dtype="bf16"):
    """``rows`` tokens at positions below ``far``; the first ``rotary`` of ``dim`` turn."""
    return {"name": name, "kind": "rotary", "rows": rows, "far": far, "heads": heads[0],
            "kv_heads": heads[1], "dim": dim, "rotary": rotary, "scaling": scaling,
            "interleaved": interleaved, "dtype": dtype}


def _append(name, batch, new, ctx, heads, dim, pool, rotary, scaling="none", interleaved=False,
            dtype="bf16", block=16):
    """``new``: (fewest, most) rows appended per sequence behind ``ctx`` cached ones."""
    return {"name": name, "kind": "append", "batch": batch, "new_lo": new[0], "new_hi": new[1],
            "ctx_lo": ctx[0], "ctx_hi": ctx[1], "heads": heads[0], "kv_heads": heads[1],
            "dim": dim, "pool": pool, "rotary": rotary, "scaling": scaling,
            "interleaved": interleaved, "dtype": dtype, "block": block}


def _attend(name, batch, rows, ctx, heads, dim, pool, dtype="bf16", block=16, window=0):
    """``rows`` and ``ctx``: (fewest, most) per sequence; ``ctx`` counts the rows."""
    return {"name": name, "kind": "attend", "batch": batch, "rows_lo": rows[0],
            "rows_hi": rows[1], "ctx_lo": ctx[0], "ctx_hi": ctx[1], "heads": heads[0],
            "kv_heads": heads[1], "dim": dim, "pool": pool, "dtype": dtype, "block": block,
            "window": window}


def _load(name, batch, ctx, kv_heads, dim, pool, dtype="bf16", block=16):
    return {"name": name, "kind": "load", "batch": batch, "ctx_lo": ctx[0], "ctx_hi": ctx[1],
            "kv_heads": kv_heads, "dim": dim, "pool": pool, "dtype": dtype, "block": block}


def listed():
    return [
        # one decode token: one launch's latency
        _rotary("rotary_1", 1, 4096, (16, 16), 128, 128),
        # a long prompt far beyond the trained length, scaled frequencies, neighbouring pairs
        _rotary("rotary_16384", 16384, 1 << 20, (16, 4), 128, 64, "yarn", True),
        # one token of one sequence into an fp8 cache
        _append("append_1", 1, (1, 1), (700, 700), (16, 16), 128, "fp8_block", 128),
        # the serving batch's verify windows into a bf16 cache
        _append("append_32", 32, (5, 5), (100, 250), (16, 4), 128, "same", 128, "bands"),
        # ragged chunks into an fp8 cache with a scale per vector, behind a prefix
        _append("append_chunks_6", 6, (100, 700), (30, 200), (32, 8), 96, "fp8_vector", 96),
        # prompts into an int8 cache
        _append("append_prompts_8", 8, (2048, 2048), (0, 0), (16, 4), 128, "int8_block", 128),
        # one token of one sequence: the latency of an attention call
        _attend("attend_1", 1, (1, 1), (700, 700), (16, 16), 128, "int8_block"),
        # the serving batch's verify windows over an fp8 cache
        _attend("attend_32", 32, (5, 5), (1024, 8192), (16, 4), 128, "fp8_block"),
        # long contexts in int8, single tokens
        _attend("attend_long_64", 64, (1, 1), (16384, 32768), (16, 8), 128, "int8_block"),
        # prompts that have just been appended
        _attend("attend_prompts_8", 8, (2048, 2048), (2048, 2048), (16, 4), 128, "int8_block"),
        # a few short sequences moved out of the cache
        _load("load_4", 4, (40, 300), 4, 128, "fp8_block"),
        # a batch of long ones
        _load("load_16", 16, (2000, 8192), 8, 128, "int8_block"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((16, 16), (16, 4), (16, 8), (32, 8), (55, 55))
_SCALINGS = ("none", "linear", "ntk", "yarn", "bands")


def draw(rng):
    """A case of the listed ones' ranges; none costs more than the largest listed one."""
    kind = rng.choice(("rotary", "append", "append", "attend", "attend", "attend", "load"))
    heads = rng.choice(_HEADS)
    dim = rng.choice((64, 96, 128, 128, 256))
    part = rng.choice((1, 1, 2))  # all of the head turns, or half of it
    scaling, interleaved = rng.choice(_SCALINGS), rng.random() < 0.3
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    block = rng.choice((8, 16, 16, 32, 64))
    if kind == "rotary":
        most = 60_000_000 // (sum(heads) * dim)
        case = _rotary("", min(_log(rng, 1, 16384), most), _log(rng, 4096, 1 << 20), heads, dim,
                       dim // part, scaling, interleaved, rng.choice((dtype, dtype, "fp32")))
    elif kind == "append":
        pool = rng.choice(("same", "fp8_vector", "fp8_block", "fp8_block", "int8_block",
                           "int8_block"))
        new = _log(rng, 1, 2048)
        batch = max(1, min(_log(rng, 1, 64), 60_000_000 // ((sum(heads) + heads[1]) * dim * new)))
        before = rng.choice((0, rng.randint(1, 300)))
        case = _append("", batch, (max(1, new // rng.choice((1, 2, 4))), new),
                       (before // 2, before), heads, dim, pool, dim // part, scaling, interleaved,
                       dtype, block)
    elif kind == "attend":
        pool = rng.choice(("fp8_block", "int8_block"))
        rows = rng.choice((1, 1, rng.randint(2, 33), _log(rng, 64, 2048)))
        ctx = rows + _log(rng, 1, 32768 if rows < 64 else 2048)
        batch = _log(rng, 1, 64)
        batch = min(batch, int(8e8 / (heads[1] * dim * ctx)),
                    int(1.3e11 / (4 * rows * heads[0] * dim * ctx)),
                    int(1e9 / (heads[0] * rows * ctx)))
        case = _attend("", max(1, batch), (max(1, rows // rng.choice((1, 2))), rows),
                       (max(rows, ctx // rng.choice((1, 2, 8))), ctx), heads, dim, pool, dtype,
                       block, rng.choice((0, 0, 0, 1024)))
    else:
        pool = rng.choice(("fp8_vector", "fp8_block", "int8_block"))
        ctx = _log(rng, 1, 16384)
        batch = max(1, min(_log(rng, 1, 64), 120_000_000 // (heads[1] * dim * ctx)))
        case = _load("", batch, (max(1, ctx // rng.choice((1, 2, 8))), ctx), heads[1], dim, pool,
                     dtype, block)
    return {k: v for k, v in case.items() if k != "name"}


def _shape(case):
    """What belongs to the case (outputs keep their shapes, ``work`` its count): lengths and
    row counts.  Everything else comes from the seed."""
    key = repr(sorted((k, v) for k, v in case.items() if k != "name"))
    r = np.random.RandomState(zlib.crc32(key.encode()))
    kind, s = case["kind"], {}
    if kind == "rotary":
        return s
    n = case["batch"]
    ctx = r.randint(case["ctx_lo"], case["ctx_hi"] + 1, n)
    if kind == "append":
        s["rows"] = r.randint(case["new_lo"], case["new_hi"] + 1, n)
        s["rows"][0] = case["new_hi"]
        s["ctx"] = ctx + s["rows"]
        s["most"] = case["ctx_hi"] + case["new_hi"]
    elif kind == "attend":
        s["rows"] = r.randint(case["rows_lo"], case["rows_hi"] + 1, n)
        s["rows"][0] = case["rows_hi"]
        s["ctx"] = np.maximum(ctx, s["rows"])
        s["most"] = int(s["ctx"].max())
    else:
        s["rows"] = s["ctx"] = ctx
        s["most"] = int(ctx.max())
    return s


# -------------------------------------------------------------------------- frequencies

# Arguments of the scaled forms: a context 8 times the 4096 positions that were trained.
_SCALE_ARGS = {
    "none": {},
    "linear": {"factor": 8.0},
    "ntk": {"factor": 8.0},
    "yarn": {"factor": 8.0, "original_length": 4096, "fast": 32.0, "slow": 1.0},
    "bands": {"factor": 8.0, "original_length": 4096, "fast": 4.0, "slow": 1.0},
}
_BASE = 10000.0


def _frequencies(case):
    """Radians per position of every pair, and the factor on the sines and cosines."""
    r, scaling = case["rotary"], case["scaling"]
    a = _SCALE_ARGS[scaling]
    base = _BASE * (a["factor"] ** (r / (r - 2)) if scaling == "ntk" else 1.0)
    i = np.arange(r // 2)
    f = base ** (-2.0 * i / r)
    amplitude = 1.0
    if scaling == "linear":
        f = f / a["factor"]
    elif scaling == "yarn":
        # the pair that turns n times within the trained length has index at(n)
        low, high = (r * math.log(a["original_length"] / (2 * math.pi * n)) / (2 * math.log(base))
                     for n in (a["fast"], a["slow"]))
        low, high = max(math.floor(low), 0), min(math.ceil(high), r - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        f = f * (1 - ramp) + f / a["factor"] * ramp
        amplitude = 0.1 * math.log(a["factor"]) + 1
    elif scaling == "bands":
        turns = a["original_length"] * f / (2 * math.pi)
        keep = np.clip((turns - a["slow"]) / (a["fast"] - a["slow"]), 0, 1)
        f = f * (keep + (1 - keep) / a["factor"])
    return f, amplitude


# ------------------------------------------------------------------------------ inputs

def _rand_codes(shape, pool, g):
    """Codes of N(0, 1) values over 5 / 448 (fp8) or 4.5 / 127 (int8), filled in pieces."""
    dtype, top = _CODES[pool]
    scale = top / 5.0 if dtype == _FP8 else top / 4.5
    out = torch.empty(shape, dtype=dtype, device=_DEV)
    flat = out.view(-1)
    step = 1 << 28
    for i in range(0, flat.numel(), step):
        m = min(step, flat.numel() - i)
        x = torch.randn(m, generator=g, device=_DEV, dtype=torch.float16)
        x = x.mul_(scale).clamp_(-top, top)
        flat[i:i + m] = (x if dtype == _FP8 else x.round_()).to(dtype)
    return out


def _dev(x, dtype):
    return torch.as_tensor(np.ascontiguousarray(x)).to(dtype).to(_DEV)


def _prepare_pool(case, sh, g, h):
    n, bs = len(sh["ctx"]), case["block"]
    width = -(-sh["most"] // bs)
    blocks = n * width
    shape = (blocks, 2, bs, case["kv_heads"], case["dim"])  # two layers, the second one is used
    s = {"tables": torch.randperm(blocks, generator=h).int().view(n, width).to(_DEV),
         "lengths": _dev(sh["ctx"], torch.int32),
         "cu": _dev(np.concatenate([[0], np.cumsum(sh["rows"])]), torch.int32),
         "max_rows": int(sh["rows"].max()), "total": int(sh["rows"].sum()), "ks": None, "vs": None}
    if case["pool"] == "same":
        k, v = (torch.randn(shape, generator=g, device=_DEV, dtype=_DTYPES[case["dtype"]])
                for _ in range(2))
    else:
        k, v = (_rand_codes(shape, case["pool"], g) for _ in range(2))
        top = _CODES[case["pool"]][1]
        # a scale per token and head, or per block and head
        held = shape[:-1] if case["pool"] == "fp8_vector" else shape[:2] + shape[3:4]
        s["ks"], s["vs"] = ((torch.rand(held, generator=g, device=_DEV) * 0.5 + 0.75).mul_(
            4.0 / top)[:, 1] for _ in range(2))
    s["k"], s["v"] = k[:, 1], v[:, 1]
    return s


def _prepare_turns(case, s):
    f, s["amplitude"] = _frequencies(case)
    s["frequencies"] = _dev(f, torch.float64)


def prepare(case, seed):
    h = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=_DEV).manual_seed(seed)
    sh = _shape(case)
    kind, dt = case["kind"], _DTYPES[case["dtype"]]
    if kind == "rotary":
        rows, d = case["rows"], case["dim"]
        s = {"positions": torch.randint(0, case["far"], (rows,), generator=h).to(_DEV)}
        s["q"], s["key"] = (torch.randn(rows, heads, d, generator=g, device=_DEV, dtype=dt)
                            for heads in (case["heads"], case["kv_heads"]))
        _prepare_turns(case, s)
    else:
        s = _prepare_pool(case, sh, g, h)
        total, d = s["total"], case["dim"]
        if kind == "append":
            s["key"], s["value"] = (torch.randn(total, case["kv_heads"], d, generator=g,
                                                device=_DEV, dtype=dt) for _ in range(2))
            # the cached rows and the new ones, all of which are read back afterwards
            s["cu_all"] = _dev(np.concatenate([[0], np.cumsum(sh["ctx"])]), torch.int32)
            s["all"], s["max_all"] = int(sh["ctx"].sum()), int(sh["ctx"].max())
            _prepare_turns(case, s)
        if kind != "load":
            s["q"] = torch.randn(total, case["heads"], d, generator=g, device=_DEV, dtype=dt) * 1.5
    s["case"] = case
    return s


# ------------------------------------------------------------------- the framework's calls

@functools.lru_cache(maxsize=None)
def _plan(rotary, scaling, interleaved):
    """A model's rotation: made once, as a program that serves the model keeps it."""
    return _package().Rotary(rotary, _BASE, interleaved=interleaved, scaling=scaling,
                             device=_DEV, **_SCALE_ARGS[scaling])


@functools.lru_cache(maxsize=None)
def _backend(dtype, dim, block):
    return _package().create_backend("auto", _DEV, _DTYPES[dtype], dim, block)


def _own_run(s):
    case, pkg = s["case"], _package()
    kind = case["kind"]
    if kind == "rotary":
        return pkg.apply_rotary(s["q"], s["key"], s["positions"],
                                _plan(case["rotary"], case["scaling"], case["interleaved"]))
    pools = (s["k"], s["v"])
    if kind == "append":
        q = pkg.append_kv(*pools, s["key"], s["value"], s["tables"], s["lengths"], s["cu"],
                          s["max_rows"], s["ks"], s["vs"], q=s["q"],
                          rotary=_plan(case["rotary"], case["scaling"], case["interleaved"]))
        if case["pool"] == "same":
            return (q, *pools)
        return (q, s["ks"], s["vs"],
                *pkg.load_kv(*pools, s["tables"], s["lengths"], s["cu_all"], s["max_all"],
                             s["all"], s["ks"], s["vs"], dtype=_DTYPES[case["dtype"]]))
    if kind == "load":
        return pkg.load_kv(*pools, s["tables"], s["lengths"], s["cu"], s["max_rows"], s["total"],
                           s["ks"], s["vs"], dtype=_DTYPES[case["dtype"]])
    backend = _backend(case["dtype"], case["dim"], case["block"])
    if case["rows_hi"] > 1:
        return backend.prefill(s["q"], *pools, s["tables"], s["lengths"], s["cu"], s["max_rows"],
                               s["ks"], s["vs"], window=case["window"])
    if case["window"]:
        return backend.windowed(s["q"], *pools, s["tables"], s["lengths"], case["window"],
                                s["ks"], s["vs"])
    return backend(s["q"], *pools, s["tables"], s["lengths"], s["ks"], s["vs"])


# ------------------------------------------------------------------------- plain forms

def _turn(x, positions, s):
    """The rows of x [row, head, dim] turned by their positions, float32."""
    case = s["case"]
    r, x = case["rotary"], x.float()
    angle = positions.double()[:, None] * s["frequencies"]
    cos, sin = ((f(angle) * s["amplitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(y, -1).flatten(-2) if case["interleaved"] else torch.cat(y, -1)
    return torch.cat([y, x[..., r:]], -1)


def _places(s, cu, total):
    """(sequence, position) of every row of the packed windows that end at the lengths."""
    cu = cu.long()
    row = torch.arange(total, device=_DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    return seq, s["lengths"][seq].long() - cu[seq + 1] + row


def _code(x, pool):
    """x over its scale, as a code."""
    dtype, top = _CODES[pool]
    x = x.clamp(-top, top)
    return x.to(dtype) if dtype == _FP8 else x.round().to(dtype)


def _append_blocks(cache, scale, rows, first, block, offset, s):
    """Block scales: the largest new value of a block over the largest code, or the block's own
    scale where earlier tokens keep it above; these are held over the new scale."""
    pool = s["case"]["pool"]
    top = _CODES[pool][1]
    new = torch.zeros(scale.shape, device=_DEV).index_reduce_(0, block, rows.abs().amax(-1), "amax")
    new = (new * torch.tensor(1.0 / top, device=_DEV)).clamp_min(_TINY)
    # the blocks in which sequences go on behind cached tokens: their first rows' ones
    b, o = block[first], offset[first]
    old, went = scale[b], (o > 0)[:, None]
    new[b] = torch.where(went, torch.maximum(old, new[b]), new[b])
    values = cache[b].float() * old[:, None, :, None]
    before = torch.arange(cache.shape[1], device=_DEV)[None, :] < o[:, None]
    again = before[..., None, None] & (new[b] > old)[:, None, :, None]
    # (codes move as their bytes: 8-bit floats have few operations)
    move = torch.where(again, _code(values / new[b][:, None, :, None], pool).view(torch.uint8),
                       cache[b].view(torch.uint8))
    raw = cache.view(torch.uint8)
    raw[b] = move
    scale[block] = new[block]
    raw[block, offset] = _code(rows / new[block][..., None], pool).view(torch.uint8)


def _append_plain(s):
    case = s["case"]
    bs, pool = case["block"], case["pool"]
    seq, position = _places(s, s["cu"], s["total"])
    block = s["tables"][seq, position // bs].long()
    offset = position % bs
    first = s["cu"][:-1].long()
    key = _turn(s["key"], position, s)
    q = _turn(s["q"], position, s).to(s["q"].dtype)
    sides = ((s["k"], s["ks"], key), (s["v"], s["vs"], s["value"].float()))
    if pool == "same":
        s["k"][block, offset] = key.to(s["k"].dtype)
        s["v"][block, offset] = s["value"]
        return q, s["k"], s["v"]
    if pool == "fp8_vector":
        _append_vectors(*sides[0], block, offset)
        _append_vectors(*sides[1], block, offset)
    else:
        _append_blocks(*sides[0], first, block, offset, s)
        _append_blocks(*sides[1], first, block, offset, s)
    return (q, s["ks"], s["vs"], *_load_plain(s, s["cu_all"], s["all"]))


def _append_vectors(cache, scale, rows, block, offset):
    new = (rows.abs().amax(-1) * torch.tensor(1.0 / 448.0, device=_DEV)).clamp_min(_TINY)
    scale[block, offset] = new
    cache.view(torch.uint8)[block, offset] = _code(rows / new[..., None],
                                                   "fp8_vector").view(torch.uint8)


def _load_plain(s, cu, total):
    case = s["case"]
    seq, position = _places(s, cu, total)
    block = s["tables"][seq, position // case["block"]].long()
    offset = position % case["block"]

    def values(cache, scale):
        x = cache.view(torch.uint8)[block, offset].view(cache.dtype).float()
        held = scale[block] if scale.ndim == 2 else scale[block, offset]
        return (x * held[..., None]).to(_DTYPES[case["dtype"]])

    return values(s["k"], s["ks"]), values(s["v"], s["vs"])


def _attend_plain(s):
    """All sequences padded to the longest: rows [sequence, kv head, row x head of its group]."""
    case = s["case"]
    n, hkv, d, bs = case["batch"], case["kv_heads"], case["dim"], case["block"]
    group, most = case["heads"] // hkv, s["max_rows"]
    cu, lengths = s["cu"].long(), s["lengths"].long()
    tables = s["tables"].long()
    length = tables.shape[1] * bs

    def gathered(cache, scale):
        x = cache.view(torch.uint8)[tables].view(cache.dtype).float()  # [n, width, bs, hkv, d]
        x = x * scale[tables][:, :, None, :, None]
        return x.view(n, length, hkv, d).transpose(1, 2)

    count = cu[1:] - cu[:-1]
    at = torch.arange(most, device=_DEV)
    row = (cu[:-1, None] + at).clamp(max=s["total"] - 1)
    q = s["q"].float()[row]  # [n, most, heads, d]; rows behind a sequence's last are dropped
    q = q.view(n, most, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, most * group, d)
    x = torch.matmul(q, gathered(s["k"], s["ks"]).transpose(2, 3)) * (1.0 / math.sqrt(d))
    end = lengths[:, None] - count[:, None] + at + 1  # keys below it
    key = torch.arange(length, device=_DEV)
    sees = key < end[..., None]
    if case["window"]:
        sees = sees & (key >= end[..., None] - case["window"])
    sees = sees.repeat_interleave(group, 1)[:, None]
    x = torch.where(sees, x, torch.full((), -torch.inf, device=_DEV))
    e = torch.exp(x - x.amax(-1, keepdim=True))
    e = e / e.sum(-1, keepdim=True)
    o = torch.matmul(e, gathered(s["v"], s["vs"]).contiguous())
    o = o.view(n, hkv, most, group, d).permute(0, 2, 1, 3, 4).reshape(n, most, hkv * group, d)
    seq, _ = _places(s, s["cu"], s["total"])
    return o[seq, torch.arange(s["total"], device=_DEV) - cu[seq]].to(s["q"].dtype)


def run(s):
    if own:
        return _own_run(s)
    kind = s["case"]["kind"]
    if kind == "rotary":
        return (_turn(s["q"], s["positions"], s).to(s["q"].dtype),
                _turn(s["key"], s["positions"], s).to(s["key"].dtype))
    if kind == "append":
        return _append_plain(s)
    if kind == "load":
        return _load_plain(s, s["cu"], s["total"])
    return _attend_plain(s)


# -------------------------------------------------------------------------------- work

_ELT = {"bf16": 2, "fp16": 2, "fp32": 4}


def work(case):
    sh = _shape(case)
    kind, elt, d = case["kind"], _ELT[case["dtype"]], case["dim"]
    if kind == "rotary":
        size = case["rows"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * size * d * elt + 8 * case["rows"], "flops": 3 * size * case["rotary"]}
    hkv, bs, pool = case["kv_heads"], case["block"], case["pool"]
    code = elt if pool == "same" else 1

    def held(tokens):
        """Bytes of that many positions of one sequence's keys and values in the cache."""
        scales = {"same": 0, "fp8_vector": tokens}.get(pool, -(-tokens // bs))
        return 2 * hkv * (tokens * d * code + 4 * scales)

    if kind == "append":
        rows = int(sh["rows"].sum())
        bytes_ = 2 * rows * case["heads"] * d * elt + 2 * rows * hkv * d * elt
        bytes_ += sum(held(int(n)) for n in sh["rows"])
        if pool != "same":  # the sequences read back whole
            bytes_ += sum(held(int(n)) + 2 * hkv * int(n) * d * elt for n in sh["ctx"])
        return {"bytes": bytes_, "flops": rows * (3 * (case["heads"] + hkv) * case["rotary"] +
                                                  4 * hkv * d)}
    if kind == "load":
        return {"bytes": sum(held(int(n)) + 2 * hkv * int(n) * d * elt for n in sh["ctx"]),
                "flops": 2 * hkv * d * int(sh["ctx"].sum())}
    bytes_, flops = 0, 0
    for ctx, rows in zip(sh["ctx"], sh["rows"]):
        ctx, rows = int(ctx), int(rows)
        sees = ctx - rows + 1 + np.arange(rows, dtype=np.int64)
        keys = ctx
        if case["window"]:
            keys = min(keys, case["window"] + rows - 1)
            sees = np.minimum(sees, case["window"])
        bytes_ += held(keys) + 2 * rows * case["heads"] * d * elt + 4 * -(-keys // bs)
        flops += 4 * case["heads"] * d * int(sees.sum())
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------------------------- exact

def _exact_angles(case, positions):
    """cos and sin [row, pair] in float64, pair by pair from the scaling's definition."""
    r, scaling, a = case["rotary"], case["scaling"], _SCALE_ARGS[case["scaling"]]
    cos, sin = [], []
    for i in range(r // 2):
        f = _BASE ** (-2.0 * i / r)
        amplitude = 1.0
        if scaling == "linear":
            f /= a["factor"]
        elif scaling == "ntk":
            f *= a["factor"] ** (-2.0 * i / (r - 2))
        elif scaling == "yarn":
            # pairs below `low` keep their frequency, from `high` on it is divided
            index = [r * math.log(a["original_length"] / (2 * math.pi * n)) / (2 * math.log(_BASE))
                     for n in (a["fast"], a["slow"])]
            low, high = max(math.floor(index[0]), 0), min(math.ceil(index[1]), r - 1)
            t = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f = (1 - t) * f + t * f / a["factor"]
            amplitude = 1 + 0.1 * math.log(a["factor"])
        elif scaling == "bands":
            wave = 2 * math.pi / f
            if wave > a["original_length"] / a["slow"]:
                f /= a["factor"]
            elif wave > a["original_length"] / a["fast"]:
                t = (a["original_length"] / wave - a["slow"]) / (a["fast"] - a["slow"])
                f = t * f + (1 - t) * f / a["factor"]
        angle = positions.double() * f
        cos.append(amplitude * angle.cos())
        sin.append(amplitude * angle.sin())
    return torch.stack(cos, 1), torch.stack(sin, 1)


def _exact_turn(case, x, positions):
    """As complex numbers: pair i times amplitude e^(i angle)."""
    r = case["rotary"]
    cos, sin = _exact_angles(case, positions)
    y = x.double().clone()
    a, b = ((slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else
            (slice(0, r // 2), slice(r // 2, r)))
    z = torch.complex(y[..., a], y[..., b]) * torch.complex(cos, sin)[:, None]
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_code(x, pool):
    """The nearest value that a code stands for (ties to even): whole numbers up to 127, or
    three mantissa bits behind the leading one, steps of 2^-9 below 2^-6, up to 448."""
    top = _CODES[pool][1]
    if pool == "int8_block":
        return x.clamp(-top, top).round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return ((x / step).round() * step).clamp(-top, top)


def _exact_append(s):
    case, sh = s["case"], _shape(s["case"])
    bs, pool = case["block"], case["pool"]
    starts = np.concatenate([[0], np.cumsum(sh["rows"])])
    tables = s["tables"].tolist()
    positions = torch.cat([torch.arange(int(c) - int(n), int(c), device=_DEV)
                           for c, n in zip(sh["ctx"], sh["rows"])])
    out = [_exact_turn(case, s["q"], positions)]
    pools, scales, loaded = [], [], []
    for cache, scale, rows in ((s["k"], s["ks"], _exact_turn(case, s["key"], positions)),
                               (s["v"], s["vs"], s["value"].double())):
        c = cache.to(torch.float64) if pool == "same" else cache.float().double()
        f = None if scale is None else scale.double().clone()
        for i, (ctx, n) in enumerate(zip(sh["ctx"].tolist(), sh["rows"].tolist())):
            at = ctx - n
            while at < ctx:
                block, o = tables[i][at // bs], at % bs
                m = min(bs - o, ctx - at)
                first = int(starts[i]) + at - (ctx - n)
                new = rows[first:first + m]
                if pool == "same":
                    c[block, o:o + m] = new
                elif pool == "fp8_vector":
                    f[block, o:o + m] = (new.abs().amax(-1) / 448).clamp_min(_TINY)
                    c[block, o:o + m] = _exact_code(new / f[block, o:o + m, :, None], pool)
                else:
                    up = (new.abs().amax(-1).amax(0) / _CODES[pool][1]).clamp_min(_TINY)
                    if o:
                        up = torch.maximum(up, f[block])
                        again = _exact_code(c[block, :o] * (f[block] / up)[None, :, None], pool)
                        c[block, :o] = torch.where((up > f[block])[None, :, None], again,
                                                   c[block, :o])
                    f[block] = up
                    c[block, o:o + m] = _exact_code(new / up[None, :, None], pool)
                at += m
        pools.append(c)
        scales.append(f)
        if pool != "same":
            loaded.append(torch.cat([_exact_rows(c, f, tables[i], int(ctx), bs)
                                     for i, ctx in enumerate(sh["ctx"])]))
    return (*out, *pools) if pool == "same" else (*out, *scales, *loaded)


def _exact_rows(c, f, table, ctx, bs):
    """The first ctx positions of one sequence as numbers."""
    blocks = torch.tensor(table[:-(-ctx // bs)], device=_DEV)
    held = f[blocks][:, None, :, None] if f.ndim == 2 else f[blocks][..., None]
    return (c[blocks] * held).flatten(0, 1)[:ctx]


def _exact_attend(s):
    """Sequence by sequence and head by head."""
    case, sh = s["case"], _shape(s["case"])
    hkv, d, bs = case["kv_heads"], case["dim"], case["block"]
    group = case["heads"] // hkv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=_DEV)
    tables, begin = s["tables"].tolist(), 0
    for i, (ctx, rows) in enumerate(zip(sh["ctx"].tolist(), sh["rows"].tolist())):
        blocks = torch.tensor(tables[i][:-(-ctx // bs)], device=_DEV)
        key = torch.arange(ctx, device=_DEV)[None]
        end = torch.arange(ctx - rows + 1, ctx + 1, device=_DEV)[:, None]
        hidden = (key >= end) | ((key < end - case["window"]) if case["window"] else key < 0)
        for kvh in range(hkv):
            k, v = ((c[:, :, kvh][blocks].float().double() *
                     f.double()[blocks, kvh][:, None, None]).flatten(0, 1)[:ctx]
                    for c, f in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            for h in range(kvh * group, (kvh + 1) * group):
                x = s["q"][begin:begin + rows, h].double() @ k.t() / math.sqrt(d)
                out[begin:begin + rows, h] = torch.softmax(
                    x.masked_fill(hidden, -torch.inf), -1) @ v
        begin += rows
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return tuple(_exact_turn(case, x, s["positions"]) for x in (s["q"], s["key"]))
    if kind == "append":
        return _exact_append(s)
    if kind == "load":
        sh, tables = _shape(case), s["tables"].tolist()
        return tuple(torch.cat([_exact_rows(c.float().double(), f.double(), tables[i], int(ctx),
                                            case["block"]) for i, ctx in enumerate(sh["ctx"])])
                     for c, f in ((s["k"], s["ks"]), (s["v"], s["vs"])))
    return _exact_attend(s)
