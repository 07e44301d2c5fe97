"""Performance cases of the draft-tree verify round on one MI355X.

A round that verifies a tree of drafted tokens instead of a chain: node 0 of a request's
window is its last committed token, nodes 1 .. W are drafts, each the child of an earlier
node.  Five operators carry it, each reached as an engine reaches it:

* ``tree_attend``: one layer's attention of the window's nodes over a paged KV pool; a node
  sees the cached prefix, its ancestors and itself (``AttentionBackend.tree``);
* ``tree_accept``: the stochastic acceptance of the drafts along the tree, from target and
  draft distributions to the accepted path and the token after it (``tree_accept``);
* ``greedy_tree``: the greedy one, from target logits (``greedy_tree_accept``);
* ``commit``: the keys and values of the accepted nodes move to the positions behind the
  prefix, in every layer (``commit_tree_kv``);
* ``logprobs``: log probability, rank and entropy of given tokens with the top alternatives
  of their rows (``token_logprobs``).

``listed()`` gives the fixed cases, ``draw(rng)`` one more of the same ranges;
``prepare`` makes a case's inputs from a seed, ``run`` is the timed pass -- the plain torch
form, or with ``own`` the framework's call -- ``work`` what it cannot do without and
``exact`` the same outputs in float64 from the definition.
"""

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
_SCALE = 5.0 / 448.0  # a per-tensor scale that covers N(0, 1) values


# ------------------------------------------------------------------------------- cases

def _attend(name, batch, nodes, ctx, heads, dim, kv="same", dtype="bf16", block=16, window=0):
    """``nodes`` and ``ctx``: (fewest, most) per request, uniform; ``ctx`` counts the nodes.
    ``kv``: "same" (the pool in q's type), "fp8" (per-tensor scales) or "fp8_vector" (one
    scale per token and kv head)."""
    return {"name": name, "kind": "tree_attend", "batch": batch, "nodes_lo": nodes[0],
            "nodes_hi": nodes[1], "ctx_lo": ctx[0], "ctx_hi": ctx[1], "heads": heads[0],
            "kv_heads": heads[1], "dim": dim, "kv": kv, "dtype": dtype, "block": block,
            "window": window}


def _accept(name, n, width, vocab):
    return {"name": name, "kind": "tree_accept", "n": n, "width": width, "vocab": vocab}


def _greedy(name, n, width, vocab, logits):
    return {"name": name, "kind": "greedy_tree", "n": n, "width": width, "vocab": vocab,
            "logits": logits}


def _commit(name, n, width, layers, kv_heads, dim, dtype, block=16):
    return {"name": name, "kind": "commit", "n": n, "width": width, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "block": block}


def _logprobs(name, n, width, vocab, top, logits, every=False):
    """``every``: all n * (width + 1) logit rows; else the rows of a few tokens a request."""
    return {"name": name, "kind": "logprobs", "n": n, "width": width, "vocab": vocab, "top": top,
            "logits": logits, "every": every}


def listed():
    return [
        # one request, a small tree on a short context: one launch's latency
        _attend("tree_attend_1", 1, (16, 16), (700, 700), (16, 16), 128),
        # the serving batch: GQA 4, contexts up to 8192, trees of up to 32 nodes
        _attend("tree_attend_32", 32, (20, 32), (1024, 8192), (16, 4), 128),
        # wide trees on many heads of a size that is no power of two
        _attend("tree_attend_wide_16", 16, (64, 64), (2048, 2048), (55, 55), 96),
        # long contexts in fp8 with per-tensor scales
        _attend("tree_attend_fp8_64", 64, (16, 16), (16384, 32768), (16, 8), 128, kv="fp8"),
        # a few requests with small trees, sampled
        _accept("tree_accept_4", 4, 8, 49152),
        # a large batch of sampled requests
        _accept("tree_accept_128", 128, 15, 65536),
        # one greedy request with a large vocabulary, bf16 logits
        _greedy("greedy_tree_1", 1, 16, 151936, "bf16"),
        # the serving batch, greedy, float32 logits
        _greedy("greedy_tree_32", 32, 31, 49152, "fp32"),
        # the accepted path of one request over 24 layers
        _commit("commit_1", 1, 16, 24, 4, 128, "bf16"),
        # a large batch over 32 layers of an fp8 pool
        _commit("commit_64", 64, 31, 32, 8, 128, "fp8"),
        # the emitted tokens of one request with 5 alternatives each, bf16 logits
        _logprobs("logprobs_1", 1, 16, 151936, 5, "bf16"),
        # every verify row of a batch with 20 alternatives, float32 logits
        _logprobs("logprobs_160", 32, 4, 49152, 20, "fp32", every=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ones' ranges; none costs more than the largest listed one."""
    kind = rng.choice(("tree_attend", "tree_attend", "tree_attend", "tree_accept", "greedy_tree",
                       "commit", "logprobs"))
    if kind == "tree_attend":
        heads = rng.choice(((16, 16), (16, 4), (16, 8), (32, 8), (55, 55)))
        dim = rng.choice((64, 96, 128, 128, 256))
        kv = rng.choice(("same", "same", "fp8", "fp8_vector"))
        nodes = _log(rng, 2, 96)
        ctx = max(nodes + rng.randint(0, 64), _log(rng, 64, 32768))
        batch = _log(rng, 1, 64)
        batch = min(batch, int(8e8 / (heads[1] * dim * ctx)),
                    int(1.5e11 / (4 * nodes * heads[0] * dim * ctx)))
        case = _attend("", max(1, batch), (max(1, nodes // rng.choice((1, 2))), nodes),
                       (max(nodes, ctx // rng.choice((1, 2, 8))), ctx), heads, dim, kv,
                       rng.choice(("bf16", "bf16", "fp16")), rng.choice((8, 16, 16, 32)),
                       rng.choice((0, 0, 0, 1024)))
    elif kind == "commit":
        n, layers = _log(rng, 1, 64), rng.randint(4, 32)
        case = _commit("", n, rng.randint(2, 48), layers, rng.choice((4, 8, 16)),
                       rng.choice((64, 96, 128)), rng.choice(("bf16", "fp8")),
                       rng.choice((8, 16, 32)))
        if n * layers * case["kv_heads"] * case["dim"] > 2_000_000:
            case["layers"] = max(1, 2_000_000 // (n * case["kv_heads"] * case["dim"]))
    else:
        vocab = _log(rng, 8000, 152000)
        logits = rng.choice(("fp32", "bf16", "fp16"))
        if kind == "tree_accept":
            width = rng.randint(1, 31)
            n = _log(rng, 1, 128)
            case = _accept("", max(1, min(n, 100_000_000 // (vocab * (width + 1)))), width, vocab)
        else:
            width = rng.randint(1, 31)
            n = max(1, min(_log(rng, 1, 64), 45_000_000 // (vocab * (width + 1))))
            if kind == "greedy_tree":
                case = _greedy("", n, width, vocab, logits)
            else:
                every = n * (width + 1) * vocab < 7_500_000
                case = _logprobs("", n, width, vocab, rng.randint(1, 20), logits, every)
    return {k: v for k, v in case.items() if k != "name"}


def _shape(case):
    """What belongs to the case (outputs keep their shapes, ``work`` its count): lengths, tree
    shapes, accepted counts.  Everything else comes from the seed."""
    key = repr(sorted((k, v) for k, v in case.items() if k != "name"))
    r = np.random.RandomState(zlib.crc32(key.encode()))
    s = {}
    if case["kind"] == "tree_attend":
        n = case["batch"]
        s["nodes"] = r.randint(case["nodes_lo"], case["nodes_hi"] + 1, n)
        s["nodes"][0] = case["nodes_hi"]
        s["ctx"] = np.maximum(r.randint(case["ctx_lo"], case["ctx_hi"] + 1, n), s["nodes"])
        s["parents"] = [_tree(r, int(m) - 1) for m in s["nodes"]]
    else:
        n, w = case["n"], case["width"]
        s["drafts"] = r.randint(max(1, w - w // 4), w + 1, n)
        s["drafts"][0] = w
        s["parents"] = np.stack([_tree(r, w) for _ in range(n)])
        if case["kind"] == "commit":
            s["ctx"] = r.randint(0, 4 * case["block"], n)  # positions before the root
            s["path"], s["accepted"] = _paths(r, s["drafts"], w)
        if case["kind"] == "logprobs":
            s["emitted"] = np.minimum(1 + r.randint(0, 5, n), w + 1)
    return s


def _tree(r, drafts):
    """Parents of nodes 1 .. drafts (0 is the root): mostly later nodes, some siblings."""
    u = r.rand(drafts) ** 0.8
    return np.minimum((u * np.arange(1, drafts + 1)).astype(np.int64), np.arange(drafts))


def _paths(r, drafts, width):
    """Accepted paths: node 0, then ascending nodes.  A path's nodes are in place already or
    lie behind the positions that it fills, so that a pass can be repeated."""
    path = np.full((len(drafts), width + 1), -1, dtype=np.int64)
    acc = np.zeros(len(drafts), dtype=np.int64)
    for i, d in enumerate(drafts):
        a = int(min(r.randint(1, 7), d // 2))
        nodes = np.sort(r.choice(np.arange(a + 1, d + 1), a, replace=False)) if a else []
        if a and r.rand() < 0.5:
            nodes[0] = 1
        path[i, :a + 1] = [0, *nodes]
        acc[i] = a
    return path, acc


# ------------------------------------------------------------------------------ inputs

def _rand_codes(shape, g):
    """fp8 codes of N(0, 1) values over _SCALE, filled in pieces."""
    out = torch.empty(shape, dtype=_FP8, device=_DEV)
    flat = out.view(-1)
    step = 1 << 28
    for i in range(0, flat.numel(), step):
        m = min(step, flat.numel() - i)
        x = torch.randn(m, generator=g, device=_DEV, dtype=torch.float16)
        flat[i:i + m] = x.mul_(1.0 / _SCALE).clamp_(-448, 448).to(_FP8)
    return out


def _dev(x, dtype):
    return torch.as_tensor(np.ascontiguousarray(x)).to(dtype).to(_DEV)


def _mask_words(parents, words):
    """Rows of one request: bit j of word w set where the node sees node 64 w + j."""
    seen = []
    for i in range(len(parents) + 1):
        bits = (seen[parents[i - 1]] if i else 0) | (1 << i)
        seen.append(bits)
    out = np.zeros((len(seen), words), dtype=np.uint64)
    for i, bits in enumerate(seen):
        for w in range(words):
            out[i, w] = (bits >> (64 * w)) & 0xFFFFFFFFFFFFFFFF
    return out.view(np.int64)


def _prepare_attend(case, sh, g, h):
    n, bs = case["batch"], case["block"]
    dt = _DTYPES[case["dtype"]]
    width = -(-case["ctx_hi"] // bs)
    blocks = n * width
    words = -(-case["nodes_hi"] // 64)
    s = {"tables": torch.randperm(blocks, generator=h).int().view(n, width).to(_DEV),
         "lengths": _dev(sh["ctx"], torch.int32),
         "cu": _dev(np.concatenate([[0], np.cumsum(sh["nodes"])]), torch.int32),
         "max_q": case["nodes_hi"],
         "mask": _dev(np.concatenate([_mask_words(p, words) for p in sh["parents"]]), torch.int64),
         "bounds": [(int(c), int(m)) for c, m in zip(sh["ctx"], sh["nodes"])]}
    shape = (blocks, 2, bs, case["kv_heads"], case["dim"])  # two layers, the second one read
    if case["kv"] == "same":
        k, v = (torch.randn(shape, generator=g, device=_DEV, dtype=dt) for _ in range(2))
        ks = vs = None
    else:
        k, v = _rand_codes(shape, g), _rand_codes(shape, g)
        if case["kv"] == "fp8":
            ks, vs = (torch.tensor(_SCALE * x, device=_DEV) for x in (1.0, 0.9))
        else:
            ks, vs = ((torch.rand(shape[:-1], generator=g, device=_DEV) * 0.5 + 0.75).mul_(
                _SCALE)[:, 1] for _ in range(2))
    s["k"], s["v"], s["ks"], s["vs"] = k[:, 1], v[:, 1], ks, vs
    s["q"] = torch.randn(int(sh["nodes"].sum()), case["heads"], case["dim"], generator=g,
                         device=_DEV, dtype=dt) * 1.5
    if own:
        s["kernel"] = _package().create_backend("auto", _DEV, dt, case["dim"], bs)
    return s


def _prepare_rows(case, sh, g):
    """Target and draft logits of every node: the target's are the draft's with noise."""
    n, w, vocab = case["n"], case["width"], case["vocab"]
    draft = torch.randn(n, w, vocab, generator=g, device=_DEV).mul_(3.0)
    target = torch.empty(n, w + 1, vocab, device=_DEV)
    target[:, :w] = draft
    target[:, w] = draft[:, 0].flip(1)
    target += torch.randn(target.shape, generator=g, device=_DEV)
    return draft, target


def _prepare_accept(case, sh, g, h):
    n, w, vocab = case["n"], case["width"], case["vocab"]
    draft, target = _prepare_rows(case, sh, g)
    s = {"parents": _dev(sh["parents"], torch.int64), "drafts": _dev(sh["drafts"], torch.int64),
         "u_accept": torch.rand(n, w, generator=g, device=_DEV),
         "u_final": torch.rand(n, generator=g, device=_DEV)}
    s["q"] = draft.softmax(-1)
    s["p"] = target.softmax(-1)
    # each draft is drawn from its parent's draft distribution
    s["tokens"] = torch.empty(n, w, dtype=torch.int64, device=_DEV)
    at = torch.arange(n, device=_DEV)
    for j in range(w):
        s["tokens"][:, j] = torch.multinomial(s["q"][at, s["parents"][:, j]], 1,
                                              generator=g)[:, 0]
    return s


def _prepare_greedy(case, sh, g, h):
    n, w, vocab = case["n"], case["width"], case["vocab"]
    draft, target = _prepare_rows(case, sh, g)
    target = target.to(_DTYPES[case["logits"]])
    parents = sh["parents"]
    s = {"parents": _dev(parents, torch.int64), "drafts": _dev(sh["drafts"], torch.int64),
         "logits": target}
    # a node's children are the draft's best tokens in order, of which the first is most
    # often the target's best
    rank = np.zeros((n, w), dtype=np.int64)
    for i in range(n):
        seen = {}
        for j in range(w):
            rank[i, j] = seen.get(parents[i, j], 0)
            seen[parents[i, j]] = rank[i, j] + 1
    best = draft.topk(min(vocab, int(rank.max()) + 1), dim=-1).indices
    at = torch.arange(n, device=_DEV)[:, None]
    pick = best[at, s["parents"], _dev(rank, torch.int64)]
    sure = torch.rand(n, w, generator=g, device=_DEV) < 0.6
    first = _dev(rank == 0, torch.bool) & sure
    s["tokens"] = torch.where(first, target.float().argmax(-1)[at, s["parents"]], pick)
    return s


def _prepare_commit(case, sh, g, h):
    n, bs = case["n"], case["block"]
    width = (4 * bs + case["width"] + 1) // bs + 1
    shape = (n * width, case["layers"], bs, case["kv_heads"], case["dim"])
    if case["dtype"] == "fp8":
        k, v = _rand_codes(shape, g), _rand_codes(shape, g)
    else:
        k, v = (torch.randn(shape, generator=g, device=_DEV, dtype=_DTYPES[case["dtype"]])
                for _ in range(2))
    return {"k": k, "v": v, "starts": _dev(sh["ctx"], torch.int64),
            "tables": torch.randperm(n * width, generator=h).int().view(n, width).to(_DEV),
            "path": _dev(sh["path"], torch.int64), "accepted": _dev(sh["accepted"], torch.int64)}


def _prepare_logprobs(case, sh, g, h):
    n, w, vocab = case["n"], case["width"], case["vocab"]
    logits = (torch.randn(n * (w + 1), vocab, generator=g, device=_DEV) * 3.0).to(
        _DTYPES[case["logits"]])
    if case["every"]:
        rows, count = None, n * (w + 1)
        pick = torch.arange(count, device=_DEV)
    else:
        rows = torch.cat([i * (w + 1) + torch.randperm(w + 1, generator=h)[:int(m)]
                          for i, m in enumerate(sh["emitted"])]).to(_DEV)
        count, pick = rows.shape[0], rows
    # half of the tokens among the likely ones, half anywhere
    likely = logits[pick].float().topk(min(32, vocab), dim=-1).indices
    at = torch.randint(0, likely.shape[1], (count,), generator=h).to(_DEV)
    tokens = torch.randint(0, vocab, (count,), generator=h).to(_DEV)
    half = (torch.rand(count, generator=h) < 0.5).to(_DEV)
    tokens = torch.where(half, likely[torch.arange(count, device=_DEV), at], tokens)
    return {"logits": logits, "rows": rows, "tokens": tokens}


def prepare(case, seed):
    h = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=_DEV).manual_seed(seed)
    sh = _shape(case)
    kind = case["kind"]
    if kind == "tree_attend":
        s = _prepare_attend(case, sh, g, h)
    elif kind == "tree_accept":
        s = _prepare_accept(case, sh, g, h)
    elif kind == "greedy_tree":
        s = _prepare_greedy(case, sh, g, h)
    elif kind == "commit":
        s = _prepare_commit(case, sh, g, h)
    else:
        s = _prepare_logprobs(case, sh, g, h)
    s["case"] = case
    if own:
        _package()
    return s


# ------------------------------------------------------------------- the framework's calls

def _own_run(s):
    case, pkg = s["case"], _package()
    kind = case["kind"]
    if kind == "tree_attend":
        return s["kernel"].tree(s["q"], s["k"], s["v"], s["tables"], s["lengths"], s["cu"],
                                s["max_q"], s["mask"], s["ks"], s["vs"], window=case["window"])
    if kind == "tree_accept":
        return tuple(pkg.tree_accept(s["tokens"], s["parents"], s["drafts"], s["q"], s["p"],
                                     s["u_accept"], s["u_final"]))
    if kind == "greedy_tree":
        return tuple(pkg.greedy_tree_accept(s["tokens"], s["parents"], s["drafts"], s["logits"]))
    if kind == "commit":
        pkg.commit_tree_kv(s["k"], s["v"], s["tables"], s["starts"], s["path"], s["accepted"],
                           case["block"])
        return _pools(s)
    return tuple(pkg.token_logprobs(s["logits"], s["tokens"], rows=s["rows"], top_n=case["top"]))


# ------------------------------------------------------------------------- plain forms

def _pools(s):
    """The pools, 8-bit ones as the bytes of their codes: a move keeps every bit."""
    return tuple(x.view(torch.uint8) if x.dtype == _FP8 else x for x in (s["k"], s["v"]))


def _gathered(s, i, ctx, dtype):
    """Keys and values of request i, [kv_head, position, dim], in ``dtype``."""
    bs = s["k"].shape[1]
    blocks = s["tables"][i, :-(-ctx // bs)].long()
    out = []
    for pool, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        x = pool[blocks].to(dtype)
        if scale is not None:
            x = x * (scale.to(dtype) if scale.ndim == 0 else scale[blocks].to(dtype)[..., None])
        out.append(x.flatten(0, 1)[:ctx].transpose(0, 1).contiguous())
    return out


def _tree_attend(s, dtype):
    case, out = s["case"], []
    hkv, d = case["kv_heads"], case["dim"]
    group = case["heads"] // hkv
    begin = 0
    for i, (ctx, nodes) in enumerate(s["bounds"]):
        k, v = _gathered(s, i, ctx, dtype)
        q = s["q"][begin:begin + nodes].to(dtype)
        # rows of one kv head: (node, head of its group)
        q = q.view(nodes, hkv, group, d).transpose(0, 1).reshape(hkv, nodes * group, d)
        x = torch.matmul(q, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(d))
        at = torch.arange(nodes, device=_DEV)
        words = s["mask"][begin:begin + nodes]
        sees = ((words[:, at // 64] >> (at % 64)) & 1).bool()
        sees = torch.cat([torch.ones(nodes, ctx - nodes, dtype=torch.bool, device=_DEV), sees], 1)
        if case["window"]:
            # the last `window` of the positions that the node sees
            left = sees.flip(1).cumsum(1).flip(1)
            sees = sees & (left <= case["window"])
        sees = sees.repeat_interleave(group, 0)
        x = torch.where(sees, x, torch.full_like(x, -torch.inf))
        e = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
        out.append(o.view(hkv, nodes, group, d).transpose(0, 1).reshape(nodes, hkv * group, d))
        begin += nodes
    return torch.cat(out)


def _tree_accept(s):
    """Every draft in index order: a request stands at one node; a draft whose parent it is
    is accepted with the odds of target to draft weight, or what the draft distribution
    proposes is taken off the target's."""
    tokens, parents, p, q = s["tokens"], s["parents"], s["p"], s["q"]
    n, w = tokens.shape
    vocab = p.shape[-1]
    at = torch.arange(n, device=_DEV)
    node = torch.zeros(n, dtype=torch.int64, device=_DEV)
    off = torch.zeros(n, dtype=torch.float64, device=_DEV)  # multiples of q taken off p
    mass = torch.ones(n, dtype=torch.float64, device=_DEV)  # what is left of p
    count = torch.zeros_like(node)
    path = torch.full((n, w + 1), -1, dtype=torch.int64, device=_DEV)
    path[:, 0] = 0
    out = torch.zeros((n, w + 1), dtype=torch.int64, device=_DEV)

    def left():
        rows = q[at, node.clamp(max=w - 1)].double()
        return (p[at, node].double() - off[:, None] * rows).clamp_min(0)

    for j in range(w):
        here = (parents[:, j] == node) & (j < s["drafts"])
        t = tokens[:, j]
        px = p[at, node, t].double()
        qx = q[at, node.clamp(max=w - 1), t].double()
        yes = here & (s["u_accept"][:, j].double() * mass * qx < px - off * qx)
        no = here & ~yes
        off = torch.where(no, off + mass, off)
        mass = torch.where(no, left().sum(1), mass)
        node = torch.where(yes, torch.full_like(node, j + 1), node)
        off = torch.where(yes, torch.zeros_like(off), off)
        mass = torch.where(yes, torch.ones_like(mass), mass)
        place = torch.arange(w + 1, device=_DEV)[None]
        out = torch.where(yes[:, None] & (place == count[:, None]), t[:, None], out)
        count = count + yes
        path = torch.where(yes[:, None] & (place == count[:, None]), node[:, None], path)
    cdf = left().cumsum(1)
    total = cdf[:, -1]
    u = torch.minimum(s["u_final"].double() * total,
                      torch.nextafter(total, torch.zeros_like(total)))
    final = torch.searchsorted(cdf, u[:, None], right=True)[:, 0].clamp(0, vocab - 1)
    bad = ~(torch.isfinite(total) & (total > 0))
    out[at, count] = final
    return path, out, count, final, bad


def _greedy_tree(s):
    tokens, parents, x = s["tokens"], s["parents"], s["logits"].float()
    n, w = tokens.shape
    vocab = x.shape[-1]
    best = x.amax(-1, keepdim=True)
    columns = torch.arange(vocab, device=_DEV)
    targets = torch.where(x == best, columns, torch.full_like(columns, vocab)).amin(-1)
    at = torch.arange(n, device=_DEV)
    node = torch.zeros(n, dtype=torch.int64, device=_DEV)
    count = torch.zeros_like(node)
    path = torch.full((n, w + 1), -1, dtype=torch.int64, device=_DEV)
    path[:, 0] = 0
    place = torch.arange(w + 1, device=_DEV)[None]
    for j in range(w):
        yes = (parents[:, j] == node) & (j < s["drafts"]) & (tokens[:, j] == targets[at, node])
        node = torch.where(yes, torch.full_like(node, j + 1), node)
        count = count + yes
        path = torch.where(yes[:, None] & (place == count[:, None]), node[:, None], path)
    return targets, path, count, targets[at, node]


def _commit_moves(s):
    """(block, token) of the sources and targets of every accepted node."""
    path, starts, tables, bs = s["path"], s["starts"], s["tables"].long(), s["case"]["block"]
    n, w = path.shape
    j = torch.arange(w, device=_DEV)[None]
    live = (j <= s["accepted"][:, None]) & (path >= 0)
    # rows that do not move copy their root onto itself
    src = torch.where(live, starts[:, None] + path, starts[:, None])
    dst = torch.where(live, starts[:, None] + j, starts[:, None])
    at = torch.arange(n, device=_DEV)[:, None]
    return (tables[at, src // bs], src % bs), (tables[at, dst // bs], dst % bs)


def _commit_plain(s):
    (sb, so), (db, do) = _commit_moves(s)
    for pool in _pools(s):
        rows = pool.transpose(1, 2)  # [block, token, layer, ...]
        rows[db, do] = rows[sb, so]
    return _pools(s)


def _logprob_rows(s, dtype):
    case = s["case"]
    x = (s["logits"] if s["rows"] is None else s["logits"][s["rows"]]).to(dtype)
    at = torch.arange(x.shape[0], device=_DEV)
    t = s["tokens"]
    d = x - x.amax(-1, keepdim=True)
    e = torch.exp(d).double()
    total = e.sum(-1)
    lse = total.log()
    logprob = d[at, t].double() - lse
    entropy = lse - (e * d.double()).sum(-1) / total
    mine = x[at, t][:, None]
    before = (x > mine) | ((x == mine) & (torch.arange(x.shape[1], device=_DEV) < t[:, None]))
    rank = before.sum(-1) + 1
    value, order = x.sort(dim=-1, descending=True, stable=True)
    top = order[:, :case["top"]].contiguous()
    top_logprob = d.gather(1, top).double() - lse[:, None]
    return logprob, rank, entropy, top_logprob, top


def run(s):
    if own:
        return _own_run(s)
    case = s["case"]
    kind = case["kind"]
    if kind == "tree_attend":
        return _tree_attend(s, torch.float32).to(s["q"].dtype)
    if kind == "tree_accept":
        return _tree_accept(s)
    if kind == "greedy_tree":
        return _greedy_tree(s)
    if kind == "commit":
        return _commit_plain(s)
    logprob, rank, entropy, top_logprob, top = _logprob_rows(s, torch.float32)
    return logprob.float(), rank, entropy.float(), top_logprob.float(), top


# -------------------------------------------------------------------------------- work

_ELT = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}


def work(case):
    sh = _shape(case)
    kind = case["kind"]
    if kind == "tree_attend":
        elt = _ELT[case["dtype"]]
        kv = {"same": elt, "fp8": 1, "fp8_vector": 1}[case["kv"]]
        bytes_, flops = 0, 0
        for ctx, nodes, parents in zip(sh["ctx"], sh["nodes"], sh["parents"]):
            depth = np.ones(int(nodes), dtype=np.int64)
            for i in range(1, int(nodes)):
                depth[i] = depth[parents[i - 1]] + 1
            sees = int(ctx - nodes) + depth
            keys = int(ctx)
            if case["window"]:
                # the shallowest node reaches furthest back
                keys = min(keys, int(nodes) + max(0, case["window"] - 1))
                sees = np.minimum(sees, case["window"])
            per_key = 2 * case["kv_heads"] * (case["dim"] * kv +
                                              (4 if case["kv"] == "fp8_vector" else 0))
            bytes_ += keys * per_key + 2 * int(nodes) * case["heads"] * case["dim"] * elt
            bytes_ += 4 * -(-int(ctx) // case["block"]) + 8 * int(nodes)
            flops += 4 * case["heads"] * case["dim"] * int(sees.sum())
        return {"bytes": bytes_, "flops": flops}
    n, w = case["n"], case["width"]
    small = n * (w + 1) * 32
    if kind == "tree_accept":
        # the rows of the node where each request stops: its token is drawn from what is
        # left of p after q, which takes a sum and a search over the vocabulary
        return {"bytes": 2 * 4 * n * case["vocab"] + small, "flops": 6 * n * case["vocab"]}
    if kind == "greedy_tree":
        size = n * (w + 1) * case["vocab"]
        return {"bytes": size * _ELT[case["logits"]] + small, "flops": size}
    if kind == "commit":
        j = np.arange(w + 1)[None]
        live = (j <= sh["accepted"][:, None]) & (sh["path"] != j)
        row = case["layers"] * case["kv_heads"] * case["dim"] * _ELT[case["dtype"]]
        return {"bytes": 4 * int(live.sum()) * row + small, "flops": 0}
    rows = n * (w + 1) if case["every"] else int(sh["emitted"].sum())
    size = rows * case["vocab"]
    return {"bytes": size * _ELT[case["logits"]] + rows * (40 + 12 * case["top"]),
            "flops": 5 * size}


# ------------------------------------------------------------------------------- exact

def _exact_accept(s):
    """Request by request from the definition: the weights left at a node are the target's,
    then max(weights - mass * q, 0) after every rejected child."""
    tokens, parents = s["tokens"].tolist(), s["parents"].tolist()
    drafts, u = s["drafts"].tolist(), s["u_accept"].tolist()
    n, w = s["tokens"].shape
    path = torch.full((n, w + 1), -1, dtype=torch.int64)
    out = torch.zeros((n, w + 1), dtype=torch.int64)
    count, final, bad = [], [], []
    for i in range(n):
        node, steps = 0, 0
        weights = s["p"][i, 0].double()
        mass = 1.0
        path[i, 0] = 0
        for j in range(drafts[i]):
            if parents[i][j] != node:
                continue
            t = tokens[i][j]
            proposal = s["q"][i, node].double()
            if u[i][j] * mass * float(proposal[t]) < float(weights[t]):
                out[i, steps] = t
                steps += 1
                node = j + 1
                path[i, steps] = node
                weights, mass = s["p"][i, node].double(), 1.0
            else:
                weights = torch.relu(weights - mass * proposal)
                mass = float(weights.sum())
        cdf = weights.cumsum(0)
        total = float(cdf[-1])
        target = min(float(s["u_final"][i]) * total, float(np.nextafter(total, 0.0)))
        token = min(int((cdf <= target).sum()), weights.shape[0] - 1)
        out[i, steps] = token
        count.append(steps)
        final.append(token)
        bad.append(not (math.isfinite(total) and total > 0))
    return (path.to(_DEV), out.to(_DEV), torch.tensor(count, device=_DEV),
            torch.tensor(final, device=_DEV), torch.tensor(bad, device=_DEV))


def _exact_greedy(s):
    tokens, parents, drafts = s["tokens"].tolist(), s["parents"].tolist(), s["drafts"].tolist()
    x = s["logits"]
    n, w = s["tokens"].shape
    # the first of the largest: a stable order by descending value
    targets = torch.stack([row.double().sort(dim=-1, descending=True, stable=True).indices[:, 0]
                           for row in x])
    best = targets.tolist()
    path = torch.full((n, w + 1), -1, dtype=torch.int64)
    count, last = [], []
    for i in range(n):
        node, steps = 0, 0
        path[i, 0] = 0
        while True:
            hits = [j for j in range(drafts[i])
                    if parents[i][j] == node and tokens[i][j] == best[i][node]]
            if not hits:
                break
            node = hits[0] + 1
            steps += 1
            path[i, steps] = node
        count.append(steps)
        last.append(best[i][node])
    return targets, path.to(_DEV), torch.tensor(count, device=_DEV), torch.tensor(last,
                                                                                  device=_DEV)


def _exact_commit(s):
    k, v = (x.clone() for x in _pools(s))
    bs, tables = s["case"]["block"], s["tables"].tolist()
    starts, path, accepted = (s[x].tolist() for x in ("starts", "path", "accepted"))
    for i in range(len(starts)):
        for j in range(1, accepted[i] + 1):
            src, dst = starts[i] + path[i][j], starts[i] + j
            for pool in (k, v):
                pool[tables[i][dst // bs], :, dst % bs] = pool[tables[i][src // bs], :, src % bs]
    return k, v


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "tree_attend":
        return _exact_attend(s)
    if kind == "tree_accept":
        return _exact_accept(s)
    if kind == "greedy_tree":
        return _exact_greedy(s)
    if kind == "commit":
        return _exact_commit(s)
    return _exact_logprobs(s)


def _exact_attend(s):
    """Request by request and kv head by kv head, the visible positions from each node's
    walk to the root."""
    case, sh = s["case"], _shape(s["case"])
    hkv, d = case["kv_heads"], case["dim"]
    group = case["heads"] // hkv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=_DEV)
    begin = 0
    for i, (ctx, nodes) in enumerate(s["bounds"]):
        sees = np.zeros((nodes, ctx), dtype=bool)
        sees[:, :ctx - nodes] = True
        for node in range(nodes):
            a = node
            while True:
                sees[node, ctx - nodes + a] = True
                if a == 0:
                    break
                a = int(sh["parents"][i][a - 1])
            if case["window"]:
                seen = np.flatnonzero(sees[node])
                sees[node, seen[:-case["window"]]] = False
        hidden = torch.as_tensor(~sees).to(_DEV)
        k, v = _gathered(s, i, ctx, torch.float64)
        for kvh in range(hkv):
            for h in range(kvh * group, (kvh + 1) * group):
                x = s["q"][begin:begin + nodes, h].double() @ k[kvh].t() / math.sqrt(d)
                x = torch.softmax(x.masked_fill(hidden, -torch.inf), -1)
                out[begin:begin + nodes, h] = x @ v[kvh]
        begin += nodes
    return out


def _exact_logprobs(s):
    case, tokens = s["case"], s["tokens"].tolist()
    rows = range(len(tokens)) if s["rows"] is None else s["rows"].tolist()
    logprob, rank, entropy, top_logprob, top = [], [], [], [], []
    for r, t in zip(rows, tokens):
        x = s["logits"][r].double()
        lp = torch.log_softmax(x, -1)
        order = x.sort(descending=True, stable=True).indices
        logprob.append(lp[t])
        rank.append((order == t).nonzero()[0, 0] + 1)
        entropy.append(-(lp.exp() * lp).sum())
        top.append(order[:case["top"]])
        top_logprob.append(lp[top[-1]])
    return (torch.stack(logprob), torch.stack(rank), torch.stack(entropy),
            torch.stack(top_logprob), torch.stack(top))
