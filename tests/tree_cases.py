"""Seeded draft trees and a plain float64 attention over them, shared by the tree tests."""

import math

import numpy as np
import torch

from tests.attn_cases import random_tables

FP8 = torch.float8_e4m3fn


def random_parents(drafts, g):
    """Parents of nodes 1 .. drafts; node 0 is the root."""
    u = torch.rand(max(drafts, 1), generator=g)
    return [min(j, int(float(u[j]) ** 0.8 * (j + 1))) for j in range(drafts)]


def ancestor_bits(parents):
    """Python integers: bit j set where the node sees node j (its ancestors and itself)."""
    seen = []
    for i in range(len(parents) + 1):
        seen.append((seen[parents[i - 1]] if i else 0) | (1 << i))
    return seen


def pack_bits(rows, words):
    out = np.zeros((len(rows), words), dtype=np.uint64)
    for r, bits in enumerate(rows):
        for w in range(words):
            out[r, w] = (bits >> (64 * w)) & 0xFFFFFFFFFFFFFFFF
    return torch.from_numpy(out.view(np.int64))


class Case:
    """CPU tensors of one call.  Positions that no sequence owns hold NaN."""


def make_case(nodes, ctx, hq, hkv, dim, dtype=torch.bfloat16, kv="same", block=16, seed=0,
              bits=None, words=None, layers=2, sharp=1.5):
    g = torch.Generator().manual_seed(seed)
    c = Case()
    n = len(nodes)
    need = [max(1, math.ceil(x / block)) for x in ctx]
    num_blocks = sum(need) + 3
    c.tables = random_tables([max(x, 1) for x in ctx], block, num_blocks, g)
    shape = (num_blocks, layers, block, hkv, dim)
    owned = torch.zeros(num_blocks, block, dtype=torch.bool)
    for s in range(n):
        pos = torch.arange(ctx[s])
        owned[c.tables[s, pos // block].long(), pos % block] = True
    c.k_scale = c.v_scale = None
    if kv == "same":
        k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    else:
        k, v = ((torch.randn(shape, generator=g) * 60).clamp(-448, 448).to(FP8) for _ in range(2))
        if kv == "fp8":
            c.k_scale, c.v_scale = torch.tensor(1 / 60.0), torch.tensor(1 / 50.0)
        else:
            c.k_scale, c.v_scale = ((torch.rand(shape[:-1], generator=g) + 0.5) / 60
                                    for _ in range(2))
            for x in (c.k_scale, c.v_scale):
                x.transpose(1, 2)[~owned] = math.nan
            c.k_scale, c.v_scale = c.k_scale[:, -1], c.v_scale[:, -1]
    for x in (k, v):
        y = x.float().transpose(1, 2)
        y[~owned] = math.nan
        x.copy_(y.transpose(1, 2).to(x.dtype))
    c.k, c.v = k[:, -1], v[:, -1]
    c.q = (torch.randn(sum(nodes), hq, dim, generator=g) * sharp).to(dtype)
    c.lengths = torch.tensor(ctx, dtype=torch.int32)
    c.cu = torch.tensor(np.concatenate([[0], np.cumsum(nodes)]), dtype=torch.int32)
    c.max_q = max(nodes)
    c.words = words or max(1, -(-c.max_q // 64))
    c.parents = [random_parents(m - 1, g) for m in nodes]
    c.bits = bits if bits is not None else [ancestor_bits(p) if m else []
                                            for m, p in zip(nodes, c.parents)]
    c.mask = pack_bits([b for rows in c.bits for b in rows], c.words)
    c.nodes, c.ctx, c.block = nodes, ctx, block
    return c


def visible(c, s, window=0):
    """[nodes, ctx] booleans of sequence s, from the definition."""
    m, length = c.nodes[s], c.ctx[s]
    base = length - m
    sees = np.zeros((m, length), dtype=bool)
    for i in range(m):
        for p in range(length):
            sees[i, p] = p < base or (c.bits[s][i] >> (p - base)) & 1
        if window:
            at = np.flatnonzero(sees[i])
            sees[i, at[:-window]] = False
    return torch.from_numpy(sees)


def gathered(c, s):
    """float64 keys and values of sequence s, [kv_head, position, dim]."""
    pos = torch.arange(c.ctx[s])
    blocks, off = c.tables[s, pos // c.block].long(), pos % c.block
    out = []
    for pool, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x = pool[blocks, off].double()
        if scale is not None:
            x = x * (scale.double() if scale.ndim == 0 else scale[blocks, off].double()[..., None])
        out.append(x.transpose(0, 1))
    return out


def reference(c, window=0, fine=False):
    """(output, tolerance) in float64, [rows, heads, dim].

    The tolerance counts the roundings of a kernel that takes scores in float32, weights in q's
    16-bit type (float32 for float32 q) next to a float32 denominator, and rounds the output
    once.  With u the type's half step and A = sum p |v|: u A for the weights, u |out| for the
    output; each score is off by at most D 2^-24 sum |q k| / sqrt(D), which moves a weight and
    the denominator by that much each; float32 sums over the keys, L 2^-24 A; and fp16 weights
    below 2^-14 are multiples of 2^-24 next to a sum of at least 1, so they add 2^-25 of the
    values as the product holds them (codes where a scale is in the weight).

    ``fine`` counts what a kernel leaves that keeps the largest fp16 weight at 2^7 or more:
    2^-32 of the values; and with a scale in the weight, the largest product of weight and scale
    there too (up to 2^4 lower where the running maximum has moved since it was taken): 2^-28
    of it times the codes.
    """
    rows, hq, dim = c.q.shape
    hkv = c.k.shape[2]
    group = hq // hkv
    out = torch.zeros(rows, hq, dim, dtype=torch.float64)
    tol = torch.zeros_like(out)
    u = torch.finfo(c.q.dtype).eps / 2
    begin = 0
    for s, m in enumerate(c.nodes):
        if m and c.ctx[s]:
            sees = visible(c, s, window)
            k, v = gathered(c, s)
            for h in range(hq):
                q = c.q[begin:begin + m, h].double()
                kk, vv = k[h // group], v[h // group]
                x = (q @ kk.nan_to_num(0, 0, 0).t() / math.sqrt(dim)).masked_fill(~sees, -math.inf)
                size = (q.abs() @ kk.nan_to_num(0, 0, 0).abs().t() / math.sqrt(dim))
                size = size.masked_fill(~sees, 0).amax(-1, keepdim=True)
                p = torch.softmax(x, -1).nan_to_num(0.0)  # a row that sees nothing
                o, a = p @ vv.nan_to_num(0, 0, 0), p @ vv.nan_to_num(0, 0, 0).abs()
                es = 2 * dim * 2.0 ** -24 * size
                t = a * (u + es + (c.ctx[s] + 8) * 2.0 ** -24) * 1.01 + u * o.abs()
                if c.q.dtype == torch.float16:
                    held = vv
                    if c.v_scale is not None and c.v_scale.ndim == 3:
                        pos = torch.arange(c.ctx[s])
                        held = held / c.v_scale[c.tables[s, pos // c.block].long(),
                                                pos % c.block][:, h // group, None].double()
                    unit = 2.0 ** -25
                    if fine and held is not vv:
                        y = c.v_scale[c.tables[s, pos // c.block].long(), pos % c.block][:, h // group]
                        unit = 2.0 ** -28 * (p * y.double().abs()).amax(-1, keepdim=True)
                    elif fine:
                        unit = 2.0 ** -32
                    t = t + unit * (sees.double() @ held.abs().nan_to_num(0, 0, 0)) + 2.0 ** -25
                out[begin:begin + m, h] = o
                tol[begin:begin + m, h] = t
        begin += m
    return out, tol
