"""Plain float64 tree attention of large cases: visibility and products as whole matrices."""

import math

import torch


def sees(c, s, window=0):
    """[nodes, ctx] booleans of sequence s; a context shorter than the tree holds its last nodes."""
    m, length = c.nodes[s], c.ctx[s]
    bits = torch.tensor([[(b >> j) & 1 for j in range(m)] for b in c.bits[s]], dtype=torch.bool)
    node = torch.arange(length) - (length - m)
    vis = torch.ones(m, length, dtype=torch.bool)
    vis[:, node >= 0] = bits.view(m, m)[:, node[node >= 0]]
    if window:
        vis &= vis.flip(1).cumsum(1).flip(1) <= window
    return vis


def dense(c, window=0, second=False):
    """(output, tolerance) in float64, [rows, heads, dim].

    With u the half step of q's type and A = sum p |v|: a weight rounded to that type is off by
    u of itself (float32 q: 2^-24), and by u^2 where a second product takes what the first
    rounding dropped, itself rounded (``second``); the output is rounded once, u |out|.  A
    score is a float32 sum of D products, off by D 2^-24 sum |q k| / sqrt(D), and moves a weight and
    the denominator by that much each.  Float32 sums over the keys, two products a key with
    ``second``: (2 L + 8) 2^-24 A.  fp16 weights are held 2^7 or more above their place, so one
    below the type's smallest step is off by 2^-32 of the values; where a scale is in the weight,
    by 2^-28 of the largest such product times the codes; an fp16 output by 2^-25 below its
    smallest step.
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
            vis = sees(c, s, window).repeat_interleave(group, 0)  # rows (node, q head of the group)
            pos = torch.arange(c.ctx[s])
            blocks, off = c.tables[s, pos // c.block].long(), pos % c.block
            for h in range(hkv):
                x, scale = [], []
                for pool, sc in ((c.k, c.k_scale), (c.v, c.v_scale)):
                    y = pool[blocks, off, h].double()
                    f = None
                    if sc is not None:
                        f = sc.double() if sc.ndim == 0 else sc[blocks, off, h].double()[:, None]
                        y = y * f
                    x.append(y.nan_to_num(0, 0, 0))
                    scale.append(f)
                k, v = x
                q = c.q[begin:begin + m, h * group:(h + 1) * group].double().reshape(m * group, dim)
                score = (q @ k.t() / math.sqrt(dim)).masked_fill(~vis, -math.inf)
                size = (q.abs() @ k.abs().t() / math.sqrt(dim)).masked_fill(~vis, 0).amax(-1, keepdim=True)
                p = torch.softmax(score, -1).nan_to_num(0.0)
                o, a = p @ v, p @ v.abs()
                es = 2 * dim * 2.0 ** -24 * size
                t = a * ((u * u if second else u) + es + (2 * c.ctx[s] + 8) * 2.0 ** -24) * 1.01 + u * o.abs()
                if c.q.dtype == torch.float16:
                    held, unit = v, 2.0 ** -32
                    if c.v_scale is not None and c.v_scale.ndim == 3:
                        f = scale[1].nan_to_num(1.0)
                        held = v / f
                        unit = 2.0 ** -28 * (p * f[:, 0].abs()).amax(-1, keepdim=True)
                    t = t + unit * (vis.double() @ held.abs()) + 2.0 ** -25
                where = slice(begin, begin + m), slice(h * group, (h + 1) * group)
                out[where] = o.view(m, group, dim)
                tol[where] = t.view(m, group, dim)
        begin += m
    return out, tol
