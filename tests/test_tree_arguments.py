"""Refusals of the draft-tree operators, and their schemas, without a GPU."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

NULL, FAKE = None, 0x1000


def lib(pkg):
    from vllm_rlt_amd import _lib
    return _lib.library()


def attend(pkg, seqs=2, max_q=5, rows=10, hq=16, hkv=4, d=128, bs=16, q_dtype=2, kv_dtype=2,
           scale_mode=0, scales=NULL, window=0, mask=FAKE, words=1, stride=1, width=8, blocks=64,
           ws_bytes=1 << 30, q=FAKE, ws=FAKE):
    return lib(pkg).rlt_tree_attention(
        q, hq * d, d, FAKE, FAKE, bs * hkv * d, hkv * d, d, bs * hkv * d, hkv * d, d, blocks,
        FAKE, width, width, FAKE, FAKE, mask, stride, words, seqs, max_q, rows, scales, scales,
        scale_mode, 0, 0, 0, hq, hkv, d, bs, q_dtype, kv_dtype, window, FAKE, hq * d, d, ws,
        ws_bytes, NULL)


def test_tree_attention_statuses(pkg):
    assert attend(pkg, seqs=0) == 0 and attend(pkg, rows=0) == 0 and attend(pkg, max_q=0) == 0
    assert attend(pkg, hq=6) == 1
    assert attend(pkg, blocks=0) == 1
    assert attend(pkg, window=-1) == 1
    assert attend(pkg, q=NULL) == 1
    assert attend(pkg, mask=NULL) == 1
    assert attend(pkg, mask=FAKE + 4) == 1
    assert attend(pkg, max_q=65) == 1             # one word holds 64 nodes
    assert attend(pkg, words=2, stride=1) == 1
    assert attend(pkg, q_dtype=3, kv_dtype=3, scale_mode=1, scales=FAKE) == 1
    assert attend(pkg, kv_dtype=3) == 1           # an fp8 pool without scales
    assert attend(pkg, scale_mode=1, scales=FAKE) == 1
    assert attend(pkg, kv_dtype=3, scale_mode=1) == 1
    assert attend(pkg, kv_dtype=1) == 2           # a pool of another 16-bit type
    assert attend(pkg, max_q=257, words=5, stride=5) == 2
    assert attend(pkg, d=257) == 2
    assert attend(pkg, width=1 << 28) == 2
    assert attend(pkg, ws_bytes=16) == 3
    size = lib(pkg).rlt_tree_attention_workspace_size
    assert size(2, 5, 16, 4, 128, 2) > 0 and size(2, 5, 16, 4, 80, 2) == 0
    assert size(2, -1, 4, 4, 128, 2) == 0


def test_round_statuses(pkg):
    L = lib(pkg)

    def greedy(n=2, w=4, vocab=100, stride=100, dtype=0, x=FAKE, ws=FAKE, nbytes=1 << 20):
        return L.rlt_greedy_tree_accept(FAKE, FAKE, FAKE, x, dtype, stride, n, w, vocab, FAKE, FAKE,
                                        FAKE, FAKE, ws, nbytes, NULL)

    assert greedy(n=0) == 0
    assert greedy(n=-1) == 1 and greedy(vocab=0) == 1 and greedy(stride=99) == 1
    assert greedy(x=NULL) == 1
    assert greedy(w=256) == 2 and greedy(dtype=3) == 2
    assert greedy(vocab=(1 << 20) + 1, stride=1 << 21) == 2
    assert greedy(ws=NULL) == 3 and greedy(nbytes=8) == 3 and greedy(ws=FAKE + 4) == 3

    def sampled(n=2, w=4, vocab=100, p=FAKE, q=FAKE):
        return L.rlt_tree_accept(FAKE, FAKE, FAKE, q, p, FAKE, FAKE, n, w, vocab, FAKE, FAKE, FAKE,
                                 FAKE, FAKE, NULL)

    assert sampled(n=0) == 0
    assert sampled(w=-1) == 1 and sampled(p=NULL) == 1 and sampled(q=NULL) == 1
    assert sampled(w=256) == 2 and sampled(vocab=(1 << 20) + 1) == 2

    def logprobs(dtype=0, stride=100, m=5, vocab=100, rows=NULL, count=5, top=3, lp=FAKE, tl=FAKE,
                 ws=FAKE, nbytes=1 << 20):
        return L.rlt_token_logprobs(FAKE, dtype, stride, m, vocab, rows, FAKE, count, top, lp, FAKE,
                                    FAKE, tl, FAKE, ws, nbytes, NULL)

    assert logprobs(count=0) == 0
    assert logprobs(stride=99) == 1 and logprobs(count=6) == 1 and logprobs(top=-1) == 1
    assert logprobs(lp=NULL) == 1 and logprobs(tl=NULL) == 1
    assert logprobs(dtype=3) == 2 and logprobs(top=65) == 2
    assert logprobs(vocab=2, stride=2, top=3) == 2 and logprobs(rows=FAKE, count=65536) == 2
    assert logprobs(ws=NULL) == 3 and logprobs(nbytes=8) == 3

    def commit(n=2, planes=1, width=4, bs=16, path_width=5, layers=2, per=256, elt=2, k=FAKE):
        return L.rlt_kv_commit_path(FAKE, n, planes, width, bs, FAKE, FAKE, path_width, path_width,
                                    FAKE, layers, 10, k, FAKE, 4096, 2048, 128, per, elt, NULL)

    assert commit(n=0) == 0 and commit(path_width=1) == 0 and commit(width=0) == 0
    assert commit(planes=0) == 1 and commit(bs=0) == 1 and commit(per=0) == 1 and commit(k=NULL) == 1
    assert commit(path_width=257) == 2 and commit(layers=40000) == 2
    assert L.rlt_tree_masks(FAKE, 4, 4, FAKE, 2, FAKE, 1, 0, NULL) == 0
    assert L.rlt_tree_masks(FAKE, 3, 4, FAKE, 2, FAKE, 1, 5, NULL) == 1
    assert L.rlt_tree_masks(FAKE, 4, 4, NULL, 2, FAKE, 1, 5, NULL) == 1
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_launches_of_more_threads_than_an_axis_holds(pkg):
    L = lib(pkg)
    assert attend(pkg, seqs=1 << 21, ws_bytes=1 << 40) == 2
    assert attend(pkg, seqs=1 << 25, d=80, ws_bytes=1 << 40) == 2
    assert L.rlt_tree_accept(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 22, 4, 10, FAKE, FAKE,
                             FAKE, FAKE, FAKE, NULL) == 2
    assert L.rlt_greedy_tree_accept(FAKE, FAKE, FAKE, FAKE, 0, 10, 1 << 16, 255, 10, FAKE, FAKE, FAKE,
                                    FAKE, FAKE, 1 << 40, NULL) == 2
    assert L.rlt_kv_commit_path(FAKE, 1 << 23, 2, 4, 16, FAKE, FAKE, 5, 5, FAKE, 2, 10, FAKE, FAKE,
                                4096, 2048, 128, 256, 2, NULL) == 2
    assert L.rlt_tree_masks(FAKE, 256, 256, FAKE, 2, FAKE, 5, 5, NULL) == 2


def test_host_tensors_are_refused(pkg):
    i64 = dict(dtype=torch.int64)
    t, d = torch.zeros(2, 3, **i64), torch.zeros(2, **i64)
    p = torch.zeros(2, 4, 9)
    with pytest.raises(ValueError, match="ROCm"):
        pkg.tree_accept(t, t, d, p[:, :3], p, torch.zeros(2, 3), torch.zeros(2))
    with pytest.raises(ValueError, match="ROCm"):
        pkg.greedy_tree_accept(t, t, d, p)
    with pytest.raises(ValueError, match="ROCm"):
        pkg.token_logprobs(p[0], torch.zeros(4, **i64))
    with pytest.raises(ValueError, match="ROCm"):
        pkg.tree_masks(t, torch.zeros(3, dtype=torch.int32), 4)
    pool = torch.zeros(4, 2, 8, 2, 16)
    with pytest.raises(ValueError, match="ROCm"):
        pkg.commit_tree_kv(pool, pool, torch.zeros(2, 2, dtype=torch.int32), d,
                           torch.zeros(2, 4, **i64), d, 8)
    q = torch.zeros(4, 2, 64)
    kernel = pkg.MI355XPagedAttention()
    cache = torch.zeros(4, 16, 1, 64)
    args = (q, cache, cache, torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
            torch.zeros(2, dtype=torch.int32), 4, torch.zeros(4, 1, **i64))
    with pytest.raises(ValueError, match="ROCm"):
        kernel.tree(*args)
    for window in (-1, 1.5, True):
        with pytest.raises(ValueError, match="window"):
            kernel.tree(*args, window=window)


def test_operators_are_cpp_with_shape_functions(pkg):
    for op in ("tree_attention", "tree_masks", "tree_accept", "greedy_tree_accept", "token_logprobs",
               "commit_tree_kv"):
        assert op in pkg.ops.OPS
        kernels = torch._C._dispatch_dump(f"rlt_mi355x::{op}")
        assert "CUDA: registered at" in kernels and "torch_bindings.cpp" in kernels, op
    ops = torch.ops.rlt_mi355x
    assert "!) key_pool" in str(ops.commit_tree_kv.default._schema)
    with pytest.raises(NotImplementedError, match="CPU"):
        ops.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long))
    with FakeTensorMode():
        i64 = dict(dtype=torch.int64)
        q = torch.empty(10, 16, 128, dtype=torch.bfloat16)
        kc = torch.empty(64, 16, 4, 128, dtype=torch.bfloat16)
        i32 = dict(dtype=torch.int32)
        out = ops.tree_attention(q, kc, kc, torch.empty(2, 8, **i32), torch.empty(2, **i32),
                                 torch.empty(3, **i32), 5, torch.empty(10, 1, **i64))
        assert out.shape == q.shape and out.dtype == q.dtype
        t, d = torch.empty(3, 7, **i64), torch.empty(3, **i64)
        p = torch.empty(3, 8, 50)
        res = ops.tree_accept(t, t, d, torch.empty(3, 7, 50), p, torch.empty(3, 7), torch.empty(3))
        assert [tuple(x.shape) for x in res] == [(3, 8), (3, 8), (3,), (3,), (3,)]
        assert res[4].dtype == torch.bool
        res = ops.greedy_tree_accept(t, t, d, p)
        assert [tuple(x.shape) for x in res] == [(3, 8), (3, 8), (3,), (3,)]
        res = ops.token_logprobs(p[0], torch.empty(8, **i64), None, 4)
        assert [tuple(x.shape) for x in res] == [(8,), (8,), (8,), (8, 4), (8, 4)]
        assert ops.tree_masks(t, torch.empty(4, **i32), 20).shape == (20, 1)
