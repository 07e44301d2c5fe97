"""Pools that share memory: the moves of two workgroups would race, so such calls are refused."""

import pytest
import torch

NULL, FAKE = None, 0x1000


def test_c_entry_refuses_shared_memory(pkg):
    from vllm_rlt_amd import _lib

    def commit(key=FAKE, value=FAKE, blocks=10, layers=2, bs=16, strides=(4096, 2048, 128), n=2):
        return _lib.library().rlt_kv_commit_path(
            FAKE, n, 1, 4, bs, FAKE, FAKE, 5, 5, FAKE, layers, blocks, key, value, *strides, 256, 2, NULL)

    assert commit() == 1 and commit(n=0) == 0
    for strides in ((0, 2048, 128), (4096, 0, 128), (4096, 2048, 0)):
        assert commit(value=FAKE + 1024, strides=strides) == 1


@pytest.mark.gpu
def test_operator_refuses_shared_memory(pkg, dev):
    """Refused before a launch; views side by side in one allocation are taken."""
    tables = torch.arange(4, device=dev).view(1, 4).int()
    starts, accepted = torch.tensor([3], device=dev), torch.tensor([2], device=dev)
    path = torch.tensor([[0, 2, 4]], device=dev)
    rest = (tables, starts, path, accepted, 4)
    both = torch.randn(9, 2, 4, 2, 16, device=dev)
    old = both.clone()
    shared = both[:1].expand(8, 2, 4, 2, 16)
    layer = both[:8, :1].expand(8, 2, 4, 2, 16)
    token = both[:8, :, :1].expand(8, 2, 4, 2, 16)
    other = torch.randn(9, 2, 4, 2, 16, device=dev)[:8]
    for k, v in ((both, both), (both[:8], both[:8]), (both[:8], both[1:]), (both[1:], both[:8]),
                 (shared, other[:1].expand(8, 2, 4, 2, 16)), (layer, other[:, :1].expand_as(layer)),
                 (token, other[:, :, :1].expand_as(token))):
        with pytest.raises(ValueError, match="overlap"):
            pkg.commit_tree_kv(k, v, *rest)
    torch.cuda.synchronize()
    assert torch.equal(both, old)
    # keys and values of one allocation: interleaved by layer, and one behind the other
    for k, v in ((both[:, :1], both[:, 1:]), (both[:4], both[4:8])):
        a, b = k.clone(), v.clone()
        pkg.commit_tree_kv(k, v, *rest)
        pkg.commit_tree_kv(a, b, *rest)
        assert torch.equal(k, a) and torch.equal(v, b)
    assert not torch.equal(both, old)
