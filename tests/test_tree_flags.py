"""The flags of the tree attention entry, and the operator's option, without a GPU."""

import torch
from torch._subclasses.fake_tensor import FakeTensorMode

NULL, FAKE = None, 0x1000


def test_flags(pkg):
    from vllm_rlt_amd import _lib

    def attend(flags, rows=10, ws_bytes=16):
        return _lib.library().rlt_tree_attention_flags(
            FAKE, 2048, 128, FAKE, FAKE, 8192, 512, 128, 8192, 512, 128, 64, FAKE, 8, 8, FAKE, FAKE, FAKE,
            1, 1, 2, 5, rows, NULL, NULL, 0, 0, 0, 0, 16, 4, 128, 16, 2, 2, 0, flags, FAKE, 2048, 128,
            FAKE, ws_bytes, NULL)

    assert attend(0, rows=0) == 0 and attend(1, rows=0) == 0
    assert attend(2) == 1 and attend(-1) == 1
    assert attend(0) == 3 and attend(1) == 3  # the workspace is too small


def test_operator_option(pkg):
    op = torch.ops.rlt_mi355x.tree_attention
    assert "bool compensate=False" in str(op.default._schema)
    with FakeTensorMode():
        i32 = dict(dtype=torch.int32)
        q, kc = torch.empty(10, 16, 128), torch.empty(64, 16, 4, 128)
        args = (q, kc, kc, torch.empty(2, 8, **i32), torch.empty(2, **i32), torch.empty(3, **i32), 5,
                torch.empty(10, 1, dtype=torch.int64), None, None, 0)
        assert op(*args, True).shape == op(*args).shape == q.shape
