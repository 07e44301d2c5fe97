"""Tree attention calls that hold no work, or hold it for some sequences only."""

import pytest
import torch

from tests.test_gpu_tree_edges import attend
from tests.tree_cases import make_case

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype,kv,dim", [(BF, "same", 128), (HF, "fp8", 64), (F32, "same", 32)])
def test_calls_without_sequences_or_nodes(pkg, dev, dtype, kv, dim):
    """Rows but no sequence, sequences of no nodes, no rows: nothing is read, shapes and types are
    the queries'; a sequence without rows or without keys stands beside others."""
    c = make_case([5, 9], [70, 130], 4, 2, dim, dtype, kv, seed=9)
    none = torch.zeros(0, dtype=torch.int32)
    for over in (dict(block_tables=c.tables[:0], context_lengths=none, cu_seqlens_q=torch.zeros(1, dtype=torch.int32)),
                 dict(max_seqlen_q=0),
                 dict(q=c.q[:0], tree_mask=c.mask[:0], cu_seqlens_q=torch.zeros(3, dtype=torch.int32))):
        got = attend(pkg, dev, c, **over)
        assert got.shape == over.get("q", c.q).shape and got.dtype == dtype and got.device == dev
    got = attend(pkg, dev, c, cu_seqlens_q=torch.tensor([0, 0, 14], dtype=torch.int32),
                 max_seqlen_q=14, context_lengths=torch.tensor([70, 0], dtype=torch.int32))
    assert got.shape == c.q.shape and (got == 0).all()
