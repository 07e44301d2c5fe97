"""Tree attention at the ends of its arguments."""

import pytest
import torch

from tests.tree_cases import make_case
from tests.tree_dense import dense

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def attend(pkg, dev, c, kernel=None, **over):
    kernel = kernel or pkg.MI355XPagedAttention()
    a = dict(q=c.q, key_cache=c.k, value_cache=c.v, block_tables=c.tables, context_lengths=c.lengths,
             cu_seqlens_q=c.cu, max_seqlen_q=c.max_q, tree_mask=c.mask, key_scale=c.k_scale,
             value_scale=c.v_scale)
    a.update(over)
    return kernel.tree(**{k: v.to(dev) if torch.is_tensor(v) else v for k, v in a.items()})


def close(got, want, tol):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - tol
    assert over.max() <= 0, f"{float(over.max())} beyond the tolerance"


@pytest.mark.parametrize("dtype,kv,dim", [(BF, "same", 64), (HF, "fp8_vector", 128), (BF, "same", 80),
                                          (F32, "same", 64)])
@pytest.mark.parametrize("window", [(1 << 31) - 1, (1 << 31) - 200, 64, 33])
def test_windows_past_the_cache(pkg, dev, dtype, kv, dim, window):
    """A window of any size, up to the largest integer, over a tree whose cache is shorter than
    it, and over others: a window that covers the cache hides nothing."""
    c = make_case([70, 9, 3], [70, 40, 3], 4, 2, dim, dtype, kv, seed=dim)
    c.ctx = [64, 40, 2]  # nodes 0 .. 5 of the first tree, and node 0 of the last, do not exist
    lengths = torch.tensor(c.ctx, dtype=torch.int32)
    close(attend(pkg, dev, c, context_lengths=lengths, window=window), *dense(c, window))
