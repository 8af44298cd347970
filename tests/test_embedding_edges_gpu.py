"""The embedding's gradient where its kernels change over: vocabularies and position counts at the limits of
the sort, both sides of the one-launch sum, and runs at the borders of chunks."""
import pytest
import torch

import _ext
from embedding import embedding

pytestmark = pytest.mark.gpu
dev = "cuda"


def test_the_largest_vocabulary_that_is_accepted():
    """The sort's 2^22 groups of 512 tokens: the entry behind the last one is start[2^31], which an int does not
    hold.  600 positions (the sorted path), among them the ends of the vocabulary and of its last group."""
    V = 2 ** 31 - 1025
    last_group = 510 * 2 ** 22 + 2 ** 22 - 1          # the largest token whose low 22 bits are all ones
    tokens = torch.randint(0, V, (600,), generator=torch.Generator().manual_seed(0))
    tokens[:6] = torch.tensor([0, V - 1, last_group, last_group, 2 ** 22 - 1, V - 1])
    g = torch.randint(1, 5, (600, 1), generator=torch.Generator().manual_seed(1)).half()
    table = torch.zeros(1, 1, device=dev, dtype=torch.half).expand(V, 1)   # (the gradient reads its shape alone)
    grad = torch.ops.krsi.embedding_bwd(g.to(dev), tokens.to(dev), table, 1.0, -1)
    ids, at = torch.unique(tokens, return_inverse=True)
    want = torch.zeros(len(ids)).index_add_(0, at, g[:, 0].float())
    assert torch.equal(grad[ids.to(dev), 0].float().cpu(), want)
    assert int(torch.count_nonzero(grad)) == len(ids)
    assert _ext.device_status() == 0
