"""The multiclass linear model on dense rows (``dense_head``): building the rows repeats bit by bit."""
import pytest
import torch

from test_head import U, near


@pytest.mark.gpu
def test_repeated_features_add_up_the_same_every_time(cuda):
    """A feature named many times in a row: the order of its sum does not change from call to call."""
    from ytk_learn_amd.models.continuous.multiclass import dense_rows
    from ytk_learn_amd.ops.sparse import SparseMatrix

    g = torch.Generator().manual_seed(5)
    n, F, each = 64, 7, 700
    cols = torch.randint(0, F, (n * each,), generator=g, dtype=torch.int32)
    vals = torch.randn(n * each, generator=g) * 10.0 ** torch.randint(-6, 7, (n * each,), generator=g)
    X = SparseMatrix((torch.arange(n + 1) * each).to(cuda), cols.to(cuda), vals.to(cuda), F)
    first = dense_rows(X)
    exact = torch.zeros(n, F, dtype=torch.float64)
    at = (torch.repeat_interleave(torch.arange(n), each), cols.long())
    exact.index_put_(at, vals.double(), accumulate=True)
    size = torch.zeros(n, F, dtype=torch.float64).index_put_(at, vals.double().abs(), accumulate=True)
    near(first, exact, each * U * size, "rows")
    for _ in range(8):
        assert torch.equal(dense_rows(X), first)
