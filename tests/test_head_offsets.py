"""Class head where the scores lie far from 0: common offsets, and groups of 64 classes that hold nothing but
switched-off classes or the label.

Bounds as in test_head.py: they count |bias| in every score's rounding, so they grow with the offset.
"""
import pytest
import torch

from test_head import BOTH, Ref, label_targets, list_targets, lists, make
from ytk_learn_amd.ops import head

SHIFTS = [0.0, -80.0, -95.0, -120.0, -300.0, 120.0]
# few rows and tiled ones in either type
ROWS = [1, 5, 150, 300]


def _shifted(V, shift, dtype, dev):
    b = torch.full((V,), shift, dtype=dtype, device=dev)
    assert bool((b.double() == shift).all())
    return b


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("shift", SHIFTS)
def test_label_alone_in_its_group(cuda, dtype, n, shift):
    """One class; and a last group of one class that is every row's label."""
    for V in (1, 65, 193):
        x, w, _, _ = make(n, 64, V, dtype, cuda)
        y = torch.full((n,), V - 1, device=cuda)
        b = _shifted(V, shift, dtype, cuda)
        r = head.softmax_head_loss(x, w, y, bias=b)
        Ref(x, w, *label_targets(y), bias=b).check(r, db=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("shift", SHIFTS)
def test_whole_groups_switched_off(cuda, dtype, n, shift):
    """Groups at -inf beside live classes of any offset, losses of labels and of lists. A switched-off class has no gradient."""
    V = 400
    x, w, y, _ = make(n, 64, V, dtype, cuda)
    off = torch.zeros(V, dtype=torch.bool, device=cuda)
    off[64:192] = True
    off[384:] = True
    on = (~off).nonzero()[:, 0]
    y = on[y % len(on)]
    b = _shifted(V, shift, dtype, cuda)
    b[off] = float("-inf")
    r = head.softmax_head_loss(x, w, y, bias=b)
    Ref(x, w, *label_targets(y), bias=b).check(r, db=True)
    assert bool((r.dw[off] == 0).all()) and bool((r.db[off] == 0).all())
    idx, tl = lists(n, len(on), 6)
    idx = torch.where(idx >= 0, on.cpu()[idx.clamp(min=0)], idx)
    for T in (1.0, 0.25):  # (a small temperature stretches the scores)
        r = head.distill_head_loss(x, w, idx.to(cuda), tl.to(cuda), bias=b, temperature=T)
        Ref(x, w, idx, list_targets(idx, tl, T), bias=b, T=T).check(r, db=True)
        assert bool((r.dw[off] == 0).all()) and bool((r.db[off] == 0).all())
