"""Class head where the scores lie far from 0: common offsets, groups of 64 classes that hold nothing but
switched-off classes or the label, and masks of large negative biases.

Bounds as in test_head.py: they count |bias| in every score's rounding, so they grow with the offset.
"""
import pytest
import torch

from test_head import BOTH, Ref, U, label_targets, list_targets, lists, make, near, topk_ref
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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", ROWS)
def test_groups_masked_by_large_biases(cuda, dtype, n):
    """Whole groups at a large negative bias count for nothing, whatever its size and the temperature: the results are
    those of the other classes alone. (At -1e4 / 3.5 and below e^z is 0 in any precision beside scores around 0.)"""
    V = 400
    x, w, y, _ = make(n, 64, V, dtype, cuda)
    off = torch.zeros(V, dtype=torch.bool, device=cuda)
    off[0:128] = True
    off[300::3] = True
    keep = ~off
    on = keep.nonzero()[:, 0]
    y = on[y % len(on)]
    sub = Ref(x, w[keep], *label_targets(torch.cumsum(keep, 0)[y] - 1))
    idx, tl = lists(n, len(on), 6)
    at = torch.where(idx >= 0, on.cpu()[idx.clamp(min=0)], idx)
    temps = (1.0, 1.5, 2.0, 3.0, 3.5)
    subs = {T: Ref(x, w[keep], idx, list_targets(idx, tl, T), T=T) for T in temps}
    lowest = torch.finfo(dtype).min
    for low in (-1e4, -3e7, -1e9, -1e30, -2.445e38, lowest, float("-inf")):
        b = torch.zeros(V, dtype=dtype, device=cuda)
        b[off] = low
        calls = [(sub, head.softmax_head_loss(x, w, y, bias=b)), (sub, head.softmax_head_loss(x, w, y, bias=b, want_dx=False, want_dw=False))]
        calls += [(subs[T], head.distill_head_loss(x, w, at.to(cuda), tl.to(cuda), bias=b, temperature=T)) for T in temps]
        for ref, r in calls:
            near(r.loss, ref.loss, ref.eloss, f"loss at {low}")
            near(r.lse, ref.lse, ref.elin, f"lse at {low}")
            if r.dx is None:
                continue
            near(r.dx, ref.dx, ref.edx, f"dx at {low}")
            near(r.dw[keep], ref.dw, ref.edw, f"dw at {low}")
            assert bool((r.dw[off] == 0).all()) and bool((r.db[off] == 0).all())
        for T in temps:
            _, c, l = head.head_topk(x, w, 5, bias=b, temperature=T)
            assert torch.equal(c, topk_ref(x, w, b, T, 5)[1])
            near(l, subs[T].lse, subs[T].elin, f"lse at {low}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", ROWS)
def test_label_at_the_lowest_bias(cuda, dtype, n):
    """A label whose class is switched off by the type's lowest value has that score, not an infinite one."""
    x, w, y, _ = make(n, 64, 200, dtype, cuda)
    off = int(y[0])
    mine = y == off
    keep = torch.arange(200, device=cuda) != off
    lowest = torch.finfo(dtype).min
    b = torch.zeros(200, dtype=dtype, device=cuda)
    b[off] = lowest
    r = head.softmax_head_loss(x, w, y, bias=b)
    sub = Ref(x, w[keep], *label_targets(torch.where(mine, torch.zeros_like(y), torch.cumsum(keep, 0)[y] - 1)))
    other = ~mine.cpu()
    near(r.lse, sub.lse, sub.elin, "lse")
    near(r.loss[~mine], sub.loss[other], sub.eloss[other], "loss")
    far = torch.full((int(mine.sum()),), -lowest, dtype=torch.float64)  # the scores around 0 are lost in its rounding
    near(r.loss[mine], far, 4 * U * far, "loss at the lowest")
    # D is -1 there and p elsewhere, as for any other score that far off
    b[off] = -1e30
    for a, c in zip(r[2:], head.softmax_head_loss(x, w, y, bias=b)[2:]):
        assert bool(a.isfinite().all()) and torch.equal(a, c)
