"""Class head where the scores lie far from 0 or close together: common offsets, groups of 64 classes that hold nothing but
switched-off classes or the label, masks of large negative biases, and scores nearer to each other than fp32 tells apart.

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


def _close_scores(kind, n, d, V, dtype, dev):
    """Scores that 64-bit sums tell apart and 32-bit ones do not."""
    g = torch.Generator().manual_seed(V + n)
    x, w = torch.randn(n, d, generator=g), torch.randn(V, d, generator=g)
    b = None
    if kind == "bias":  # a common bias of 64 and differences of 1e-6: below its rounding of 4e-6
        w, b = w * 1e-7, torch.full((V,), 64.0)
    elif kind == "column":  # a common product of 10^6 beside the others
        x[:, d // 2], w[:, d // 2] = 1000.0, 1000.0
    elif kind == "cancel":  # 3 is lost beside 10^9, which another column takes away again
        w = w * (0.5 / d ** 0.5)
        x[:, 0] = x[:, d // 2] = x[:, d - 1] = 1.0
        w[:, 0], w[:, d - 1] = 1e9, -1e9
        w[:, d // 2] = (torch.arange(V) * 7919 % V).float() / V
    elif kind == "outlier":  # the same in one class alone, beside ordinary ones
        w = w * (0.5 / d ** 0.5)
        x[:, 0] = x[:, d // 2] = x[:, d - 1] = 1.0
        w[V - 2] = 0.0
        w[V - 2, 0], w[V - 2, d // 2], w[V - 2, d - 1] = 1e9, 12.0, -1e9
    elif kind == "same":  # every class alike
        w[:] = w[0]
    elif kind == "zero":
        w[:] = 0.0
    return x.to(dtype).to(dev), w.to(dtype).to(dev), None if b is None else b.to(dtype).to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("kind", ["bias", "column", "cancel", "outlier", "same", "zero"])
@pytest.mark.parametrize("n,d,V,k", [(1, 64, 3000, 5), (7, 130, 3000, 256), (70, 64, 700, 40), (300, 64, 3000, 1), (300, 72, 1009, 200),
                                     (2, 40, 140001, 30)])
def test_topk_of_scores_that_32_bits_mix_up(cuda, dtype, kind, n, d, V, k):
    """The k best and their order are those of the 64-bit sums, whatever the 32-bit scores say."""
    x, w, b = _close_scores(kind, n, d, V, dtype, cuda)
    T = 2.0 if k % 2 == 0 else 1.0
    v, c, _ = head.head_topk(x, w, k, bias=b, temperature=T)
    z = x.double() @ w.double().t()
    z = (z if b is None else z + b.double()) / T
    # the two 64-bit sums add in other orders: each is off by d 2^-53 sum |x||w| at most
    e = (d + 4) * 2.0 ** -53 * (x.double().abs() @ w.double().abs().t() + (0 if b is None else b.double().abs())) / T
    rv, rc = z.sort(dim=1, descending=True, stable=True)
    got = z.gather(1, c)
    bound = e.amax(1, keepdim=True)
    assert all(len(set(r)) == k for r in c.tolist())
    assert bool(((got - rv[:, :k]).abs() <= 2 * bound).all())
    apart = (rv[:, :k] - rv[:, 1:k + 1] > 4 * bound) & (torch.cat([rv.new_full((n, 1), float("inf")), rv[:, :k - 1]], 1) - rv[:, :k] > 4 * bound)
    assert torch.equal(c[apart], rc[:, :k][apart])
    if kind in ("same", "zero"):
        assert c.tolist() == [list(range(k))] * n
    else:
        assert float(apart.double().mean()) > 0.5
    near(v, rv[:, :k].cpu(), (1.01 * U * rv[:, :k].abs() + 2 * bound).cpu() + 1e-40, "values")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", [3, 300])
def test_topk_of_close_scores_in_pieces_strides_and_graphs(cuda, dtype, n, monkeypatch):
    """Rows scored again in 64 bits, beside ordinary ones: the same answers from transposed weights, in pieces of rows, and from a
    captured call replayed on other inputs."""
    k, V, d = 40, 1500, 64
    sets = []
    for seed in range(3):
        x, w, b = _close_scores("bias", n, d, V, dtype, cuda)
        x = x.roll(seed, 0)
        x[::2] *= 2.0 ** (20 + seed)  # scores that 32 bits do tell apart
        sets.append((x, w.roll(seed, 0), b))
    want = [head.head_topk(*s[:2], k, bias=s[2]) for s in sets]
    for (x, w, b), (v, c, l) in zip(sets, want):
        assert torch.equal(c, topk_ref(x, w, b, 1.0, k)[1])
        got = head.head_topk(x, w.t().contiguous().t(), k, bias=b)
        assert torch.equal(got[0], v) and torch.equal(got[1], c)
    x, w, b = (t.clone() for t in sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        head.head_topk(x, w, k, bias=b)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = head.head_topk(x, w, k, bias=b)
    for i in (1, 2, 0, 1):
        for t, s in zip((x, w, b), sets[i]):
            t.copy_(s)
        g.replay()
        eager = head.head_topk(x, w, k, bias=b)
        torch.cuda.synchronize()
        for a, e, u in zip(out, eager, want[i]):
            assert torch.equal(a, e) and torch.equal(a, u)
    monkeypatch.setattr(head, "PIECE_BYTES", 1 << 10)
    for s, u in zip(sets, want):
        for a, e in zip(head.head_topk(*s[:2], k, bias=s[2]), u):
            assert torch.equal(a, e)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n,d,V", [(2, 1 << 21, 3), (140, 1 << 21, 3), (2, 3, 1 << 21), (140, 2, 1 << 21)])
def test_most_features_and_classes(cuda, dtype, n, d, V):
    """The documented limits: 2^21 features, 2^21 classes."""
    g = torch.Generator(device=cuda).manual_seed(d + n)
    x = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    w = (torch.randn(V, d, generator=g, device=cuda) * (2.0 / d ** 0.5)).to(dtype)
    y = torch.randint(0, V, (n,), generator=g, device=cuda)
    r = head.softmax_head_loss(x, w, y)
    v, c, l = head.head_topk(x, w, min(V, 9))
    z = x.double() @ w.double().t()
    assert torch.equal(c, z.sort(dim=1, descending=True, stable=True).indices[:, :9])
    lse = torch.logsumexp(z, 1)
    # a score is a sum of d products: off by at most (d + 64) u sum |x||w|, and that is at most |x| |w|
    ez = (d + 64) * U * (x.double().norm(dim=1) * w.double().norm(dim=1).max())
    near(r.lse, lse.cpu(), (ez + (128 + V / 64) * U * (1 + lse.abs())).cpu(), "lse")
    near(l, lse.cpu(), (ez + (128 + V / 64) * U * (1 + lse.abs())).cpu(), "lse of the best")
    near(r.loss, (lse - z.gather(1, y[:, None])[:, 0]).cpu(), (2 * ez + (256 + V / 32) * U * (1 + lse.abs())).cpu(), "loss")
    D = torch.softmax(z, 1)
    D[torch.arange(n, device=cuda), y] -= 1
    rel = torch.expm1((2 * ez).clamp(max=1.0))[:, None] + 2.0 ** -6
    for got, D2, o in ((r.dx, D, w), (r.dw, D.t(), x)):
        eD = (D.abs() * rel + 2.0 ** -38) if D2 is D else (D.abs() * rel + 2.0 ** -38).t()
        want = D2 @ o.double()
        bound = eD @ o.double().abs() + 2.0 ** -7 * want.abs() + 1e-30
        bad = (got.double() - want).abs() > bound
        assert not bool(bad.any()), float(((got.double() - want).abs() / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", [5, 150])
@pytest.mark.parametrize("T", [1e-6, 1e-3, 1e3, 1e6])
def test_distill_at_extreme_temperatures(cuda, dtype, n, T):
    """The documented limits of the temperature, with a group switched off."""
    V = 200
    x, w, _, _ = make(n, 64, V, dtype, cuda)
    b = torch.zeros(V, dtype=dtype, device=cuda)
    b[64:128] = float("-inf")
    idx, tl = lists(n, 64, 6)
    for tlse in (None, torch.logsumexp(tl.double() / T, 1).float()):
        r = head.distill_head_loss(x, w, idx.to(cuda), tl.to(cuda), bias=b, temperature=T, top_lse=None if tlse is None else tlse.to(cuda))
        assert all(bool(t.isfinite().all()) for t in r)
        if tlse is None or T >= 1:  # (t / T - top_lse of 10^6 has a rounding of its own, which q shows)
            Ref(x, w, idx, list_targets(idx, tl, T, tlse), bias=b, T=T).check(r, db=True)
