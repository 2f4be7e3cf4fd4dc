"""Class head on operands whose scores are exact in fp32, and on rows that are sure of their label: what is left is the rounding
of the softmax itself, so a missing plane of a product or a cancelled difference shows.

u = 2^-24. A row's sum of exponentials is off by (additions in a group, over groups, exponentials) 64 + V / 64 + 64 of u
and 2 u |z - max| for the arguments, as in test_head.py.
"""
import pytest
import torch

from test_head import BOTH, H, U, make, near
from ytk_learn_amd.ops import head


def _exact_scores(kind, n, d, V):
    """fp32 operands of up to three bf16 planes whose hi parts cancel in pairs of features. Every product and partial sum is a
    multiple of one unit below 2^24 of it, so any order of sums is exact."""
    g = torch.Generator().manual_seed(n + d)
    sign = torch.tensor([1.0, -1.0]).repeat(d // 2)
    if kind == "both middle":  # (1 + 2^-9 a)(1 + 2^-9 b) - (1 + 2^-9 a): 2^-9 b + 2^-18 a b
        a = torch.randint(0, 2, (n, d // 2), generator=g).repeat_interleave(2, 1)
        b = torch.randint(0, 2, (V, d // 2), generator=g)
        x = 1 + a / 512
        w = torch.stack([1 + b / 512, -torch.ones(V, d // 2)], 2).reshape(V, d)
        return x, w
    # 2^17 + 2^9 e + c (hi, middle and low plane) less 2^17 + 2^9 e, times 1: c
    rows = n if kind == "x in three planes" else V
    e = torch.randint(0, 2, (rows, d // 2), generator=g)
    c = torch.randint(0, 4, (rows, d // 2), generator=g)
    wide = torch.stack([131072.0 + 512 * e + c, 131072.0 + 512 * e], 2).reshape(rows, d)
    other = sign * torch.randint(0, 2, (n + V - rows, d // 2), generator=g).repeat_interleave(2, 1)
    return (wide / 64, other) if rows == n and kind == "x in three planes" else (other, wide / 64)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["x in three planes", "w in three planes", "both middle"])
@pytest.mark.parametrize("n,d,V", [(1, 64, 300), (20, 128, 300), (70, 96, 300), (150, 64, 300), (150, 512, 200), (300, 256, 1000)])
def test_every_plane_takes_part(cuda, kind, n, d, V):
    x, w = _exact_scores(kind, n, d, V)
    z = x.double() @ w.double().t()
    assert torch.equal(z, z.float().double())
    y = torch.arange(n) % V
    lse = torch.logsumexp(z, 1)
    tol = (128 + V / 64 + 2 * (z - z.amax(1, keepdim=True)).abs().amax(1).clamp(max=100)) * U + 4 * U * lse.abs()
    zy = z.gather(1, y[:, None])[:, 0]
    for grads in (False, True):
        r = head.softmax_head_loss(x.to(cuda), w.to(cuda), y.to(cuda), want_dx=grads, want_dw=grads)
        near(r.lse, lse, tol, "lse")
        near(r.loss, lse - zy, tol + 8 * U * (lse.abs() + zy.abs()), "loss")
    v, _, l = head.head_topk(x.to(cuda), w.to(cuda), 3)
    near(l, lse, tol, "lse of the top 3")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 40, 150, 300])
def test_student_that_is_its_teacher(cuda, n):
    """Every class on the list with the student's own score: p and q cancel to the rounding of each."""
    V, d = 200, 64
    g = torch.Generator().manual_seed(n)
    x, w = torch.randint(-8, 9, (n, d), generator=g) / 8.0, torch.randint(-4, 5, (V, d), generator=g) / 4.0
    z = x.double() @ w.double().t()  # multiples of 1/32 below 2^9
    idx = torch.stack([torch.randperm(V, generator=g) for _ in range(n)])
    r = head.distill_head_loss(x.to(cuda), w.to(cuda), idx.to(cuda), z.gather(1, idx).float().to(cuda))
    p = torch.softmax(z, 1)
    # p: the sum's rounding and its exponentials'; q: expf, a sum of 200 and two products; both relative
    rel = (128 + V / 64 + 16 + 200 + 5 * (z - z.amax(1, keepdim=True)).abs()) * U
    near(r.dx, torch.zeros(n, d, dtype=torch.float64), (p * rel) @ w.double().abs() + 1e-30, "dx")
    near(r.dw, torch.zeros(V, d, dtype=torch.float64), (p * rel).t() @ x.double().abs() + 1e-30, "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", [1, 40, 300])
def test_gradients_of_confident_rows(cuda, dtype, n):
    """Rows sure of their label: D at the label is -(1 - p) to its own size, not to that of 1."""
    d, V = 520, 700
    x, w, y, _ = make(n, d, V, dtype, cuda)
    x = (x.float() + 2.5 * w[y].float()).to(dtype)
    z = (x.double() @ w.double().t()).cpu()
    az = x.double().abs().cpu() @ w.double().abs().t().cpu()
    ez = ((6 * d + 20 if dtype == torch.float32 else d + 12) * U * az).amax(1, keepdim=True)
    D = torch.softmax(z, 1)
    at = y.cpu()[:, None]
    rest = D.scatter(1, at, 0.0).sum(1, keepdim=True)
    D.scatter_(1, at, -rest)
    assert float(rest.median()) < 0.05
    r = head.softmax_head_loss(x, w, y)
    span = (z - z.amax(1, keepdim=True)).abs().clamp(max=150)
    # p and 1 - p are off by twice a score's error and the sum's, E by 2^-11 and D by 2^-8 on bf16 inputs
    rel = torch.expm1(2 * ez + (128 + V / 64 + 32 + 3 * span) * U) + (2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11 + H)
    aD = D.abs() * (rel + (6 * V + 16 if dtype == torch.float32 else V + 16) * U) + rest * 2.0 ** -32
    out = 2.0 ** -24 if dtype == torch.float32 else H
    dx = D @ w.double().cpu()
    near(r.dx, dx, aD @ w.double().abs().cpu() + 1.01 * out * (dx.abs() + aD @ w.double().abs().cpu()) + 1e-38, "dx")
