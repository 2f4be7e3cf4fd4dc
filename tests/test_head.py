"""Class head over many classes (csrc/hip/head.hip, ops/head.py) against plain formulas in 64 bits.

Tolerances are bounds by arithmetic, element by element, with u = 2^-24 (fp32), h = 2^-8 (bf16 rounding):

* a score is a sum of d products (bf16: exact in fp32; fp32: six plane products each, operands cut below
  2^-26) accumulated in fp32:  |dz| <= c u sum |x||w| (+ a few u of |z|), c = d + 8 (bf16), 6 d + 16 (fp32);
* lse of scores that are off by at most e is off by at most e, plus the rounding of its sum (the groups are added
  in fp32) and of its own value;
* p = e^(z - lse) is off by the factor e^(|dz| + |dlse|), the exponential's own error (8 u; bf16 inputs:
  |z - m| 2^-24 log2 e and E's 2^-11), and D is rounded to bf16 on bf16 inputs (h |D|);
* a gradient product adds the error of D times |operand|, its own fp32 sums and the final rounding.
"""
import itertools

import pytest
import torch

from ytk_learn_amd.ops import head

U, H = 2.0 ** -24, 2.0 ** -8


class Ref:
    """Plain 64-bit loss and gradients with the bounds above."""

    def __init__(self, x, w, idx, q_of, bias=None, weight=None, T=1.0, base=False, live=None):
        x64, w64 = x.double().cpu(), w.double().cpu()
        fp32 = x.dtype == torch.float32
        n, d = x64.shape
        V = w64.shape[0]
        self.live = torch.ones(n, dtype=torch.bool) if live is None else live.cpu()
        x64 = torch.where(self.live[:, None], x64, torch.zeros_like(x64))
        z = x64 @ w64.t()
        az = x64.abs() @ w64.abs().t()
        if bias is not None:
            z = z + bias.double().cpu()
            az = az + bias.double().cpu().abs().nan_to_num(posinf=0.0, neginf=0.0)
        z, az = z / T, az / T
        ez = (((6 * d + 16) if fp32 else (d + 8)) * U + 4 * U) * az
        if base:
            z, ez = torch.cat([z, z.new_zeros(n, 1)], 1), torch.cat([ez, ez.new_zeros(n, 1)], 1)
        lse = torch.logsumexp(z, 1)
        sums = (64 + z.shape[1] / 64 + 64) * U  # additions in a group, over groups, exponentials
        elin = ez.amax(1) + sums + (z - z.amax(1, keepdim=True)).abs().nan_to_num(posinf=0.0).clamp(max=100).amax(1) * 2 * U
        self.lse, self.elin = lse, elin + 4 * U * lse.abs()
        g = torch.ones(n, dtype=torch.float64) if weight is None else weight.double().cpu()
        g = torch.where(self.live, g, torch.zeros_like(g))
        idx, q, logq = idx.cpu(), *q_of
        at = idx.clamp(min=0, max=z.shape[1] - 1)
        zt = z.gather(1, at)
        term = torch.where(q > 0, q * (logq - zt + lse[:, None]), torch.zeros_like(q)).sum(1)
        self.loss = torch.where(g != 0, g * T * T * term, torch.zeros_like(g))
        k = q.shape[1]
        eq = 16 * U * (1 + logq.abs().nan_to_num(posinf=0.0, neginf=0.0))  # relative, of q
        tt = torch.where(q > 0, (q * (ez.gather(1, at) + self.elin[:, None] + (8 + k) * U * (logq.abs() + zt.abs() + lse.abs()[:, None]))
                                 + eq * q * ((logq - zt + lse[:, None]).abs() + 1)), torch.zeros_like(q)).sum(1)
        self.eloss = g.abs() * T * T * tt + 4 * U * self.loss.abs() + 1e-30
        s = q.sum(1)
        p = (z - lse[:, None]).exp()
        D = ((p * s[:, None]).scatter_add(1, at, -q) * (g * T)[:, None])
        D = torch.where((g != 0)[:, None] & (s != 0)[:, None], D, torch.zeros_like(D))
        rel = ez + elin[:, None] + 32 * U + (0.0 if fp32 else 2.0 ** -11) + (z - z.amax(1, keepdim=True)).abs().clamp(max=150) * 3 * U
        rel = rel + (eq.amax(1) + k * U)[:, None]
        eD = p * s[:, None] * torch.expm1(rel.clamp(max=20)) + torch.zeros_like(p).scatter_add(1, at, q * (eq + k * U + 4 * U))
        eD = eD * (g * T).abs()[:, None] + (2.0 ** -40 if fp32 else 2.0 ** -38) * (g * T).abs()[:, None]
        eD = eD + (2.0 ** -22 if fp32 else H) * (D.abs() + eD)
        D, eD = D[:, :V], eD[:, :V]
        eD = torch.where((g != 0)[:, None], eD, torch.zeros_like(eD))
        out = U if fp32 else H
        terms = 6 if fp32 else 1
        aD = D.abs() + eD
        self.D = D
        self.dx = D @ w64
        self.edx = eD @ w64.abs() + (terms * V + 16) * U * (aD @ w64.abs()) + 2 * out * self.dx.abs() + 1e-38
        self.dw = D.t() @ x64
        self.edw = eD.t() @ x64.abs() + (terms * n + 16) * U * (aD.t() @ x64.abs()) + 2 * out * self.dw.abs() + 1e-38
        self.db = D.sum(0)
        self.edb = eD.sum(0) + (n + 8) * U * aD.sum(0) + 2 * out * self.db.abs() + 1e-38

    def check(self, r, dx=True, dw=True, db=False):
        near(r.lse[self.live.to(r.lse.device)], self.lse[self.live], self.elin[self.live], "lse")
        near(r.loss, self.loss, self.eloss, "loss")
        for name, want in (("dx", dx), ("dw", dw), ("db", db)):
            t = getattr(r, name)
            if not want:
                assert t is None, name
                continue
            near(t, getattr(self, name), getattr(self, "e" + name), name)


def near(got, ref, bound, name):
    got = got.double().cpu()
    assert got.shape == ref.shape, name
    same = (got == ref) | (got.isnan() & ref.isnan())
    bad = ~(same | ((got - ref).abs() <= bound))
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst "
                                 f"{float(((got - ref).abs() / bound)[bad].max()):.3g} times the bound")


def make(n, d, V, dtype, dev, seed=0, bias=False):
    g = torch.Generator().manual_seed(seed * 7919 + n * 31 + d * 7 + V)
    x = torch.randn(n, d, generator=g)
    w = torch.randn(V, d, generator=g) * (2.0 / d ** 0.5)
    y = (torch.rand(n, generator=g) ** 2 * V).long().clamp(max=V - 1)
    x = x + 3 * torch.rand(n, 1, generator=g) * w[y]
    b = (torch.randn(V, generator=g) * 0.5).to(dtype).to(dev) if bias else None
    return x.to(dtype).to(dev), w.to(dtype).to(dev), y.to(dev), b


def label_targets(labels, live=None):
    q = torch.ones(labels.shape[0], 1, dtype=torch.float64)
    if live is not None:
        q = q * live.cpu().double()[:, None]
    return labels[:, None], (q, torch.zeros_like(q))


def list_targets(idx, tl, T, tlse=None):
    idx, t = idx.cpu(), tl.double().cpu() / T
    t = torch.where(idx >= 0, t, torch.full_like(t, -float("inf")))
    norm = tlse.double().cpu() if tlse is not None else torch.logsumexp(t, 1)
    logq = t - torch.where(norm.isinf(), torch.zeros_like(norm), norm)[:, None]
    return logq.exp(), torch.where(idx >= 0, logq, torch.zeros_like(logq))


def lists(n, V, k, seed=0, ragged=True):
    g = torch.Generator().manual_seed(seed + n + V + k)
    idx = torch.randint(0, V, (n, k), generator=g)  # classes named twice among them
    tl = torch.randn(n, k, generator=g) * 2 + 3
    if ragged:
        idx = torch.where(torch.arange(k)[None] < torch.randint(0, k + 1, (n, 1), generator=g), idx, torch.full_like(idx, -1))
    return idx, tl


BOTH = [torch.float32, torch.bfloat16]
# one row, one class, one feature, sizes around the tiles (32, 64, 128, 256) and odd ones
SIZES = [(1, 1, 1), (1, 64, 2), (2, 3, 64), (3, 65, 65), (31, 64, 127), (64, 128, 129), (65, 200, 331), (130, 72, 256),
         (257, 64, 257), (300, 333, 500), (33, 520, 1009)]


# ------------------------------------------------------------------ CPU path
@pytest.mark.parametrize("dtype", BOTH)
def test_loss_cpu(dtype):
    x, w, y, b = make(17, 9, 13, dtype, "cpu", bias=True)
    live = torch.arange(17) % 5 != 0
    lab = torch.where(live, y, torch.full_like(y, -100))
    wt = torch.rand(17)
    r = head.softmax_head_loss(x, w, lab, bias=b, weight=wt)
    Ref(x, w, *label_targets(lab, live), bias=b, weight=wt, live=live).check(r, db=True)
    zb = torch.cat([x.double() @ w.double().t(), torch.zeros(17, 1, dtype=torch.float64)], 1)
    r = head.softmax_head_loss(x, w, torch.full((17,), 13), base_class=True, want_dx=False, want_dw=False)
    assert torch.allclose(r.loss.double(), torch.logsumexp(zb, 1), rtol=1e-6)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_cpu(tail):
    x, w, _, _ = make(12, 7, 20, torch.float32, "cpu")
    idx, tl = lists(12, 20, 6)
    tlse = torch.logsumexp(tl / 2, 1) + 0.1 if tail else None
    r = head.distill_head_loss(x, w, idx, tl, temperature=2.0, top_lse=tlse)
    Ref(x, w, idx, list_targets(idx, tl, 2.0, tlse), T=2.0).check(r)


def test_topk_cpu():
    x, w, _, b = make(5, 6, 30, torch.float32, "cpu", bias=True)
    w[7] = w[3]
    b[7] = b[3]
    v, c, l = head.head_topk(x, w, 30, bias=b)
    z = x.double() @ w.double().t() + b.double()
    assert torch.equal(c, z.sort(dim=1, descending=True, stable=True).indices)
    assert torch.allclose(l.double(), torch.logsumexp(z, 1), rtol=1e-6)
    assert bool(((c == 3).nonzero()[:, 1] + 1 == (c == 7).nonzero()[:, 1]).all())  # equal scores: the lower class first


def test_gradient_is_the_derivative():
    """Central differences of the CPU path's loss: fp32 outputs, so steps of 2^-8 on 64-bit-exact scores."""
    torch.manual_seed(0)
    x, w, y, b = make(4, 3, 6, torch.float32, "cpu", bias=True)
    idx, tl = lists(4, 6, 3, ragged=False)
    for f in (lambda x, w, b: head.softmax_head_loss(x, w, y, bias=b, weight=torch.tensor([1.0, 0.5, 2.0, 0.0])),
              lambda x, w, b: head.distill_head_loss(x, w, idx, tl, bias=b, temperature=2.0)):
        r = f(x, w, b)
        for t, grad in ((x, r.dx), (w, r.dw), (b, r.db)):
            for i in range(0, t.numel(), 2):
                step = 2.0 ** -8
                old = float(t.view(-1)[i])
                t.view(-1)[i] = old + step
                hi = f(x, w, b).loss.double().sum()
                t.view(-1)[i] = old - step
                lo = f(x, w, b).loss.double().sum()
                t.view(-1)[i] = old
                # third derivative of order |coefficient|^3 T^-1 <= ~64, losses rounded to 2^-24 of <= ~16 each
                assert abs(float((hi - lo) / (2 * step)) - float(grad.view(-1)[i])) < 64 * step ** 2 / 6 + 4 * 16 * U / step


def _refusals(dev):
    x, w, y, b = make(4, 8, 6, torch.float32, dev, bias=True)
    idx, tl = torch.zeros(4, 3, dtype=torch.int64, device=dev), torch.zeros(4, 3, device=dev)
    ce, di, tk = head.softmax_head_loss, head.distill_head_loss, head.head_topk
    return [
        (ValueError, lambda: ce(x[0], w, y)), (ValueError, lambda: ce(x, w[:, :7], y)), (TypeError, lambda: ce(x.half(), w.half(), y)),
        (TypeError, lambda: ce(x.bfloat16(), w, y)), (ValueError, lambda: ce(x, w, y[:3])), (ValueError, lambda: ce(x, w, y.float())),
        (ValueError, lambda: ce(x, w, y, bias=b[:5])), (ValueError, lambda: ce(x, w, y, bias=b.bfloat16())),
        (ValueError, lambda: ce(x, w, y, weight=torch.ones(5, device=dev))), (ValueError, lambda: ce(x, w, y, weight=y)),
        (ValueError, lambda: ce(x[:, :0], w[:, :0], y)), (ValueError, lambda: ce(x, w[:0], y)),
        (ValueError, lambda: di(x, w, idx[:3], tl[:3])), (ValueError, lambda: di(x, w, idx, tl[:, :2])),
        (ValueError, lambda: di(x, w, idx[:, :0], tl[:, :0])), (ValueError, lambda: di(x, w, idx, tl.bfloat16())),
        (TypeError, lambda: di(x, w, idx.float(), tl)), (ValueError, lambda: di(x, w, idx, tl, temperature=0.0)),
        (ValueError, lambda: di(x, w, idx, tl, temperature=float("nan"))), (ValueError, lambda: di(x, w, idx, tl, temperature=1e-30)), (ValueError, lambda: di(x, w, idx, tl, top_lse=tl)),
        (ValueError, lambda: di(x, w, idx.repeat(1, 100), tl.repeat(1, 100))),
        (ValueError, lambda: tk(x, w, 0)), (ValueError, lambda: tk(x, w, 7)), (ValueError, lambda: tk(x, w.repeat(100, 1), 257)),
        (ValueError, lambda: tk(x, w, 2, temperature=-1.0)),
    ]


def test_refusals_cpu():
    for i, (err, call) in enumerate(_refusals("cpu")):
        with pytest.raises(err):
            call()
            print("accepted:", i)


@pytest.mark.gpu
def test_refusals_gpu(cuda):
    for err, call in _refusals(cuda):
        with pytest.raises(err):
            call()
    x, w, y, _ = make(4, 8, 6, torch.float32, cuda)
    with pytest.raises(ValueError):
        head.softmax_head_loss(x, w.cpu(), y)
    with pytest.raises(ValueError):
        head.softmax_head_loss(x, w, y.cpu())


# ------------------------------------------------------------------ loss
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n,d,V", SIZES)
def test_loss_sizes(cuda, dtype, n, d, V):
    x, w, y, b = make(n, d, V, dtype, cuda, bias=n % 2 == 1)
    r = head.softmax_head_loss(x, w, y, bias=b)
    assert r.loss.dtype == r.lse.dtype == torch.float32 and r.dx.dtype == r.dw.dtype == dtype
    Ref(x, w, *label_targets(y), bias=b).check(r, db=b is not None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("want", list(itertools.product([False, True], repeat=2)))
def test_loss_parts(cuda, dtype, want):
    """Row weights, ignored rows, int32 labels, the class without weights; gradients one by one."""
    x, w, y, b = make(150, 96, 300, dtype, cuda, bias=True)
    y[::7] = 300  # the class without weights
    live = torch.arange(150, device=cuda) % 4 != 1
    wt = torch.rand(150, device=cuda) - 0.2
    lab = torch.where(live, y, torch.full_like(y, -7)).int()
    r = head.softmax_head_loss(x, w, lab, bias=b, weight=wt, ignore_index=-7, base_class=True, want_dx=want[0], want_dw=want[1])
    i, t = label_targets(y, live)
    Ref(x, w, i, t, bias=b, weight=wt, base=True, live=live).check(r, *want, db=want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
def test_loss_strides(cuda, dtype):
    """Transposed, pitched, offset, stepped, repeated operands give what contiguous ones give."""
    x, w, y, b = make(70, 64, 140, dtype, cuda, bias=True)
    whole = head.softmax_head_loss(x, w, y, bias=b)

    def pitched(t, by, off):
        p = torch.full((t.shape[0], t.shape[1] + by), float("nan"), dtype=dtype, device=cuda)
        p[:, off:off + t.shape[1]] = t
        return p[:, off:off + t.shape[1]]

    for x2, w2 in ((x.t().contiguous().t(), w), (x, w.t().contiguous().t()), (pitched(x, 64, 0), pitched(w, 8, 8)),
                   (pitched(x, 3, 1), pitched(w, 5, 2)), (x.repeat_interleave(2, 1)[:, ::2], w.repeat_interleave(3, 0)[::3])):
        r = head.softmax_head_loss(x2, w2, y, bias=b.repeat_interleave(2)[::2])
        for a, c in zip(r, whole):
            assert torch.equal(a, c)
    one = x[:1].expand(70, 64)
    r = head.softmax_head_loss(one, w, y)
    Ref(one, w, *label_targets(y)).check(r)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", [1, 5, 150])
def test_one_feature_of_any_stride(cuda, dtype, n):
    """The transposed view of a [1, V] weight matrix, and one column that repeats or skips memory."""
    x, w, y, b = make(n, 1, 90, dtype, cuda, bias=True)
    ref = Ref(x, w, *label_targets(y), bias=b)
    wt = w.as_strided((90, 1), (1, 90))
    for xs in (x, x.as_strided((n, 1), (1, 7)), x.as_strided((n, 1), (1, 0))):
        ref.check(head.softmax_head_loss(xs, wt, y, bias=b), db=True)
        assert torch.equal(head.head_topk(xs, wt, 3, bias=b)[1], head.head_topk(x, w, 3, bias=b)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", [5, 150, 300])
@pytest.mark.parametrize("d", [8, 72, 200])
def test_loss_rows_inside_a_wider_buffer(cuda, dtype, n, d):
    """What stands between the rows (NaN) stays out, also where a row ends inside a step of the product."""
    x, w, y, b = make(n, d, 333, dtype, cuda, bias=True)
    bx = torch.full((n + 1, d + 24), float("nan"), dtype=dtype, device=cuda)
    bw = torch.full((334, d + 8), float("nan"), dtype=dtype, device=cuda)
    bx[:n, :d], bw[:333, :d] = x, w
    for x2, w2 in ((bx[:n, :d], bw[:333, :d]), (x, bw[:333, :d]), (bx[:n, :d], w)):
        r = head.softmax_head_loss(x2, w2, y, bias=b)
        Ref(x, w, *label_targets(y), bias=b).check(r, db=True)
        v, c, _ = head.head_topk(x2, w2, 4, bias=b)
        assert torch.equal(c, topk_ref(x, w, b, 1.0, 4)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
def test_no_rows(cuda, dtype):
    x, w, y, b = make(3, 8, 5, dtype, cuda, bias=True)
    r = head.softmax_head_loss(x[:0], w, y[:0], bias=b)
    assert r.loss.shape == r.lse.shape == (0,) and r.dx.shape == (0, 8) and bool((r.dw == 0).all()) and bool((r.db == 0).all())
    r = head.distill_head_loss(x[:0], w, y[:0, None], torch.zeros(0, 1, device=cuda))
    assert r.dw.shape == (5, 8) and bool((r.dw == 0).all())
    v, c, l = head.head_topk(x[:0], w, 2)
    assert v.shape == c.shape == (0, 2) and l.shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 300001), (torch.float32, 150001)])
def test_weights_beyond_32_bit_offsets(cuda, dtype, V):
    """w of more than 2^32 bytes: every class's score and gradient, in 64 bits in pieces on the GPU."""
    d, n = 8192, 3
    g = torch.Generator(device=cuda).manual_seed(3)
    w = torch.empty(V, d, dtype=dtype, device=cuda)
    for a in range(0, V, 50000):
        w[a:a + 50000] = (torch.randn(min(50000, V - a), d, generator=g, device=cuda) * (2.0 / d ** 0.5)).to(dtype)
    x = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    y = torch.tensor([V - 1, 7, V // 2], device=cuda)
    r = head.softmax_head_loss(x, w, y)
    v, c, l = head.head_topk(x, w, 5)
    z = torch.cat([x.double() @ w[a:a + 20000].double().t() for a in range(0, V, 20000)], 1)
    lse = torch.logsumexp(z, 1)
    rv, rc = z.sort(dim=1, descending=True, stable=True)
    assert torch.equal(c, rc[:, :5])
    # |x||w| sums to at most ~ 2 d 2 / sqrt(d) = 362: scores off by (6 d + 32) 2^-24 * 362 at worst, in practice far less
    near(r.lse, lse.cpu(), torch.full((n,), 1e-3, dtype=torch.float64), "lse")
    near(r.loss, (lse - z.gather(1, y[:, None])[:, 0]).cpu(), torch.full((n,), 2e-3, dtype=torch.float64), "loss")
    D = (z - lse[:, None]).exp()
    D[torch.arange(n, device=cuda), y] -= 1
    step = 2 * (H if dtype == torch.bfloat16 else 2e-3)  # D's rounding, or the scores' bound
    dx = sum(D[:, a:a + 20000] @ w[a:a + 20000].double() for a in range(0, V, 20000))
    bound = sum(D[:, a:a + 20000].abs() @ w[a:a + 20000].double().abs() for a in range(0, V, 20000)) * step
    near(r.dx, dx.cpu(), bound.cpu(), "dx")
    for a in (0, 65500, 131040, V - 70):
        dw = D[:, a:a + 70].t() @ x.double()
        near(r.dw[a:a + 70], dw.cpu(), (step * (D[:, a:a + 70].abs().t() @ x.double().abs()) + 2 * H * dw.abs() + 1e-12).cpu(), "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
def test_loss_ignored_rows_hold_anything(cuda, dtype):
    x, w, y, _ = make(90, 64, 200, dtype, cuda)
    live = torch.arange(90, device=cuda) % 3 != 0
    x[~live] = float("nan")
    x[0] = float("inf")
    lab = torch.where(live, y, torch.full_like(y, -100))
    r = head.softmax_head_loss(x, w, lab)
    Ref(x, w, *label_targets(y, live), live=live).check(r)
    wt = live.float()  # the same rows by a weight of 0
    r2 = head.softmax_head_loss(x, w, y, weight=wt)
    assert torch.equal(r2.loss, r.loss) and torch.equal(r2.dx, r.dx) and torch.equal(r2.dw, r.dw)
    r = head.softmax_head_loss(x, w, torch.full_like(y, -100), bias=torch.zeros(200, dtype=dtype, device=cuda))
    for t in (r.loss, r.dx, r.dw, r.db):
        assert bool((t == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("low", ["-inf", "lowest"])
def test_loss_masked_classes(cuda, dtype, low):
    """Classes switched off by a bias of -inf or the type's lowest value, whole groups of 64 among them."""
    x, w, y, _ = make(40, 64, 400, dtype, cuda)
    b = torch.zeros(400, dtype=dtype, device=cuda)
    off = torch.zeros(400, dtype=torch.bool, device=cuda)
    off[0:130] = True
    off[300::3] = True
    b[off] = float("-inf") if low == "-inf" else torch.finfo(dtype).min
    y = torch.where(off[y], torch.full_like(y, 200), y)
    r = head.softmax_head_loss(x, w, y, bias=b)
    keep = ~off
    at = torch.cumsum(keep, 0)[y] - 1
    sub = Ref(x, w[keep], *label_targets(at))
    near(r.loss, sub.loss, sub.eloss, "loss")
    near(r.dx, sub.dx, sub.edx, "dx")
    near(r.dw[keep], sub.dw, sub.edw, "dw")
    assert bool((r.dw[off] == 0).all()) and bool((r.db[off] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
def test_loss_wrong_labels_and_nan(cuda, dtype):
    x, w, y, _ = make(12, 64, 100, dtype, cuda)
    good = head.softmax_head_loss(x, w, torch.where(torch.arange(12, device=cuda) < 4, torch.full_like(y, -100), y))
    bad = y.clone()
    bad[0], bad[1], bad[2], bad[3] = 100, -1, 1 << 40, -(1 << 40)
    r = head.softmax_head_loss(x, w, bad)
    assert bool(r.loss[:4].isnan().all()) and torch.equal(r.loss[4:], good.loss[4:])
    assert torch.equal(r.dw, good.dw) and bool((r.dx[:4] == 0).all())
    x[5, 3] = float("nan")
    r = head.softmax_head_loss(x, w, y)
    assert bool(r.loss[5].isnan()) and bool(r.dx[5].isnan().all()) and int(r.loss.isnan().sum()) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
def test_loss_pieces(cuda, dtype, monkeypatch):
    """Several pieces of rows (the last one short) against one; a small n of many classes splits K instead."""
    x, w, y, b = make(900, 136, 600, dtype, cuda, bias=True)
    wt = torch.rand(900, device=cuda)
    ref = Ref(x, w, *label_targets(y), bias=b, weight=wt)
    monkeypatch.setattr(head, "PIECE_BYTES", 1 << 10)
    r = head.softmax_head_loss(x, w, y, bias=b, weight=wt)
    ref.check(r, db=True)
    idx, tl = lists(900, 600, 70)
    r = head.distill_head_loss(x, w, idx.to(cuda), tl.to(cuda), bias=b)
    Ref(x, w, idx, list_targets(idx, tl, 1.0), bias=b).check(r, db=True)
    v, c, l = head.head_topk(x, w, 5, bias=b)
    monkeypatch.undo()
    v2, c2, l2 = head.head_topk(x, w, 5, bias=b)
    assert torch.equal(v, v2) and torch.equal(c, c2) and torch.equal(l, l2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n,d,V", [(torch.bfloat16, 1100, 512, 16500), (torch.bfloat16, 40, 1024, 20011),
                                         (torch.float32, 700, 640, 4100), (torch.bfloat16, 4097, 1160, 264), (torch.float32, 5, 1000, 20011),
                                         (torch.float32, 50, 1031, 9000), (torch.float32, 20, 64, 40000), (torch.bfloat16, 300, 1000, 5003)])
def test_loss_larger(cuda, dtype, n, d, V):
    """Large and small tiles, K split into runs, every XCD's share of the tile order, few fp32 rows, rows that end in a step."""
    x, w, y, b = make(n, d, V, dtype, cuda, bias=True)
    r = head.softmax_head_loss(x, w, y, bias=b)
    Ref(x, w, *label_targets(y), bias=b).check(r, db=True)
    again = head.softmax_head_loss(x, w, y, bias=b)
    for a, c in zip(r, again):
        assert torch.equal(a, c)  # bitwise reproducible


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", [1, 40, 300])
def test_loss_confident_rows(cuda, dtype, n):
    """Rows sure of their label: lse and the label's score share their error, so the loss is near 0 without the scores'
    rounding: |dloss| <= 2 (1 - p_y) max |dz| + the rounding of the sum (1 + small: 8 u) and of the log."""
    x, w, y, _ = make(n, 520, 700, dtype, cuda)
    x = (x.float() + 2.5 * w[y].float()).to(dtype)
    r = head.softmax_head_loss(x, w, y, want_dx=False, want_dw=n == 40)
    z = x.double() @ w.double().t()
    ref = torch.logsumexp(z, 1) - z.gather(1, y[:, None])[:, 0]
    ez = ((6 * 520 + 20 if dtype == torch.float32 else 520 + 12) * U * (x.double().abs() @ w.double().abs().t())).amax(1)
    assert float(ref.median()) < 0.05
    near(r.loss, ref.cpu(), (2 * (1 - (-ref).exp()) * ez + 8 * U + 16 * U * ref).cpu(), "loss")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
def test_loss_many_rows(cuda, dtype):
    """More rows than one piece holds at most, few classes."""
    n = (1 << 21) + 777
    x, w, y, b = make(n, 3, 4, dtype, cuda, bias=True)
    r = head.softmax_head_loss(x, w, y, bias=b)
    Ref(x, w, *label_targets(y), bias=b).check(r, db=True)
    v, c, _ = head.head_topk(x, w, 2, bias=b)
    assert torch.equal(c, topk_ref(x, w, b, 1.0, 2)[1])


# ------------------------------------------------------------------ distillation
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n,d,V,k", [(1, 1, 1, 1), (3, 65, 65, 2), (64, 64, 200, 64), (65, 130, 513, 65), (20, 64, 700, 256)])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_sizes(cuda, dtype, n, d, V, k, tail):
    x, w, _, b = make(n, d, V, dtype, cuda, bias=True)
    idx, tl = lists(n, V, k)
    T = 2.0 if k % 2 == 0 else 1.0
    tlse = torch.logsumexp(tl / T, 1) + 0.2 if tail else None
    wt = torch.rand(n) + 0.1
    r = head.distill_head_loss(x, w, idx.to(cuda).int() if k == 2 else idx.to(cuda), tl.to(cuda), bias=b, weight=wt.to(cuda),
                               temperature=T, top_lse=None if tlse is None else tlse.to(cuda))
    Ref(x, w, idx, list_targets(idx, tl, T, tlse), bias=b, weight=wt, T=T).check(r, db=True)


@pytest.mark.gpu
def test_distill_edges(cuda):
    """No entries, -inf teacher logits, a class named throughout, classes that do not exist."""
    x, w, _, _ = make(6, 64, 100, torch.float32, cuda)
    idx = torch.tensor([[-1, -1, -1], [5, 6, 7], [9, 9, 9], [1, 2, 3], [4, 100, 5], [98, 99, 0]])
    tl = torch.tensor([[0.0, 1.0, 2.0], [1.0, -float("inf"), 0.5], [0.0, 1.0, 2.0], [-float("inf")] * 3, [1.0, 1.0, 1.0], [3.0, 2.0, 1.0]])
    r = head.distill_head_loss(x, w, idx.to(cuda), tl.to(cuda))
    assert float(r.loss[0]) == 0.0 and float(r.loss[3]) == 0.0 and bool(r.loss[4].isnan())
    assert bool((r.dx[0] == 0).all()) and bool((r.dx[3] == 0).all())
    ok = [1, 2, 5]
    sub = head.distill_head_loss(x[ok].contiguous(), w, idx[ok].to(cuda), tl[ok].to(cuda))
    ref = Ref(x[ok], w, idx[ok], list_targets(idx[ok], tl[ok], 1.0))
    ref.check(sub)
    near(r.loss[ok], ref.loss, ref.eloss, "loss")
    one = head.softmax_head_loss(x[2:3].contiguous(), w, torch.tensor([9], device=cuda))
    q = torch.softmax(tl[2].double(), 0)  # one class named three times: the label's loss less the entropy of the split
    near(r.loss[2:3], one.loss.double().cpu() + (q * q.log()).sum(), ref.eloss[1:2] * 2, "split entry")


def _weightless(dev):
    """A weight of 0 takes a row out of every gradient, whatever its list and x hold; so does an entry -1 its logit."""
    nan, inf = float("nan"), float("inf")
    x, w, _, _ = make(5, 64, 100, torch.float32, dev)
    x[1], x[3] = nan, inf
    idx = torch.tensor([[1, 2, -1], [3, 4, 5], [6, -1, 7], [8, 9, 10], [11, 12, 13]])
    tl = torch.tensor([[1.0, 2.0, nan], [nan, 1.0, 2.0], [0.5, inf, 1.0], [inf, inf, 0.0], [nan, nan, nan]])
    g = torch.tensor([1.0, 0.0, 2.0, 0.0, 0.0])
    tlse = torch.tensor([3.0, nan, 3.0, inf, nan])
    ok = [0, 2]
    for t in (None, tlse):
        r = head.distill_head_loss(x, w, idx.to(dev), tl.to(dev), weight=g.to(dev), top_lse=None if t is None else t.to(dev))
        assert bool((r.loss[[1, 3, 4]] == 0).all()) and bool((r.dx[[1, 3, 4]] == 0).all())
        ref = Ref(x[ok], w, idx[ok], list_targets(idx[ok], tl[ok], 1.0, None if t is None else t[ok]), weight=g[ok])
        ref.check(head.HeadLoss(r.loss[ok], r.lse[ok], r.dx[ok], r.dw, None))


def test_distill_weightless_rows_cpu():
    _weightless("cpu")


@pytest.mark.gpu
def test_distill_weightless_rows_gpu(cuda):
    _weightless(cuda)


@pytest.mark.gpu
def test_distill_many_rows_with_long_lists(cuda):
    """As many list entries as one launch's threads: the rows go in pieces. Only the first and last rows have a weight."""
    n, k, V, T = (1 << 20) + 777, 256, 40, 1.5
    x, w, _, b = make(n, 3, V, torch.float32, cuda, bias=True)
    at = torch.cat([torch.arange(150), torch.arange(n - 150, n)])
    g = torch.zeros(n, device=cuda)
    g[at.to(cuda)] = 1.0
    idx = torch.full((n, k), -1, dtype=torch.int32, device=cuda)
    tl = torch.zeros((n, k), device=cuda)
    i, t = lists(len(at), V, k)
    idx[at.to(cuda)], tl[at.to(cuda)] = i.int().to(cuda), t.to(cuda)
    r = head.distill_head_loss(x, w, idx, tl, bias=b, weight=g, temperature=T)
    assert int((r.loss != 0).sum()) <= len(at) and int((r.dx != 0).any(1).sum()) <= len(at)
    at = at.to(cuda)
    Ref(x[at], w, i, list_targets(i, t, T), bias=b, T=T).check(head.HeadLoss(r.loss[at], r.lse[at], r.dx[at], r.dw, r.db), db=True)


# ------------------------------------------------------------------ top k
def topk_ref(x, w, bias, T, k):
    z = x.double() @ w.double().t()
    if bias is not None:
        z = z + bias.double()
    z = z / T
    v, c = z.sort(dim=1, descending=True, stable=True)
    return v[:, :k], c[:, :k], torch.logsumexp(z, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n,d,V,k", [(1, 1, 1, 1), (1, 64, 70, 70), (2, 33, 129, 1), (7, 333, 2003, 5), (33, 64, 640, 9), (65, 128, 5000, 64),
                                     (3, 64, 30000, 256), (130, 200, 300, 256), (1, 512, 40001, 16), (5, 64, 1500, 256),
                                     (260, 64, 150001, 7), (2, 16, 600000, 30)])
def test_topk_sizes(cuda, dtype, n, d, V, k):
    x, w, _, b = make(n, d, V, dtype, cuda, bias=k % 2 == 1)
    T = 1.5 if n % 2 else 1.0
    v, c, l = head.head_topk(x, w, k, bias=b, temperature=T)
    rv, rc, rl = topk_ref(x, w, b, T, k)
    assert torch.equal(c, rc)
    # values: the 64-bit sums rounded once (1 / T multiplies: one more 64-bit rounding)
    near(v, rv.cpu(), (1.01 * U * rv.abs()).cpu() + 1e-40, "values")
    az = (x.double().abs() @ w.double().abs().t()).amax(1) + (0 if b is None else b.double().abs().max())
    near(l, rl.cpu(), (((6 * d + 32) * az / T + 200 + 8 * rl.abs() + V / 64) * U).cpu(), "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
def test_topk_ties_and_masks(cuda, dtype):
    x, w, _, _ = make(9, 64, 3000, dtype, cuda)
    w[100::7] = w[3]                # hundreds of equal scores
    b = torch.zeros(3000, dtype=dtype, device=cuda)
    b[1::2] = float("-inf")
    v, c, _ = head.head_topk(x, w, 200, bias=b)
    rv, rc, _ = topk_ref(x, w, b, 1.0, 200)
    assert torch.equal(c, rc)
    b[:] = float("-inf")
    b[17] = 0
    v, c, l = head.head_topk(x, w, 4, bias=b)
    assert c[:, 0].tolist() == [17] * 9 and c[:, 1:].tolist() == [[0, 1, 2]] * 9 and bool((v[:, 1:] == -float("inf")).all())
    z = torch.zeros_like(w)
    v, c, l = head.head_topk(x, z, 256)
    assert c.tolist() == [list(range(256))] * 9 and bool((v == 0).all())
    near(l, torch.full((9,), 3000.0, dtype=torch.float64).log(), torch.full((9,), 64 * U * 8, dtype=torch.float64), "lse")


@pytest.mark.gpu
def test_topk_nan_rows_stay_in_range(cuda):
    x, w, _, _ = make(5, 64, 1000, torch.bfloat16, cuda)
    good = head.head_topk(x, w, 20)
    x[2] = float("nan")
    w2 = w.clone()
    v, c, l = head.head_topk(x, w2, 20)
    assert bool(((c >= 0) & (c < 1000)).all()) and bool(l[2].isnan())
    assert all(len(set(r)) == 20 for r in c.tolist())
    rest = [0, 1, 3, 4]
    assert torch.equal(c[rest], good[1][rest]) and torch.equal(l[rest], good[2][rest])


# ------------------------------------------------------------------ as a program uses them
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
def test_teacher_to_student(cuda, dtype):
    """A teacher's top k written down, a student's step on it and on the labels, the student's answers."""
    xt, wt, y, b = make(200, 128, 1000, dtype, cuda, bias=True)
    v, c, _ = head.head_topk(xt, wt, 32, bias=b)
    _, _, lse2 = head.head_topk(xt, wt, 1, bias=b, temperature=2.0)
    xs, ws, _, _ = make(200, 64, 1000, dtype, cuda, seed=1)
    d = head.distill_head_loss(xs, ws, c, v, temperature=2.0, top_lse=lse2)
    Ref(xs, ws, c, list_targets(c, v, 2.0, lse2), T=2.0).check(d)
    s = head.softmax_head_loss(xs, ws, y)
    Ref(xs, ws, *label_targets(y)).check(s)
    ws2 = ws - 0.01 * (d.dw + s.dw)
    _, got, _ = head.head_topk(xs, ws2, 3)
    assert torch.equal(got, topk_ref(xs, ws2, None, 1.0, 3)[1])


@pytest.mark.gpu
def test_streams(cuda):
    """Two streams at once, each with its own operands."""
    sets = [make(300, 128, 2000, torch.bfloat16, cuda, seed=i) for i in range(2)]
    want = [head.softmax_head_loss(x, w, y) for x, w, y, _ in sets]
    top = [head.head_topk(x, w, 8) for x, w, _, _ in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for (x, w, y, _), st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append((head.softmax_head_loss(x, w, y), head.head_topk(x, w, 8)))
        torch.cuda.synchronize()
        for (a, t), b, u in zip(got, want, top):
            assert all(torch.equal(p, q) for p, q in zip(a, b) if p is not None)
            assert all(torch.equal(p, q) for p, q in zip(t, u))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BOTH)
def test_graph(cuda, dtype):
    """Captured once, replayed on new inputs between eager calls."""
    x, w, y, b = make(130, 72, 333, dtype, cuda, bias=True)
    idx, tl = (t.to(cuda) for t in lists(130, 333, 8))

    def step():
        return (*head.softmax_head_loss(x, w, y, bias=b), *head.distill_head_loss(x, w, idx, tl, bias=b, temperature=2.0),
                *head.head_topk(x, w, 9, bias=b))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        nx, nw, ny, nb = make(130, 72, 333, dtype, cuda, seed=i + 3, bias=True)
        x.copy_(nx), w.copy_(nw), y.copy_(ny), b.copy_(nb)
        g.replay()
        want = step()
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c)


# ------------------------------------------------------------------ the multiclass linear model on dense rows
def _train_dense(tmp, dev, K, dense, **kw):
    import os

    import numpy as np
    from ytk_learn_amd.config.hocon import parse_file
    from ytk_learn_amd.parallel.comm import Comm
    from ytk_learn_amd.train import train

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    rng = np.random.default_rng(7)
    W = rng.normal(size=(12, K))
    os.makedirs(tmp, exist_ok=True)
    for name, n in (("tr", 400), ("te", 90)):
        x = rng.random((n, 12)).round(4)
        y = (x @ W).argmax(1)
        with open(f"{tmp}/{name}.txt", "w") as f:
            for i in range(n):
                keep = [j for j in range(12) if (i + j) % 5]  # absent features are zeros
                f.write("%g###%d###%s\n" % (1 + i % 3, y[i], ",".join(f"{j}:{x[i, j]:.4f}" for j in keep)))
    ov = {"data.train.data_path": f"{tmp}/tr.txt", "data.test.data_path": f"{tmp}/te.txt", "model.data_path": f"{tmp}/m", "k": K,
          "loss.evaluate_metric": [], "optimization.line_search.lbfgs.convergence.max_iter": 6, "dense_head": dense}
    ov.update(kw)
    c = parse_file(os.path.join(root, "config", "model", "multiclass_linear.conf")).with_overrides(ov)
    return train("multiclass_linear", c, comm=Comm.local(dev))


def _dense_gradient(dev, K):
    """The model's loss and gradient on rows with absent and repeated features."""
    from types import SimpleNamespace

    from ytk_learn_amd.models.continuous.multiclass import MulticlassLinearModel, class_ids, dense_rows
    from ytk_learn_amd.ops.sparse import SparseMatrix

    g = torch.Generator().manual_seed(K)
    n, F = 150, 12
    count = torch.randint(0, 6, (n,), generator=g)
    indptr = torch.cat([torch.zeros(1, dtype=torch.int64), count.cumsum(0)])
    cols = torch.randint(0, F, (int(indptr[-1]),), generator=g, dtype=torch.int32)
    vals = torch.rand(int(indptr[-1]), generator=g)
    y = torch.randint(0, K, (n,), generator=g)
    X = SparseMatrix(indptr.to(dev), cols.to(dev), vals.to(dev), F)
    x = torch.zeros(n, F, dtype=torch.float64)
    x.index_put_((torch.repeat_interleave(torch.arange(n), count), cols.long()), vals.double(), accumulate=True)
    onehot = torch.nn.functional.one_hot(y, K).float().to(dev)
    W = torch.randn(F, K - 1, generator=g).to(dev)
    wt = torch.rand(n, generator=g).to(dev)
    m = MulticlassLinearModel.__new__(MulticlassLinearModel)
    m.F, m.S, m.dense = F, K - 1, {"train": (dense_rows(X), class_ids(onehot))}
    # a repeated feature's values are summed in fp32: exact operands for the reference are the rows the model holds
    near(m.dense["train"][0], x, 8 * U * x.abs(), "rows")
    out = torch.empty(F * (K - 1), device=dev)
    loss, pred = m._forward(X, SimpleNamespace(weight=wt), W.view(-1), out, "train")
    ref = Ref(m.dense["train"][0], W.t(), *label_targets(y), weight=wt, base=True)
    assert pred is None and abs(loss - float(ref.loss.sum())) <= float(ref.eloss.sum())
    near(out.view(F, K - 1).t(), ref.dw, ref.edw, "gradient")
    loss2, _ = m._forward(X, SimpleNamespace(weight=wt), W.view(-1), None, "train")
    assert loss2 == loss


@pytest.mark.parametrize("K", [2, 70])
def test_dense_head_gradient_cpu(K):
    _dense_gradient("cpu", K)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [2, 70, 300])
def test_dense_head_gradient_gpu(cuda, K):
    _dense_gradient(cuda, K)


def test_dense_head_trains_cpu(tmp_path):
    r = _train_dense(str(tmp_path / "a"), "cpu", 70, True)
    assert r.loss > 0 and r.test_loss > 0


def test_dense_head_refusals(tmp_path):
    from ytk_learn_amd.utils.errors import YtkLearnError
    for kw in ({"loss.loss_function": "multiclass_hinge"}, {"loss.evaluate_metric": ["confusion_matrix"]}):
        with pytest.raises(YtkLearnError):
            _train_dense(str(tmp_path / "r"), "cpu", 5, True, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [3, 300])
def test_dense_head_trains_gpu(cuda, tmp_path, K):
    r = _train_dense(str(tmp_path / "b"), cuda, K, True)
    assert r.loss > 0 and r.test_loss > 0
