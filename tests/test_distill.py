"""A teacher's top log-probabilities and the distillation loss with its gradient, against
64-bit math: types, odd sizes, strides, masks, ties, padding, weights, refusals."""
import math

import pytest
import torch

from turbol_b200.ops.distill import distill_loss, distill_loss_grad, topk_logprobs

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]
TYPES = [torch.bfloat16, torch.float16, torch.float32]
INF, NAN = math.inf, math.nan
# half the smallest step of fp16; 32-bit exponentials below 2^-126 are zero
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}


def sum_error(V):
    """Relative error of a sum of exponentials over V logits in fp32: the exponential itself (2^-22), its argument (the
    difference, the factor and the product rounded, up to 30 in size where a term counts: 3 x 30 x 2^-24 x ln 2), and the
    additions, V / 256 at most one after the other and some 16 in the tree."""
    return 2.0 ** -24 * (4 + 63 + V / 256 + 16)


def rows(R, V, dtype, device, seed=0, pad=0, shift=0, spread=3.0):
    """[R, V] logits; pad: elements between the rows, shift: elements before the first."""
    g = torch.Generator().manual_seed(seed * 7 + R * 1000 + V)
    buf = (torch.randn(R * (V + pad) + shift, generator=g) * spread).to(dtype).to(device)
    return buf[shift:].view(R, V + pad)[:, :V]


# ------------------------------------------------------------------ the teacher's list
def check_top(x, k, T=1.0):
    logp, ids, lse = topk_logprobs(x, k, temperature=T)
    z = x.double()
    key = torch.where(z.isnan(), -INF, z) + 0.0
    want = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    assert ids.dtype == torch.int32 and torch.equal(ids.long(), want)
    e_lse = torch.logsumexp(z / T, 1)
    e = torch.log_softmax(z / T, 1).gather(1, want)  # (not z - lse: next to the lowest value lse has lost log V)
    e = torch.where(e_lse.isposinf()[:, None], torch.where(z.gather(1, want) == INF, NAN, -INF), e)
    e = torch.where(e_lse.isneginf()[:, None], -INF, torch.where(e_lse.isnan()[:, None], NAN, e))
    for y, w in ((lse, e_lse), (logp, e)):
        assert y.dtype == torch.float32
        fine = w.isfinite()
        assert torch.equal(y.isnan(), w.isnan()) and torch.equal(y[~fine & ~w.isnan()].double(), w[~fine & ~w.isnan()])
        over = (y.double() - w).abs()[fine] - (sum_error(x.shape[1]) + 2.0 ** -24 * w.abs()[fine])
        assert not (over > 0).any(), over.max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,k,pad,shift,T", [(1, 1, 1, 0, 0, 1.0), (3, 7, 7, 0, 1, 0.5), (2, 64, 1, 0, 0, 1.0),
                                               (5, 65, 64, 3, 2, 2.0), (7, 1000, 256, 0, 0, 1.0), (64, 1024, 20, 8, 0, 1.0),
                                               (9, 4099, 3, 0, 0, 0.7), (3, 50001, 100, 7, 5, 1.3), (130, 2053, 33, 0, 0, 1.0)])
def test_top_matches_64_bits(R, V, k, pad, shift, T, dtype, device):
    check_top(rows(R, V, dtype, device, pad=pad, shift=shift), k, T)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,k", [(1, 151936, 20), (3, 128256, 64), (37, 32003, 100), (300, 9001, 17), (700, 151936, 64),
                                   (1, 2 ** 20, 256), (2, 2 ** 20 - 3, 1), (9, 200001, 256), (5000, 130, 9)])
def test_top_of_large_rows(R, V, k, dtype):
    check_top(rows(R, V, dtype, "cuda:0"), k)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(5, 5), (333, 40), (4096, 256), (20011, 64)])
def test_top_of_special_rows(V, k, dtype, device):
    """Ties over the whole row, orders that put the largest side by side, masks of -inf and of the type's lowest value,
    zeros of both signs, infinities, NaN."""
    low = torch.finfo(dtype).min
    ramp = torch.linspace(-8, 8, V)
    x = torch.randn(16, V, generator=torch.Generator().manual_seed(V))
    x[0] = 1.25
    x[1], x[2] = ramp, ramp.flip(0)
    x[3] = (torch.arange(V) % 3).float()
    x[4] = -INF
    x[5] = low
    x[6], x[6, V // 2] = -INF, 0.5
    x[7], x[7, V - 1] = low, -2.0
    x[8] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)
    x[9, V // 3] = NAN
    x[10, V // 2] = INF
    x[11, ::2] = -INF
    x[12, : V // 2] = low
    x[13] = x[13].abs() * 1e-3 - 100
    x[14] = NAN
    x[15] = torch.finfo(dtype).max
    check_top(x.to(dtype).to(device), k)


@pytest.mark.parametrize("device", DEVICES)
def test_top_of_views(device):
    """The same row everywhere (stride 0), rows of a transposed batch, no rows."""
    x = rows(1, 777, torch.bfloat16, device)
    check_top(x.expand(9, 777), 12)
    y = rows(12, 500, torch.float32, device).view(4, 3, 500).transpose(0, 1)[1]
    assert y.stride(0) == 1500
    check_top(y, 7)
    logp, ids, lse = topk_logprobs(x[:0], 5)
    assert logp.shape == (0, 5) and ids.shape == (0, 5) and lse.shape == (0,)


@pytest.mark.parametrize("device", DEVICES)
def test_top_refusals(device):
    x = rows(3, 100, torch.float32, device)
    for bad in (lambda: topk_logprobs(x, 0), lambda: topk_logprobs(x, 101), lambda: topk_logprobs(x.repeat(1, 3), 257),
                lambda: topk_logprobs(x[0], 1), lambda: topk_logprobs(x.double(), 1), lambda: topk_logprobs(x.t(), 1),
                lambda: topk_logprobs(x, 1, temperature=0.0), lambda: topk_logprobs(x, 1, temperature=NAN),
                lambda: topk_logprobs(x, 1, temperature=-1.0), lambda: topk_logprobs(x.clone().requires_grad_(), 1),
                lambda: topk_logprobs(x[:, :0], 1),
                lambda: topk_logprobs(torch.zeros(1, device=device).expand(1, 2 ** 20 + 1), 1)):
        with pytest.raises(ValueError, match="topk_logprobs"):
            bad()
    with torch.no_grad():
        topk_logprobs(x.clone().requires_grad_(), 1)


# ------------------------------------------------------------------ the loss
def lists(x, K, seed=0, T=1.0, noise=1.5):
    """A teacher near the student: ids and log-probabilities of its K largest."""
    g = torch.Generator().manual_seed(seed + 99)
    t = torch.nan_to_num(x.cpu().double(), neginf=-30.0, posinf=30.0).clamp(-30, 30)
    t = (t + noise * torch.randn(x.shape, generator=g)) / T
    top, ids = torch.topk(t, K, dim=1)
    return ids.int().to(x.device), (top - torch.logsumexp(t, 1, keepdim=True)).float().to(x.device)


def definition(x, ids, logp, w, kind, rest, T, y, c):
    """(loss, gradient, scale of the errors [R, V], factor of the loss's) in 64 bits, row by row from the classes."""
    R, V = x.shape
    loss, grads, mags, facs = [], [], [], []
    for r in range(R):
        z = x[r].cpu().double().requires_grad_()
        wr = 1.0 if w is None else float(w[r])
        yr = -1 if y is None else int(y[r])
        cr = 0.0 if yr < 0 or yr >= V else 1.0 if c is None else float(c[r])
        if wr == 0 and cr == 0:
            loss.append(0.0), grads.append(torch.zeros(V)), mags.append(torch.zeros(V)), facs.append(0.0)
            continue
        lp = torch.log_softmax(z / T, 0)
        t = {}
        for a, l in zip(ids[r].tolist(), logp[r].tolist()):
            if 0 <= a < V and l > -INF:
                t[a] = t.get(a, 0.0) + math.exp(l)
        at = torch.tensor(sorted(t), dtype=torch.long)
        tv = torch.tensor([t[a] for a in sorted(t)], dtype=torch.float64)
        total = float(tv.sum())
        kl, F = z.new_zeros(()), 0.0
        outside = torch.ones(V, dtype=torch.bool)
        outside[at] = False
        p_rest = float(lp.detach()[outside].exp().sum())
        if wr != 0:
            if not rest:
                if total > 0:
                    tv = tv / total
                    kl = (tv * (tv.log() - lp[at])).sum()
            else:
                lr = torch.logsumexp(lp[outside], 0) if outside.any() and float(x[r].cpu()[outside].max()) > -INF else None
                if kind == "forward":
                    kl = (tv * (tv.log() - lp[at])).sum()
                    tr = max(0.0, 1 - total)
                    if lr is not None and tr > 0:
                        kl = kl + tr * (math.log(tr) - lr)
                else:
                    on = lp[at] > -INF
                    kl = (lp[at][on].exp() * (lp[at][on] - tv[on].log())).sum()
                    if lr is not None:
                        kl = kl + lr.exp() * (lr - math.log(max(1 - total, 2.0 ** -20)))
                        F = abs(float(lr.detach()) - math.log(max(1 - total, 2.0 ** -20)))
            f = (lp.detach()[at] - tv.log()).abs()
            F = max([F] + f[f.isfinite()].tolist())
        whole = wr * kl + (cr * -lp[yr] if cr != 0 else 0.0)
        if whole.requires_grad:
            d, = torch.autograd.grad(whole, z)
        else:
            d = torch.zeros(V, dtype=torch.float64)
        p = lp.detach().exp()
        mag = p + torch.where(outside, p / max(p_rest, 1e-300), 0.0)
        mag[at] += tv
        if cr != 0:
            mag[yr] += 1
        loss.append(float(whole.detach())), grads.append(d)
        mags.append(mag * (2 + F) * (abs(wr) + abs(cr)) / T), facs.append((2 + F) * (abs(wr) + abs(cr)))
    return (torch.tensor(loss, dtype=torch.float64), torch.stack([g.double() for g in grads]),
            torch.stack([m.double() for m in mags]), torch.tensor(facs, dtype=torch.float64))


def compare(loss, d, x, want, g=None):
    """The loss's terms are off by the logarithms' errors (the sum's, and 2^-23 for the numbers kept in 32 bits), with the
    classes' log-ratios (F) as factor; the gradient's factors by the same and by the exponential's argument (up to 30
    where it counts), then one rounding."""
    e, ed, mag, fac = want
    delta = sum_error(x.shape[1]) + 2.0 ** -23
    l = loss.detach().cpu().double()
    assert loss.dtype == torch.float32 and torch.equal(l.isnan(), e.isnan())
    fine = e.isfinite()
    assert torch.equal(l[~fine & ~e.isnan()], e[~fine & ~e.isnan()])
    over = (l - e).abs()[fine] - (4 * delta * fac[fine] + 2.0 ** -23 * e.abs()[fine])
    assert not (over > 0).any(), over.max()
    if d is None:
        return
    assert d.dtype == x.dtype
    if g is not None:
        ed, mag = ed * g.cpu().double()[:, None], mag * g.cpu().double().abs()[:, None]
    dd = d.detach().cpu().double()
    assert torch.equal(dd.isnan(), ed.isnan())
    tol = torch.finfo(x.dtype).eps / 2 * 1.001 * ed.abs() + 8 * (delta + 2.0 ** -22 * 31) * mag + TINY[x.dtype]
    over = ((dd - ed).abs() - tol)[~ed.isnan()]
    assert not (over > 0).any(), over.max()


def run_both(x, ids, logp, w, kind, rest, T, y, c):
    """The fused form, its in-place form and the differentiable one against the definition."""
    want = definition(x, ids, logp, w, kind, rest, T, y, c)
    how = dict(kind=kind, rest=rest, temperature=T, target=y, target_weight=c)
    loss, d = distill_loss_grad(x, ids, logp, w, **how)
    compare(loss, d, x, want)
    # (the order of a row's sum follows its alignment: the same bits for the same layout)
    x = x.clone()
    loss, d = distill_loss_grad(x, ids, logp, w, **how)
    z = x.clone()
    l2, out = distill_loss_grad(z, ids, logp, w, out=z, **how)
    assert out is z and torch.equal(l2, loss) and torch.equal(z.nan_to_num(7.0), d.nan_to_num(7.0))
    leaf = x.detach().clone().requires_grad_()
    l3 = distill_loss(leaf, ids, logp, w, **how)
    # (the loss alone may be summed in another order: compared with the definition below)
    assert torch.equal(distill_loss(x, ids, logp, w, **how).nan_to_num(7.0), l3.detach().nan_to_num(7.0))
    g = torch.rand(x.shape[0], generator=torch.Generator().manual_seed(1)).to(x.device) + 0.5
    d3, = torch.autograd.grad(l3, leaf, g)
    compare(l3, d3, x, want, g)
    return loss, d


KINDS = [("forward", True), ("forward", False), ("reverse", True)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind,rest", KINDS)
@pytest.mark.parametrize("R,V,K,pad,shift,T,label", [(1, 1, 1, 0, 0, 1.0, False), (3, 7, 7, 0, 1, 0.5, True), (5, 65, 64, 3, 0, 2.0, False),
                                                     (4, 1024, 16, 0, 0, 1.0, True), (7, 1001, 256, 5, 3, 1.0, True),
                                                     (2, 20011, 50, 0, 0, 1.5, False)])
def test_loss_matches_64_bits(R, V, K, pad, shift, T, label, kind, rest, dtype, device):
    x = rows(R, V, dtype, device, pad=pad, shift=shift)
    ids, logp = lists(x, K, T=T)
    g = torch.Generator().manual_seed(5)
    w = torch.randn(R, generator=g).to(device) if label else None
    y = torch.randint(0, V, (R,), generator=g).int().to(device) if label else None
    c = torch.randn(R, generator=g).to(device) if label else None
    run_both(x, ids, logp, w, kind, rest, T, y, c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind,rest", KINDS)
@pytest.mark.parametrize("R,V,K", [(1, 151936, 64), (3, 128256, 32), (5, 200001, 100), (1, 2 ** 20, 20), (2, 2 ** 20 - 3, 256)])
def test_loss_of_large_rows(R, V, K, kind, rest, dtype):
    x = rows(R, V, dtype, "cuda:0")
    ids, logp = lists(x, K)
    y = torch.arange(R).int().cuda() * 7
    run_both(x, ids, logp, None, kind, rest, 1.0, y, torch.linspace(-1, 1, R).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,rest", KINDS)
def test_many_rows(kind, rest):
    """More rows than the machine holds at once, of different weights, against the host's math."""
    R, V, K = 1500, 9001, 30
    x = rows(R, V, torch.bfloat16, "cuda:0")
    ids, logp = lists(x, K)
    w = (torch.arange(R) % 3).float().cuda() - 0.5 * (torch.arange(R) % 3 != 0).float().cuda()
    loss, d = distill_loss_grad(x, ids, logp, w, kind=kind, rest=rest)
    cl, cd = distill_loss_grad(x.cpu(), ids.cpu(), logp.cpu(), w.cpu(), kind=kind, rest=rest)
    # two results, each as exact as the definition asks (log-ratios below 40): twice its bounds
    assert ((loss.cpu() - cl).abs() <= 2 * (4 * (sum_error(V) + 2.0 ** -23) * 42 * 1.5 + 2.0 ** -23 * cl.abs())).all()
    tol = 2.0 ** -8 * 1.001 * 2 * cd.double().abs() + 16 * (sum_error(V) + 2.0 ** -22 * 32) * 42 * 1.5
    assert ((d.cpu().double() - cd.double()).abs() <= tol).all()
    assert not d[w == 0].any() and not loss[w == 0].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind,rest", KINDS)
def test_padding_and_masks(kind, rest, dtype, device):
    """Entries without a meaning, ids that occur twice, a list of nothing, rows without weight that hold NaN, logits of
    -inf and of the type's lowest value in and outside the list, a list that covers the vocabulary."""
    R, V, K = 12, 300, 12
    x = rows(R, V, dtype, "cpu", seed=3)
    low = torch.finfo(dtype).min
    ids, logp = lists(x, K)
    ids, logp = ids.clone(), logp.clone()
    ids[0, 3:] = -1
    logp[1, 5:] = -INF
    ids[2, 4] = ids[2, 1]
    ids[3] = ids[3, 0]
    logp[3] = math.log(0.05)
    ids[4] = -1
    x[5, :] = NAN
    x[6, ::2] = -INF
    x[7, 100:] = low
    inside = torch.zeros(V, dtype=torch.bool)
    inside[ids[8].long()] = True
    x[8, ~inside] = -INF
    x[9, ids[9, 2].long()] = -INF
    x[10] = NAN
    x[11] = -INF
    w, c = torch.ones(R), torch.full((R,), 0.5)
    y = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(8)).int()
    y[2], y[6], y[7], y[8] = ids[2, 1], 1, 3, ids[8, 0]
    w[5] = c[5] = 0
    y[4] = -1
    w[0], c[1] = 0, 0
    args = [t.to(device) for t in (x, ids, logp, w, y, c)]
    x, ids, logp, w, y, c = args
    want = definition(x, ids, logp, w, kind, rest, 1.0, y, c)
    assert want[0][10:].isnan().all() and not want[0][:10].isnan().any()
    loss, d = distill_loss_grad(x, ids, logp, w, kind=kind, rest=rest, target=y, target_weight=c)
    compare(loss, d, x, want)
    assert not d[5].any() and float(loss[5]) == 0
    leaf = x.detach().clone().requires_grad_()
    l = distill_loss(leaf, ids, logp, w, kind=kind, rest=rest, target=y, target_weight=c)
    g, = torch.autograd.grad(l, leaf, torch.ones_like(l))
    compare(l, g, x, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind,rest", KINDS)
def test_a_list_of_the_whole_vocabulary(kind, rest, device):
    """Nothing outside the list."""
    x = rows(4, 100, torch.float32, device)
    ids, logp = lists(x, 100)
    run_both(x, ids, logp, None, kind, rest, 1.0, None, None)


@pytest.mark.parametrize("device", DEVICES)
def test_ids_out_of_range(device):
    """Left out and told; in rows without weight nothing is looked at."""
    x = rows(4, 50, torch.float32, device)
    ids, logp = lists(x, 5)
    ok = distill_loss_grad(x, ids, logp)
    bad, dropped = ids.clone(), ids.clone()
    bad[1, 2], dropped[1, 2] = 50, -1
    err = torch.zeros(1, dtype=torch.int32, device=device)
    w = torch.tensor([1.0, 0, 1, 1], device=device)
    distill_loss_grad(x, bad, logp, w, error=err)
    assert int(err) == 0
    loss, d = distill_loss_grad(x, bad, logp, error=err)
    assert int(err) == 1
    want = distill_loss_grad(x, dropped, logp)
    assert torch.equal(loss, want[0]) and torch.equal(d, want[1]) and torch.equal(loss[2:], ok[0][2:])
    err.zero_()
    y = torch.tensor([3, 2 ** 31 - 1, -5, 7], dtype=torch.int32, device=device)
    loss, d = distill_loss_grad(x, ids, logp, target=y, error=err)
    assert int(err) == 1
    none = torch.tensor([3, -1, -1, 7], dtype=torch.int32, device=device)
    want = distill_loss_grad(x, ids, logp, target=none)
    assert torch.equal(loss, want[0]) and torch.equal(d, want[1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind,rest", KINDS)
def test_gradient_against_differences(kind, rest, device):
    """Central differences of the loss itself (fp32 logits): off by the loss's own error over the step, and the step
    squared times the third derivative (at most some 2 + F)."""
    x = rows(2, 40, torch.float32, device, spread=1.0)
    ids, logp = lists(x, 6, noise=0.5)
    leaf = x.clone().requires_grad_()
    distill_loss(leaf, ids, logp, kind=kind, rest=rest).sum().backward()
    F = float(definition(x, ids, logp, None, kind, rest, 1.0, None, None)[3].max())
    h = 2.0 ** -5
    for j in [int(ids[0, 0]), int(ids[1, 3]), 0, 39]:
        up, down = x.clone(), x.clone()
        up[:, j] += h
        down[:, j] -= h
        step = (up[:, j] - down[:, j]).double()
        n = (distill_loss(up, ids, logp, kind=kind, rest=rest).double() -
             distill_loss(down, ids, logp, kind=kind, rest=rest).double()) / step
        tol = 2 * (4 * (sum_error(40) + 2.0 ** -23) * F + 2.0 ** -22) / (2 * h) + 4 * h * h * F
        assert ((leaf.grad[:, j].double() - n).abs() <= tol).all()


@pytest.mark.parametrize("device", DEVICES)
def test_autograd(device):
    """A sum's broadcast gradient, views as leaves, no second derivative, other inputs refused, values needed later."""
    x = rows(5, 90, torch.bfloat16, device, pad=6)
    ids, logp = lists(x, 8)
    base = torch.randn(5, 90, device=device, dtype=torch.float32).requires_grad_()
    distill_loss(base.bfloat16(), ids, logp).mean().backward()
    _, d = distill_loss_grad(base.detach().bfloat16(), ids, logp, torch.full((5,), 0.2, device=device))
    assert torch.allclose(base.grad, d.float(), rtol=2.0 ** -7, atol=1e-6)
    leaf = x.clone().requires_grad_()
    loss = distill_loss(leaf, ids, logp).sum()
    with pytest.raises((RuntimeError, ValueError)):
        g, = torch.autograd.grad(loss, leaf, create_graph=True)
        torch.autograd.grad(g.float().sum(), leaf)
    for what in ({"weight": torch.ones(5, device=device).requires_grad_()},
                 {"target": ids[:, 0].contiguous(), "target_weight": torch.ones(5, device=device).requires_grad_()}):
        with pytest.raises(ValueError, match="gradient"):
            distill_loss(x.clone().requires_grad_(), ids, logp, **what)
    with pytest.raises(ValueError, match="gradient"):
        distill_loss(x.clone().requires_grad_(), ids, logp.clone().requires_grad_())
    with pytest.raises(ValueError, match="gradient"):
        distill_loss_grad(x.clone().requires_grad_(), ids, logp)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            distill_loss(torch.autograd.forward_ad.make_dual(x.float(), torch.ones(5, 90, device=device)), ids, logp)
    # logits overwritten between the passes
    leaf = torch.randn(5, 90, device=device).requires_grad_()
    z = leaf * 1.0
    loss = distill_loss(z, ids, logp)
    with torch.no_grad():
        distill_loss_grad(z, ids, logp, out=z)
    if device != "cpu":
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.sum().backward()


@pytest.mark.parametrize("device", DEVICES)
def test_loss_refusals(device):
    x = rows(3, 100, torch.float32, device)
    ids, logp = lists(x, 4)
    w, y = torch.ones(3, device=device), torch.zeros(3, dtype=torch.int32, device=device)
    for call in (distill_loss, distill_loss_grad):
        for bad in (lambda: call(x[0], ids, logp), lambda: call(x.double(), ids, logp), lambda: call(x.t(), ids, logp),
                    lambda: call(x, ids.long(), logp), lambda: call(x, ids[:2], logp), lambda: call(x, ids, logp.double()),
                    lambda: call(x, ids, logp[:, :3]), lambda: call(x, ids.t().contiguous().t(), logp),
                    lambda: call(x, ids[:, :0], logp[:, :0]), lambda: call(x, ids, logp, w[:2]),
                    lambda: call(x, ids, logp, w.double()), lambda: call(x, ids, logp, kind="sideways"),
                    lambda: call(x, ids, logp, kind="reverse", rest=False), lambda: call(x, ids, logp, temperature=0.0),
                    lambda: call(x, ids, logp, temperature=INF), lambda: call(x, ids, logp, target=y.long()),
                    lambda: call(x, ids, logp, target_weight=w), lambda: call(x, ids, logp, target=y, target_weight=w[:1]),
                    lambda: call(x, ids.repeat(1, 65), logp.repeat(1, 65)), lambda: call(x, ids, logp, error=w)):
            with pytest.raises(ValueError, match="distill_loss"):
                bad()
    for out in (x[:2], x.bfloat16(), x.flip(1).t().contiguous().t(), x[:, :1].expand(3, 100),
                torch.empty(3, 200, device=device)[:, ::2]):
        with pytest.raises(ValueError, match="distill_loss_grad"):
            distill_loss_grad(x, ids, logp, out=out)
    buf = torch.empty(500, device=device)
    with pytest.raises(ValueError, match="overlap"):
        distill_loss_grad(buf[:300].view(3, 100), ids, logp, out=buf[100:400].view(3, 100))
    with pytest.raises(ValueError, match="overlap"):
        distill_loss_grad(x, ids, logp, buf[2:5], out=buf[:300].view(3, 100))
    loss, d = distill_loss_grad(x[:0], ids[:0], logp[:0])
    assert loss.shape == (0,) and d.shape == (0, 100)


@pytest.mark.gpu
def test_devices_are_not_mixed(dev):
    x = rows(3, 100, torch.float32, dev)
    ids, logp = lists(x, 4)
    for bad in (lambda: distill_loss(x, ids.cpu(), logp), lambda: distill_loss(x, ids, logp.cpu()),
                lambda: distill_loss(x, ids, logp, torch.ones(3)), lambda: distill_loss(x.cpu(), ids, logp),
                lambda: distill_loss_grad(x, ids, logp, out=x.cpu())):
        with pytest.raises(ValueError, match="one device"):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad,shift,opad,oshift", [(0, 0, 0, 0), (5, 0, 0, 1), (8, 3, 16, 0), (1, 1, 2, 7)])
def test_outputs_of_other_layouts(dtype, pad, shift, opad, oshift):
    """The gradient written to rows of another stride and alignment; what lies between the rows stays."""
    R, V = 9, 1003
    x = rows(R, V, dtype, "cuda:0", pad=pad, shift=shift)
    ids, logp = lists(x, 20)
    want = distill_loss_grad(x.contiguous(), ids, logp)
    buf = torch.full((R * (V + opad) + oshift + 16,), 3.0, dtype=dtype, device="cuda:0")
    out = buf[oshift:oshift + R * (V + opad)].view(R, V + opad)[:, :V]
    loss, d = distill_loss_grad(x, ids, logp, out=out)
    # (the order of a row's sum follows its alignment)
    tol = 2 * 8 * (sum_error(V) + 2.0 ** -22 * 32) * 20
    assert torch.allclose(loss, want[0], rtol=0, atol=8 * sum_error(V) * 20)
    assert torch.allclose(d.float(), want[1].float(), rtol=2 * torch.finfo(dtype).eps, atol=tol)
    rest = torch.ones_like(buf, dtype=torch.bool)
    rest[oshift:oshift + R * (V + opad)].view(R, V + opad)[:, :V] = False
    assert (buf[rest] == 3.0).all()


@pytest.mark.gpu
def test_large_offsets_streams_and_capture(dev):
    """Rows more than 2^31 elements apart, a side stream, captured and replayed calls, the same bits each time."""
    far = torch.zeros(2 ** 31 + 2 ** 12, device=dev, dtype=torch.bfloat16)
    x = far.as_strided((2, 2000), (2 ** 31 + 2 ** 10, 1))
    x.copy_(torch.randn(2, 2000, device=dev) * 3)
    check_top(x, 9)
    ids, logp = lists(x, 9)
    run = distill_loss_grad(x, ids, logp, out=x)
    assert torch.isfinite(run[1].float()).all()
    del far, x, run
    x = rows(50, 5003, torch.bfloat16, dev)
    ids, logp = lists(x, 17)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first = topk_logprobs(x, 17) + distill_loss_grad(x, ids, logp)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            out = topk_logprobs(x, 17) + distill_loss_grad(x, ids, logp)
    torch.cuda.current_stream().wait_stream(s)
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, first))
    x.copy_(rows(50, 5003, torch.bfloat16, dev, seed=4))
    a, b = lists(x, 17, seed=2)
    ids.copy_(a)
    logp.copy_(b)
    g.replay()
    assert all(torch.equal(p, q) for p, q in zip(out, topk_logprobs(x, 17) + distill_loss_grad(x, ids, logp)))


@pytest.mark.gpu
def test_forward_and_backward_in_a_graph(dev):
    x = rows(20, 3001, torch.bfloat16, dev).clone().requires_grad_()
    ids, logp = lists(x.detach(), 10)
    dl = torch.rand(20, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(distill_loss(x, ids, logp), x, dl)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss = distill_loss(x, ids, logp, kind="reverse")
        (d,) = torch.autograd.grad(loss, x, dl)
    with torch.no_grad():
        x.copy_(rows(20, 3001, torch.bfloat16, dev, seed=6))
        dl.copy_(torch.rand(20, device=dev))
    g.replay()
    l2 = distill_loss(x, ids, logp, kind="reverse")
    (d2,) = torch.autograd.grad(l2, x, dl)
    assert torch.equal(loss, l2) and torch.equal(d, d2)


@pytest.mark.parametrize("device", DEVICES)
def test_list_to_loss(device):
    """The two as they are used: a teacher's list of its own row gives no loss to the same student, and pulls another
    one towards it."""
    x = rows(6, 700, torch.float32, device, spread=2.0)
    top = topk_logprobs(x, 32)
    for kind, rest in KINDS:
        loss, d = distill_loss_grad(x, top.ids, top.logprobs, kind=kind, rest=rest)
        if rest:
            # KL of two distributions whose logarithms differ by their errors alone
            assert (loss.abs() <= 8 * (sum_error(700) + 2.0 ** -22) * 2).all()
        other = rows(6, 700, torch.float32, device, seed=9, spread=2.0)
        a, d = distill_loss_grad(other, top.ids, top.logprobs, kind=kind, rest=rest)
        b = distill_loss(other - 0.1 * d, top.ids, top.logprobs, kind=kind, rest=rest)
        assert (b < a).all()


def far_rows(V, device):
    """fp32 rows around 2^20 whose differences are whole numbers up to 8: ascending, so that the running maximum rises
    often; descending; shuffled.  And the same around 0, shifted in exact steps."""
    g = torch.Generator().manual_seed(V)
    z = torch.randint(0, 9, (3, V), generator=g).float()
    z[0], z[1] = z[0].sort().values, z[1].sort(descending=True).values
    return (z + 2.0 ** 20).to(device), z.to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1.0, 2.0 ** -10, 2.0 ** 8])
def test_logits_far_from_zero(T, device):
    """Maxima whose product with 1 / T is coarse in fp32: what counts are the differences.  (1 / T exact.)"""
    far, near = far_rows(40000, device)
    for z in (far, -far, near * 1000.0):
        check_top(z, 20, T)
    if T != 1.0:
        return
    ids, logp = lists(near, 40)
    y = torch.tensor([5, 39999, 20000], dtype=torch.int32, device=device)
    for kind, rest in KINDS:
        run_both(far, ids, logp, None, kind, rest, 1.0, y, None)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind,rest", KINDS)
def test_faint_entries(kind, rest, device):
    """Masses below 2^-149, once and twice in the list."""
    x = rows(4, 200, torch.float32, device, spread=1.0)
    ids, logp = lists(x, 6)
    logp = logp.clone()
    logp[:2, 3:] = -200.0
    ids[1, 4], ids[2, 1], logp[2, :2] = ids[1, 3], ids[2, 0], -300.0
    run_both(x, ids, logp, None, kind, rest, 1.0, None, None)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [777, 40003])
def test_gradient_of_slices(V, dtype, device):
    """Rows that begin behind the first element of an odd row (shifted tokens of a batch)."""
    x = rows(7, V, dtype, device, pad=0)[1:]
    ids, logp = lists(x, 10)
    loss, d = distill_loss_grad(x, ids, logp)
    compare(loss, d, x, definition(x, ids, logp, None, "forward", True, 1.0, None, None))
    leaf = x.detach().requires_grad_()
    l = distill_loss(leaf, ids, logp)
    l.sum().backward()
    compare(l, leaf.grad, x, definition(x, ids, logp, None, "forward", True, 1.0, None, None))
    assert leaf.grad.shape == x.shape


def by_log_masses(x, ids, logp, kind, rest):
    """(loss, gradient, scale of the errors [R, V], factor of the loss's), as `definition` gives them, in 64 bits from the
    logarithms of the classes' masses: no mass itself is formed where only its logarithm counts."""
    loss, grads, mags, facs = [], [], [], []
    for r in range(x.shape[0]):
        z = x[r].cpu().double().requires_grad_()
        lp = torch.log_softmax(z, 0)
        entries = {}
        for a, l in zip(ids[r].tolist(), logp[r].double().tolist()):
            if a >= 0 and l > -INF:
                entries.setdefault(a, []).append(l)
        at = torch.tensor(sorted(entries), dtype=torch.long)
        lt = torch.stack([torch.logsumexp(torch.tensor(entries[a], dtype=torch.float64), 0) for a in sorted(entries)])
        outside = torch.ones(len(z), dtype=torch.bool)
        outside[at] = False
        lr = torch.logsumexp(lp[outside], 0)
        F = (lp.detach()[at] - lt).abs()
        if not rest:
            lt = lt - torch.logsumexp(lt, 0)
            F = (lp.detach()[at] - lt).abs()
            kl = (lt.exp() * (lt - lp[at])).sum()
        elif kind == "forward":
            tr = max(0.0, 1 - float(lt.exp().sum()))
            kl = (lt.exp() * (lt - lp[at])).sum() + (tr * (math.log(tr) - lr) if tr > 0 else 0.0)
        else:
            tr = max(1 - float(lt.exp().sum()), 2.0 ** -20)
            kl = (lp[at].exp() * (lp[at] - lt)).sum() + lr.exp() * (lr - math.log(tr))
        d, = torch.autograd.grad(kl, z)
        p = lp.detach().exp()
        mag = p + torch.where(outside, p / p[outside].sum(), 0.0)
        mag[at] += lt.exp()
        f = 2 + float(F.max())
        loss.append(float(kl.detach())), grads.append(d), mags.append(mag * f), facs.append(f)
    return torch.tensor(loss, dtype=torch.float64), torch.stack(grads), torch.stack(mags), torch.tensor(facs).double()


def check_list(x, ids, logp, kind, rest):
    """The fused form and the differentiable one against the logarithms' form."""
    want = by_log_masses(x, ids, logp, kind, rest)
    assert want[0].isfinite().all() and want[1].isfinite().all()
    loss, d = distill_loss_grad(x, ids, logp, kind=kind, rest=rest)
    compare(loss, d, x, want)
    leaf = x.detach().clone().requires_grad_()
    l = distill_loss(leaf, ids, logp, kind=kind, rest=rest)
    g, = torch.autograd.grad(l, leaf, torch.ones_like(l))
    compare(l, g, x, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind,rest", KINDS)
@pytest.mark.parametrize("low", [-700.0, -800.0, -1e4])
def test_faint_entries_beside_a_repeated_id(low, kind, rest, device):
    """Masses that 64 bits hold as zero: of an id that occurs once beside one that occurs twice, and of the repeated id
    itself.  (Reverse: their logarithms count.)"""
    x = rows(4, 200, torch.float32, device, spread=1.0)
    ids, logp = lists(x, 6)
    logp = logp.clone()
    logp[:3, 5] = low
    ids[1, 1] = ids[1, 0]
    ids[2, 4], logp[2, 4] = ids[2, 5], low - 0.5
    check_list(x, ids, logp, kind, rest)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("offset", [-80.0, -95.0, -120.0, -800.0, -1e4, 60.0, 100.0, 1000.0])
def test_a_normalised_list_at_any_offset(offset, device):
    """Without the rest the list is divided by its sum: a common offset of its log-probabilities (a list of unlikely
    tokens, or of scores) changes nothing but their own rounding, which the 64-bit form sees too.  An id twice, and
    entries of very different weight."""
    x = rows(4, 200, torch.float32, device, spread=1.0)
    ids, logp = lists(x, 6)
    ids = ids.clone()
    logp = logp + offset
    ids[1, 1] = ids[1, 0]
    logp[2, 3] -= 30.0
    check_list(x, ids, logp, "forward", False)


@pytest.mark.parametrize("device", DEVICES)
def test_a_faint_entry_that_the_student_rules_out(device):
    """A mass that 32 bits hold as zero and 64 bits do not, on a logit of -inf: the loss is infinite as for any other."""
    x = rows(3, 100, torch.float32, device, spread=1.0)
    ids, logp = lists(x, 5)
    logp = logp.clone()
    logp[1, 2], logp[2, 2] = -150.0, -1.0
    x[1, ids[1, 2].long()] = x[2, ids[2, 2].long()] = -INF
    for rest in (True, False):
        loss, d = distill_loss_grad(x, ids, logp, rest=rest)
        assert loss.isinf().tolist() == [False, True, True] and (loss[1:] > 0).all() and d.isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind,rest", KINDS)
def test_the_kl_alone(kind, rest, device):
    """Beside the loss: without the row's weight and target; 0 in rows without weight, whatever they hold."""
    x = rows(6, 300, torch.float32, device, spread=1.0)
    ids, logp = lists(x, 7)
    w = torch.tensor([1.0, 1e-20, 0.0, -3.0, 0.0, 2.0], device=device)
    y = torch.tensor([3, 5, 7, -1, -1, 9], dtype=torch.int32, device=device)
    c = torch.tensor([1.0, 40.0, -2.0, 1.0, 1.0, 0.0], device=device)
    want = by_log_masses(x, ids, logp, kind, rest)
    x[4] = NAN
    how = dict(kind=kind, rest=rest, target=y, target_weight=c)
    kl = torch.full((6,), NAN, device=device)
    loss, d = distill_loss_grad(x, ids, logp, w, kl=kl, **how)
    plain = distill_loss_grad(x, ids, logp, w, **how)
    assert torch.equal(loss, plain[0]) and torch.equal(d, plain[1])
    on = w != 0
    compare(kl[on], None, x, [t[on.cpu()] for t in want])
    assert not kl[~on].any()
    x[0] = -INF
    distill_loss_grad(x, ids, logp, w, kl=kl, **how)
    assert kl.isnan().tolist() == [True] + [False] * 5
    for bad in (kl[:5], kl.double(), torch.empty(12, device=device)[::2], w, c, kl.clone().requires_grad_(), x.view(-1)[:6]):
        with pytest.raises(ValueError, match="distill_loss_grad"):
            distill_loss_grad(x, ids, logp, w, kl=bad, **how)
    distill_loss_grad(x[:0], ids[:0], logp[:0], kl=kl[:0])


def tight(V):
    """Relative error of a row's sum where every logit is within 4 of the largest: the exponential (2^-22), its argument
    (up to 6 in size: the factor, the difference, the fused product, 18 x 2^-24 ln 2), the additions of one of the row's
    1,024 partial sums (V / 1024, and up to 16 more where a warp has the whole of a short row) and the some 16 of joining
    them, the correction of the argument's rounding, the logarithm (2^-25), and its number's roundings (up to 14 in size)."""
    return 2.0 ** -24 * (4 + 13 + V / 1024 + 16 + 16 + 2 + 1 + 28)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1000, 9001, 50001, 151936])
def test_sums_of_near_logits(V, dtype, device):
    """Rows of equal logits, and of logits that rise by up to 4, around 0 and around 1,300 (whose product with log2(e) is
    coarse in fp32): log-probabilities, loss and gradient within the bounds of these sums, not of the worst ones.  A
    correction of the exponent left out would be off by up to 4e-5."""
    g = torch.Generator().manual_seed(V)
    R = 24
    z = torch.randint(0, 33, (R, V), generator=g).float() / 8
    z[: R // 2] = 0.0
    z[R // 2:: 2] = z[R // 2:: 2].sort(1).values
    # (multiples of 1/8 are exact in fp16 up to 256, of 1/2 up to 1024)
    c = 700 + 640 * torch.rand(R, generator=g) if dtype == torch.float32 else torch.randint(200, 250, (R,), generator=g).float()
    c = (c * 8).round() / 8
    c[::3] = 0.0
    x = (z + c[:, None]).to(dtype).to(device)
    assert torch.equal(x.cpu().float(), z + c[:, None])
    lp = torch.log_softmax(x.double(), 1)
    logp, ids, _ = topk_logprobs(x, 5)
    assert ((logp.double() - lp.gather(1, ids.long())).abs() <= tight(V)).all()
    # the target alone: loss = -log p, gradient = p - [target]
    y = torch.randint(0, V, (R,), generator=g).int().to(device)
    zero = torch.zeros(R, device=device)
    for out in (None, x.clone()):
        args = (x if out is None else out, ids, logp, zero)
        loss, d = distill_loss_grad(*args, target=y, out=out)
        at = torch.arange(R, device=device)
        assert ((loss.double() + lp[at, y.long()]).abs() <= tight(V)).all()
        want = lp.exp()
        want[at, y.long()] -= 1
        tol = (tight(V) + 18 * 2.0 ** -24 + torch.finfo(dtype).eps / 2) * want.abs() + TINY[dtype]
        tol[at, y.long()] += tight(V) * lp.exp()[at, y.long()] + 2.0 ** -23
        assert ((d.double() - want).abs() <= tol).all()
    # a teacher that agrees: every class's log-ratio is an error alone
    for kind in ("forward", "reverse"):
        loss, d = distill_loss_grad(x, ids, logp, kind=kind)
        assert (loss.abs() <= 4 * tight(V)).all()
        assert (d.double().abs() <= 4 * tight(V) * (lp.exp() + 2.0 ** -20) + TINY[dtype]).all()


@pytest.mark.gpu
def test_more_rows_than_ctas(dev):
    """More rows than the grid has CTAs: every row is reached."""
    R, V, K = 2 ** 20 + 37, 24, 3
    x = rows(R, V, torch.bfloat16, dev)
    check_top(x, K)
    top = topk_logprobs(x, K)
    w = (torch.arange(R, device=dev) % 7 != 3).float()
    other = rows(R, V, torch.bfloat16, dev, seed=1)
    loss, d = distill_loss_grad(other, top.ids, top.logprobs, w)
    last = slice(R - 2000, R)
    part = distill_loss_grad(other[last].clone(), top.ids[last].clone(), top.logprobs[last].clone(), w[last].clone())
    assert torch.equal(loss[last], part[0]) and torch.equal(d[last], part[1])
    assert loss[w != 0].isfinite().all() and (loss[w != 0] != 0).any() and not d[w == 0].any()
    out = distill_loss_grad(other, top.ids, top.logprobs, w, out=other)
    assert torch.equal(out[0], loss) and torch.equal(other, d)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1.0, 3.0])
def test_rows_of_the_lowest_value(T, dtype, device):
    """Every logit masked with the type's lowest value (or equal at its largest): a flat row, like any constant one."""
    V = 7
    ids = torch.tensor([[1, 4]] * 3, dtype=torch.int32, device=device)
    logp = torch.tensor([[-0.5, -1.5]] * 3, device=device)
    y = torch.tensor([2, 4, 0], dtype=torch.int32, device=device)
    low = torch.finfo(dtype).min
    x = torch.tensor([[low] * V, [0.0] * V, [-low] * V], dtype=dtype, device=device)
    for kind, rest in KINDS:
        loss, d = distill_loss_grad(x, ids, logp, kind=kind, rest=rest, temperature=T, target=y)
        want = definition(x[1:2].expand(3, V), ids, logp, None, kind, rest, T, y, None)
        compare(loss, d, x, want)
        leaf = x.clone().requires_grad_()
        l = distill_loss(leaf, ids, logp, kind=kind, rest=rest, temperature=T, target=y)
        g, = torch.autograd.grad(l.sum(), leaf)
        compare(l, g, x, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind,rest", KINDS)
def test_broken_rows_without_a_list(kind, rest, device):
    """NaN, +inf or no logit above -inf give NaN in a row with weight, also where its list is all padding."""
    x = rows(5, 60, torch.float32, device, spread=1.0)
    x[0, 7], x[1, 7], x[2], x[4] = NAN, INF, -INF, NAN
    ids, logp = lists(x, 3)
    w = torch.tensor([1.0, 1.0, 1.0, 1.0, 0.0], device=device)
    for pad in ("ids", "logp"):
        a = torch.full_like(ids, -1) if pad == "ids" else ids
        b = torch.full_like(logp, -INF) if pad == "logp" else logp
        kl = torch.zeros(5, device=device)
        loss, d = distill_loss_grad(x, a, b, w, kind=kind, rest=rest, kl=kl)
        broken = [True, True, True, False, False]
        assert loss.isnan().tolist() == broken and kl.isnan().tolist() == broken
        assert d.isnan().all(1).tolist() == broken and d.isnan().any(1).tolist() == broken
        leaf = x.clone().requires_grad_()
        g, = torch.autograd.grad(distill_loss(leaf, a, b, w, kind=kind, rest=rest).sum(), leaf)
        assert g.isnan().all(1).tolist() == broken and g.isnan().any(1).tolist() == broken


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["forward", "reverse"])
def test_a_rest_of_the_lowest_value(kind, dtype, device):
    """What is outside the list masked with the type's lowest value: the rest's pull is shared by its logits, and a row's
    gradient sums to zero (up to its own roundings)."""
    low = torch.finfo(dtype).min
    x = torch.tensor([[0.5, low, low, -1.0, low]], dtype=dtype, device=device)
    ids = torch.tensor([[0, 3]], dtype=torch.int32, device=device)
    logp = torch.tensor([[-0.7, -1.5]], device=device)
    loss, d = distill_loss_grad(x, ids, logp, kind=kind)
    rest = 1 - math.exp(-0.7) - math.exp(-1.5) if kind == "forward" else 0.0
    assert (d[0, [1, 2, 4]].double() + rest / 3).abs().max() <= torch.finfo(dtype).eps * rest / 3 + 2.0 ** -22
    assert abs(float(d.double().sum())) <= 5 * torch.finfo(dtype).eps


@pytest.mark.parametrize("device", DEVICES)
def test_faint_scores_that_the_student_rules_out(device):
    """Without the rest: a mass that vanishes when it is divided by the sum, on a logit of -inf."""
    x = rows(1, 50, torch.float32, device, spread=1.0)
    ids = torch.arange(40, dtype=torch.int32, device=device)[None]
    x[0, 39] = -INF
    for faint in (-100.0, -102.0, -103.0, -103.5, -150.0):
        logp = torch.full((1, 40), 0.0, device=device)
        logp[0, 39] = faint
        for shift in (0.0, 30.0, -90.0):
            kl = torch.empty(1, device=device)
            loss, _ = distill_loss_grad(x, ids, logp + shift, rest=False, kl=kl)
            assert loss.isposinf().all() and kl.isposinf().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_huge_terms_that_cancel(dtype, device):
    """A target and listed tokens masked with the type's lowest value: terms near fp32's end whose sum is within it."""
    low = torch.finfo(dtype).min
    x = torch.tensor([[0.5, low, 1.0, -1.0, 0.25]] * 3, dtype=dtype, device=device)
    ids = torch.tensor([[0, 1]] * 3, dtype=torch.int32, device=device)
    logp = torch.tensor([[-1.2, -0.7]] * 3, device=device)
    w = torch.tensor([3.5, -3.0, 1.5], device=device)
    y = torch.tensor([1, 1, 1], dtype=torch.int32, device=device)
    c = torch.tensor([-1.5, 1.75, -0.5], device=device)
    for kind, rest in KINDS[:2]:
        t = torch.tensor([math.exp(-1.2), math.exp(-0.7)], dtype=torch.float64)
        t = t if rest else t / t.sum()
        want = -(w.cpu().double() * t[1] + c.cpu().double()) * low  # (what else there is is below 2^-100 of it)
        mag = (w.cpu().double() * t[1]).abs() + c.cpu().double().abs()
        loss, d = distill_loss_grad(x, ids, logp, w, kind=kind, rest=rest, target=y, target_weight=c)
        assert d.isfinite().all()
        # the mass, its share and the loss: 8 roundings of terms of this size
        assert ((loss.cpu().double() - want).abs() <= 8 * 2.0 ** -24 * mag * -low).all(), (loss, want)
