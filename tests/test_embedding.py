"""The scaled embedding lookup and its gradient by sorted tokens against 64-bit math:
types, odd sizes, strides, repeated and invalid tokens, refusals, autograd, the same bits."""
import math

import pytest
import torch

from turbol_b200.ops.embedding import embedding, embedding_grad

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]
TYPES = [torch.bfloat16, torch.float16, torch.float32]
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}  # (added as zero below)


def half(t):
    return torch.finfo(t).eps / 2 * 1.001


def tokens(N, V, how, seed=0):
    g = torch.Generator().manual_seed(seed + N)
    ids = torch.randint(0, V, (N,), generator=g)
    if how == "one":
        ids[:] = V - 1
    elif how == "hot":  # one id for a third of the tokens, anywhere
        ids[torch.rand(N, generator=g) < 0.33] = V // 2
    elif how == "runs":
        ids = torch.arange(N) // 37 % V
    elif how == "zipf":
        ids = (V ** torch.rand(N, generator=g)).long() - 1
    elif how == "invalid":
        ids[::3] = -torch.randint(1, 2 ** 30, (len(ids[::3]),), generator=g)
    return ids


def check_lookup(ids, W, scale):
    y = embedding(ids, W, scale)
    assert y.shape == (*ids.shape, W.shape[1]) and y.dtype == W.dtype
    i = ids.long()
    want = torch.where((i >= 0)[..., None], W.double()[i.clamp_min(0)] * scale, 0.0)
    assert ((y.double() - want).abs() <= half(W.dtype) * want.abs() + 2.0 ** -24 * want.abs() + TINY[W.dtype]).all()
    return y


def exact_sums(ids, dy, V, scale):
    """(sums, sums of absolute values) in 64 bits."""
    i = ids.reshape(-1).long()
    t = (i >= 0) & (i < V)
    d = dy.reshape(i.numel(), -1)[t].double() * scale
    z = torch.zeros(V, dy.shape[-1], dtype=torch.float64, device=dy.device)
    return z.index_add(0, i[t], d), z.index_add(0, i[t], d.abs())


def check_grad(ids, dy, grad, scale, accumulate=True):
    """Every addition is off by 2^-24 of the sum of absolute values at most (n of them, and the scale's product), then one
    rounding of the result."""
    V, before = grad.shape[0], grad.double()
    s, mag = exact_sums(ids, dy, V, scale)
    n = torch.bincount(ids.reshape(-1).long()[(ids.reshape(-1) >= 0) & (ids.reshape(-1) < V)], minlength=V)
    out = embedding_grad(ids, dy, grad, scale, accumulate)
    assert out is grad
    want = s + before if accumulate else s
    tol = (n[:, None] + 2) * 2.0 ** -24 * mag + 2.0 ** -24 * want.abs() + half(grad.dtype) * want.abs() + TINY[grad.dtype]
    over = (grad.double() - want).abs() - tol
    assert not (over > 0).any(), over.max()
    if accumulate:
        assert torch.equal(grad[n == 0].double(), before[n == 0])  # rows that no id names stay
    else:
        assert not grad[n == 0].any()


CASES = [(1, 1, 1, "uniform"), (5, 3, 8, "uniform"), (33, 1, 7, "one"), (64, 1000, 1536, "zipf"), (130, 17, 257, "hot"),
         (1000, 50, 64, "runs"), (777, 2000, 100, "invalid"), (1024, 5, 33, "uniform"), (1025, 70000, 40, "zipf"),
         (3001, 300, 96, "hot")]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,H,how", CASES)
def test_matches_64_bits(N, V, H, how, dtype, device):
    g = torch.Generator().manual_seed(N)
    ids = tokens(N, V, how).to(torch.int32 if N % 2 else torch.int64).to(device)
    W = torch.randn(V, H, generator=g).to(dtype).to(device)
    dy = torch.randn(N, H, generator=g).to(dtype).to(device)
    check_lookup(ids, W, 1.0)
    check_lookup(ids, W, 39.25)
    check_grad(ids, dy, torch.randn(V, H, generator=g).to(device), 0.5)
    for G in TYPES:
        check_grad(ids, dy, torch.randn(V, H, generator=g).to(G).to(device), 1.0, accumulate=G != torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,H,how", [(6144, 151936, 1536, "zipf"), (16384, 128256, 512, "zipf"), (65537, 32003, 129, "hot"),
                                       (20000, 11, 1024, "uniform"), (40000, 3, 72, "one"), (9000, 262144, 256, "invalid"),
                                       (131072, 1000000, 16, "uniform"), (262145, 70001, 8, "zipf"), (8193, 5000, 4099, "runs"),
                                       (2048, 700, 8200, "hot"), (2049, 2 ** 27 + 1, 1, "uniform")])
def test_many_tokens(N, V, H, how, dtype):
    g = torch.Generator(device="cuda").manual_seed(N)
    ids = tokens(N, V, how).int().cuda()
    if V * H < 2 ** 27:
        check_lookup(ids, torch.randn(V, H, generator=g, device="cuda").to(dtype), 1.5)
    dy = torch.randn(N, H, generator=g, device="cuda").to(dtype)
    check_grad(ids, dy, torch.randn(V, H, generator=g, device="cuda"), 0.5)
    grads = []
    for _ in range(2):
        grads.append(torch.full((V, H), 3.0, device="cuda", dtype=dtype))
        check_grad(ids, dy, grads[-1], 2.0, accumulate=False)
    assert torch.equal(*grads)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,pad,shift", [(64, 0, 0), (64, 8, 0), (64, 3, 1), (33, 2, 5), (128, 64, 2), (8, 0, 4)])
def test_strides(H, pad, shift, dtype, device):
    """Rows of any stride and alignment; what lies between them stays."""
    N, V = 300, 90
    g = torch.Generator().manual_seed(H)
    ids = tokens(N, V, "hot").int().to(device)

    def view(n, t):
        b = torch.randn(n * (H + pad) + shift, generator=g).to(t).to(device)
        return b, b[shift:].view(n, H + pad)[:, :H]

    _, W = view(V, dtype)
    _, dy = view(N, dtype)
    check_lookup(ids, W, 3.0)
    for G in {dtype, torch.float32}:
        for acc in (True, False):
            buf, grad = view(V, G)
            before = buf.clone()
            check_grad(ids, dy, grad, 0.25, acc)
            rest = torch.ones_like(buf, dtype=torch.bool)
            rest[shift:].view(V, H + pad)[:, :H] = False
            assert torch.equal(buf[rest], before[rest])
    out = torch.empty(N, H, dtype=dtype, device=device)
    assert embedding(ids, W, 3.0, out=out) is out and torch.equal(out, embedding(ids, W, 3.0))


@pytest.mark.parametrize("device", DEVICES)
def test_shapes(device):
    """Ids of any shape, none at all, a broadcast gradient."""
    W = torch.randn(10, 16, device=device)
    ids = torch.randint(0, 10, (3, 5, 2), device=device)
    check_lookup(ids, W, 2.0)
    check_grad(ids, torch.randn(3, 5, 2, 16, device=device), torch.randn(10, 16, device=device), 1.0)
    check_grad(ids, torch.randn(1, device=device).expand(3, 5, 2, 16), torch.randn(10, 16, device=device), 1.0)
    check_grad(ids, torch.randn(3, 5, 16, 2, device=device).transpose(2, 3), torch.randn(10, 16, device=device), 1.0)
    check_lookup(ids[0, 0, 0].clone(), W, 1.0)
    none = torch.empty(0, dtype=torch.int32, device=device)
    assert embedding(none, W).shape == (0, 16)
    g = torch.ones(10, 16, device=device)
    embedding_grad(none, torch.empty(0, 16, device=device), g)
    assert (g == 1).all()
    embedding_grad(none, torch.empty(0, 16, device=device), g, accumulate=False)
    assert not g.any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("N", [40, 3000])
def test_ids_out_of_range(index, N, device):
    """Told, NaN in the lookup, left out of the gradient; padding is zero and not told."""
    V, H = 20, 24
    ids = tokens(N, V, "invalid").to(index)
    W, dy = torch.randn(V, H, device=device), torch.randn(N, H, device=device)
    err = torch.zeros(1, dtype=torch.int32, device=device)
    g = torch.zeros(V, H, device=device)
    y = embedding(ids.to(device), W, 2.0, error=err)
    embedding_grad(ids.to(device), dy, g, error=err)
    assert int(err) == 0 and not y[ids.to(device) < 0].any()
    bad = ids.clone()
    bad[7], bad[N - 1] = V, 2 ** 31 - 1 if index == torch.int32 else 2 ** 40 + 3
    z = embedding(bad.to(device), W, 2.0, error=err)
    assert int(err) == 1
    assert z[7].isnan().all() and z[N - 1].isnan().all()
    keep = torch.ones(N, dtype=torch.bool)
    keep[7] = keep[N - 1] = False
    assert torch.equal(z[keep.to(device)], y[keep.to(device)])
    err.zero_()
    g2, g3 = torch.zeros_like(g), torch.zeros_like(g)
    embedding_grad(bad.to(device), dy, g2, error=err)
    assert int(err) == 1
    bad[7] = bad[N - 1] = -1
    embedding_grad(bad.to(device), dy, g3)
    assert torch.equal(g2, g3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_values_stay(dtype, device):
    """NaN and infinities reach their own rows alone."""
    V, H, N = 30, 16, 1500
    ids = tokens(N, V, "uniform").int().to(device)
    dy = torch.randn(N, H, device=device).to(dtype)
    W = torch.randn(V, H, device=device).to(dtype)
    W[3] = math.nan
    W[4, 2] = math.inf
    y = embedding(ids, W, 2.0)
    assert y[ids == 3].isnan().all() and (y[ids == 4][:, 2] == math.inf).all() and y[(ids != 3) & (ids != 4)].isfinite().all()
    dy[ids == 5] = math.nan
    grad = embedding_grad(ids, dy, torch.zeros(V, H, device=device))
    assert grad[5].isnan().all() and grad[torch.arange(V) != 5].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_autograd(dtype, device):
    """The dense gradient, of a sum too, and the gradient of the gradient (it is linear)."""
    V, H, N = 50, 12, 200
    ids = tokens(N, V, "hot").int().to(device)
    ids[3] = -1
    W = torch.randn(V, H, device=device).to(dtype).requires_grad_()
    dy = torch.randn(N, H, device=device).to(dtype).requires_grad_()
    y = embedding(ids, W, 3.0)
    g, = torch.autograd.grad(y, W, dy, create_graph=True)
    want = embedding_grad(ids, dy.detach(), torch.empty(V, H, device=device, dtype=dtype), 3.0, accumulate=False)
    assert g.dtype == dtype and torch.equal(g, want)
    v = torch.randn(V, H, device=device).to(dtype)
    gg, = torch.autograd.grad(g, dy, v)
    assert torch.equal(gg, embedding(ids, v, 3.0))
    embedding(ids, W, 3.0).sum().backward()
    check = embedding_grad(ids, torch.ones(N, H, device=device, dtype=dtype), torch.empty_like(W.detach()), 3.0, False)
    assert torch.equal(W.grad, check)
    with torch.no_grad():
        assert not embedding(ids, W, 3.0).requires_grad


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences(device):
    """The lookup is linear: differences are exact but for the roundings of the two lookups."""
    ids = tokens(60, 9, "uniform").to(device)
    W = torch.randn(9, 5, device=device)
    dy = torch.randn(60, 5, device=device)
    g = embedding_grad(ids, dy, torch.zeros(9, 5, device=device), 1.5)
    for v, h in ((0, 0), (4, 3), (8, 4)):
        up, down = W.clone(), W.clone()
        up[v, h] += 0.5
        down[v, h] -= 0.5
        f = [(embedding(ids, a, 1.5).double() * dy.double()).sum() for a in (up, down)]
        step = float((up - down)[v, h])
        mag = float((embedding(ids, up.abs() + down.abs(), 1.5).double() * dy.abs().double()).sum())
        assert abs(float((f[0] - f[1]) / step) - float(g[v, h])) <= 64 * 2.0 ** -24 * mag / step


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    W, dy = torch.randn(9, 8, device=device), torch.randn(5, 8, device=device)
    ids = torch.arange(5, device=device, dtype=torch.int32)
    g = torch.zeros(9, 8, device=device)
    dual = torch.autograd.forward_ad
    for bad in (lambda: embedding(ids.float(), W), lambda: embedding(ids.short(), W), lambda: embedding(ids, W[0]),
                lambda: embedding(ids, W.double()), lambda: embedding(ids, W.t()), lambda: embedding(ids, W, math.inf),
                lambda: embedding(ids, W, 1e39), lambda: embedding(ids[::2], W), lambda: embedding(ids, W[:, :0]),
                lambda: embedding(ids, W[:0]), lambda: embedding(ids, W, out=torch.empty(5, 9, device=device)),
                lambda: embedding(ids, W, out=W[:5]), lambda: embedding(ids, W, error=W),
                lambda: embedding(ids, W.clone().requires_grad_(), out=dy.clone())):
        with pytest.raises(ValueError, match="embedding"):
            bad()
    for bad in (lambda: embedding_grad(ids, dy[:4], g), lambda: embedding_grad(ids, dy.double(), g),
                lambda: embedding_grad(ids, dy, g.t()), lambda: embedding_grad(ids, dy, g[0]),
                lambda: embedding_grad(ids, dy, g[:1].expand(9, 8)), lambda: embedding_grad(ids, dy, g, math.nan),
                lambda: embedding_grad(ids, g[:5], g), lambda: embedding_grad(ids, dy.clone().requires_grad_(), g),
                lambda: embedding_grad(ids, dy, g.clone().requires_grad_()), lambda: embedding_grad(ids, dy, g[:, :7])):
        with pytest.raises(ValueError, match="embedding_grad"):
            bad()
    with dual.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            embedding(ids, dual.make_dual(W, torch.ones_like(W)))
        with pytest.raises(ValueError, match="forward-mode"):
            embedding_grad(ids, dual.make_dual(dy, torch.ones_like(dy)), g)


@pytest.mark.gpu
def test_devices_are_not_mixed(dev):
    W, ids = torch.randn(9, 8, device=dev), torch.arange(5, device=dev)
    for bad in (lambda: embedding(ids.cpu(), W), lambda: embedding(ids, W.cpu()),
                lambda: embedding_grad(ids, torch.randn(5, 8), W), lambda: embedding_grad(ids.cpu(), W[:5].clone(), W)):
        with pytest.raises(ValueError, match="one device"):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [50, 5000])
def test_streams_and_capture(N, dev):
    """A side stream, two captured graphs that replay in turn, replays on other tokens, the same bits."""
    V, H = 700, 264
    ids = tokens(N, V, "hot").int().cuda()
    dy, W = torch.randn(N, H, device=dev).bfloat16(), torch.randn(V, H, device=dev).bfloat16()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        y = embedding(ids, W, 2.0)
        first = embedding_grad(ids, dy, torch.zeros(V, H, device=dev))
        torch.cuda.synchronize()
        for _ in range(2):
            g, grad = torch.cuda.CUDAGraph(), torch.zeros(V, H, device=dev)
            with torch.cuda.graph(g, stream=s):
                out = embedding(ids, W, 2.0)
                embedding_grad(ids, dy, grad, accumulate=False)
            graphs.append((g, out, grad))
    torch.cuda.current_stream().wait_stream(s)
    for k in range(2):
        for g, out, grad in graphs:
            g.replay()
        for g, out, grad in graphs:
            assert torch.equal(out, y) and torch.equal(grad, first)
        ids.copy_(tokens(N, V, "zipf", seed=k))
        y, first = embedding(ids, W, 2.0), embedding_grad(ids, dy, torch.zeros(V, H, device=dev))


@pytest.mark.gpu
def test_large_offsets(dev):
    """Rows beyond 2^31 elements of the table, the output and the gradient."""
    H, V = 4096, 2 ** 19 + 100
    W = torch.empty(V, H, device=dev, dtype=torch.float16)
    W[::4096] = 1.5
    W[-1], W[V - 100] = 2.0, 3.0
    ids = torch.tensor([0, V - 1, 4096 * 3, V - 100, V - 1], device=dev, dtype=torch.int32)
    y = embedding(ids, W, 2.0)
    assert torch.equal(y[:, 0], torch.tensor([3.0, 4.0, 3.0, 6.0, 4.0], device=dev, dtype=torch.float16))
    W.zero_()
    embedding_grad(ids, y, W)
    assert float(W[V - 1, H - 1]) == 8.0 and float(W[V - 100, 5]) == 6.0 and float(W[0, 0]) == 3.0
    del W
    many = torch.zeros(V, dtype=torch.int64, device=dev)
    many[-1] = 1
    y = embedding(many, torch.tensor([[1.0], [2.0]], device=dev).expand(2, H).contiguous().half())
    assert float(y[-1, -1]) == 2.0 and float(y[-2, -1]) == 1.0
    g = embedding_grad(many, y, torch.zeros(2, H, device=dev))
    assert (g[0] == V - 1).all() and (g[1] == 2.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,H", [(513, 70001, 128), (700, 8191, 1025), (9000, 40, 300000), (20000, 300007, 31), (4096, 3, 2900001)])
def test_zeros_beside_the_sums(N, V, H, dtype, dev):
    """Large dense gradients: every row that no id names is zero, whatever was there, the others as if added to zeros;
    the same when an id past the table or a filler token is among them."""
    g = torch.Generator().manual_seed(N)
    ids = torch.randint(0, V, (N,), generator=g)
    ids[:: 7], ids[1], ids[2] = V - 1, -1, V + 5
    if V > 1000:
        ids[(ids >= 96) & (ids < 700)] = 0  # whole stretches without a name
    ids = ids.to(dev)
    dy = torch.randn(1, H, device=dev).to(dtype).expand(N, H) if H > 10000 else torch.randn(N, H, device=dev).to(dtype)
    out = torch.full((V, H), math.nan, device=dev, dtype=dtype)
    embedding_grad(ids, dy, out, scale=0.5, accumulate=False)
    want = torch.zeros_like(out)
    embedding_grad(ids, dy, want, scale=0.5)
    assert torch.equal(out, want)
    named = torch.zeros(V, dtype=torch.bool, device=dev)
    named[ids[(ids >= 0) & (ids < V)]] = True
    assert not out[~named].any() and out[named].any(1).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("H,pad", [(8, 0), (33, 2), (512, 0), (515, 1)])
def test_first_row(H, pad, device):
    """Ids outside the table read row 0 and are told, negative ones too; not with a gradient."""
    W = torch.randn(20, H + pad, device=device)[:, :H]
    ids = torch.tensor([3, -1, 19, 20, -2 ** 31, 2 ** 31 - 1, 0], dtype=torch.int32, device=device)
    inside = torch.tensor([3, 0, 19, 0, 0, 0, 0], dtype=torch.int32, device=device)
    err = torch.zeros(1, dtype=torch.int32, device=device)
    assert torch.equal(embedding(inside, W, 2.0, first_row=True, error=err), embedding(inside, W, 2.0)) and int(err) == 0
    assert torch.equal(embedding(ids, W, 2.0, first_row=True, error=err), embedding(inside, W, 2.0)) and int(err) == 1
    err.zero_()
    embedding(ids[:2].clone(), W, 2.0, first_row=True, error=err)
    assert int(err) == 1
    far = torch.tensor([2 ** 40, -2 ** 40], device=device)
    assert torch.equal(embedding(far, W, first_row=True), W[:1].expand(2, H))
    leaf = W.clone().requires_grad_()
    with pytest.raises(ValueError, match="first_row"):
        embedding(ids, leaf, first_row=True)
    with torch.no_grad():
        embedding(ids, leaf, first_row=True)


@pytest.mark.gpu
@pytest.mark.parametrize("N,V,H,how", [(2 ** 20 + 77, 5000, 8, "hot"), (2 ** 20 + 129, 300, 33, "zipf"), (3 * 2 ** 20 + 5, 2 ** 20, 4, "uniform"),
                                       (2 ** 21 + 1, 11, 16, "runs")])
def test_longer_pieces(N, V, H, how, dev):
    """So many tokens that the sums' pieces are longer than 128 of them."""
    g = torch.Generator(device=dev).manual_seed(N)
    ids = tokens(N, V, how).int().to(dev)
    dy = torch.randn(N, H, generator=g, device=dev).bfloat16()
    check_grad(ids, dy, torch.randn(V, H, generator=g, device=dev), 0.5)
    got = [embedding_grad(ids, dy, torch.empty(V, H, device=dev), 2.0, accumulate=False) for _ in range(2)]
    assert torch.equal(*got)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [0, 40, 3000])
def test_rows_far_apart(N, dev):
    """A gradient whose rows are more than 2^32 bytes apart, overwritten: its own elements alone."""
    V, H, step = 3, 24, 2 ** 31 + 8
    buf = torch.full((2 * step + 64,), 3.0, dtype=torch.bfloat16, device=dev)
    grad = buf.as_strided((V, H), (step, 1))
    ids = torch.full((N,), 2, dtype=torch.int32, device=dev)
    dy = torch.ones(N, H, device=dev, dtype=torch.bfloat16)
    embedding_grad(ids, dy, grad, 0.5, accumulate=False)
    want = torch.zeros(V, H)
    want[2] = torch.tensor(N / 2).bfloat16().float()  # (1,500 lies halfway between two bf16 values)
    assert torch.equal(grad.float().cpu(), want)
    for a, b in ((H, step), (step + H, 2 * step), (2 * step + H, buf.numel())):
        assert bool((buf[a:b] == 3.0).all())
