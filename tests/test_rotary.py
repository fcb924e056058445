"""General rotary positions against 64-bit math: layouts, partial heads, types,
strides, padding, refusals, gradients, and the scaled tables."""
import math

import pytest
import torch

from turbol_b200.ops import reference as ref
from turbol_b200.ops.rotary import rotary, rotary_inv_freq, rotary_table

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}  # half the smallest denormal

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def exact(x, pos, table, interleaved=False, transpose=False):
    """(64-bit result, sum of the absolute products behind each element)."""
    t = table.double()
    y = ref.rotary(x.double(), pos, t, interleaved, transpose)
    # |c a| + |s b| of every element: the rotation of |x| by a table of (|c|, -|s|) or (|c|, |s|)
    lo = ref.rotary(x.double().abs(), pos, torch.stack([t[..., 0].abs(), -t[..., 1].abs()], -1), interleaved)
    hi = ref.rotary(x.double().abs(), pos, torch.stack([t[..., 0].abs(), t[..., 1].abs()], -1), interleaved)
    return y, torch.maximum(lo.abs(), hi.abs())


def check(y, x, pos, table, interleaved=False, transpose=False):
    """Two products and a sum in fp32 (each off by 2^-24 of the products' sum at most, fused or not), one rounding."""
    e, mag = exact(x, pos, table, interleaved, transpose)
    tol = HALF_STEP[x.dtype] * e.abs() * 1.001 + 3 * 2.0 ** -24 * mag + TINY[x.dtype]
    over = (y.double() - e).abs() - tol
    assert not (over > 0).any(), over.max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,R", [(1, 1, 64, 64), (7, 3, 128, 128), (33, 14, 128, 64), (5, 2, 80, 20),
                                     (129, 5, 96, 24), (3, 1, 256, 256), (4, 2, 10, 6), (2, 9, 2, 2), (65, 40, 128, 32)])
def test_matches_64_bits(T, H, D, R, interleaved, dtype, device):
    g = torch.Generator().manual_seed(T * 1000 + H)
    x = (torch.randn(T, H, D, generator=g) * 3).to(dtype).to(device)
    table = rotary_table(R, 300, 1e4, device=device)
    pos = torch.randint(0, 300, (T,), generator=g, dtype=torch.int32).to(device)
    for tr in (False, True):
        y = rotary(x, pos, table, interleaved=interleaved, transpose=tr)
        check(y, x, pos, table, interleaved, tr)
        assert torch.equal(y[..., R:], x[..., R:])
        z = x.clone()
        assert rotary(z, pos, table, interleaved=interleaved, transpose=tr, out=z) is z
        assert torch.equal(z, y)  # in place: the same bits


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,R,shift", [(76001, 1, 128, 128, 0), (26003, 3, 128, 64, 0), (8501, 9, 128, 128, 0),
                                           (4003, 19, 128, 96, 0), (4801, 16, 128, 128, 4), (6007, 17, 96, 40, 1)])
def test_many_rows(T, H, D, R, shift, interleaved, dtype):
    """Enough rows for several heads per thread, whose last share is short; vectors of every width."""
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T * H * D + 8, generator=g).to(dtype).to("cuda:0")[shift:shift + T * H * D].view(T, H, D)
    table = rotary_table(R, 500, device="cuda:0")
    pos = torch.randint(-1, 500, (T,), generator=g, dtype=torch.int32).to("cuda:0")
    check(rotary(x, pos, table, interleaved=interleaved), x, pos, table, interleaved)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_strided_rows_and_heads(interleaved, device):
    """Views: columns of a fused projection, every second head, an offset of one element, expanded rows."""
    T, H, D = 11, 6, 64
    table = rotary_table(D, 64, device=device)
    pos = torch.arange(T, dtype=torch.int32, device=device)
    buf = torch.randn(T, H * D + 40, device=device).bfloat16()
    for x in (buf[:, 8:8 + H * D].view(T, H, D), buf[:, 1:1 + H * D].view(T, H, D), buf[:, :H * D].view(T, H, D)[:, ::2],
              buf[::2, :H * D].reshape(-1, H, D)[:T], buf[:1, :H * D].view(1, H, D).expand(T, H, D),
              buf[:, :D].view(T, 1, D).expand(T, H, D), buf[:, :H * D].view(T, H, D).transpose(0, 1)):
        p = torch.arange(x.shape[0], dtype=torch.int32, device=device)
        check(rotary(x, p, table, interleaved=interleaved), x, p, table, interleaved)
    # in place on a slice: the neighbours stay
    before = buf.clone()
    x = buf[:, 8:8 + H * D].view(T, H, D)
    want = rotary(x, pos, table, interleaved=interleaved)
    rotary(x, pos, table, interleaved=interleaved, out=x)
    assert torch.equal(x, want)
    assert torch.equal(buf[:, :8], before[:, :8]) and torch.equal(buf[:, 8 + H * D:], before[:, 8 + H * D:])
    # into an output with other strides
    out = torch.zeros(H, T, D, device=device, dtype=torch.bfloat16).transpose(0, 1)
    rotary(x, pos, table, interleaved=interleaved, out=out)
    check(out, x, pos, table, interleaved)


@pytest.mark.parametrize("device", DEVICES)
def test_padding_and_positions_out_of_range(device):
    table = rotary_table(64, 10, device=device)
    x = torch.randn(5, 3, 128, device=device)
    x[1, 0, 3] = float("inf")
    pos = torch.tensor([9, -1, 10, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=device)
    err = torch.zeros(1, dtype=torch.int32, device=device)
    y = rotary(x, pos, table, error=err)
    assert torch.equal(y[1], x[1]) and torch.equal(y[4], x[4])  # padding: copied
    assert y[2].isnan().all() and y[3].isnan().all() and int(err) == 1
    check(y[:1], x[:1], pos[:1], table)
    err.zero_()
    rotary(x[:2], pos[:2].contiguous(), table, error=err)
    assert int(err) == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients(interleaved, device):
    T, H, D, R = 6, 3, 16, 8
    table = rotary_table(R, 32, scaling={"type": "yarn", "factor": 4.0, "original_max_pos": 8}, device=device)
    pos = torch.randint(0, 32, (T,), dtype=torch.int32, device=device)
    pos[2] = -1
    x = torch.randn(T, H, D, device=device, requires_grad=True)
    dy = torch.randn(T, H, D, device=device)
    y = rotary(x, pos, table, interleaved=interleaved)
    (dx,) = torch.autograd.grad(y, x, dy)
    check(dx, dy, pos, table, interleaved, transpose=True)  # the formula's
    # against differences: the map is linear, so any step gives <dy, R v> = <dx, v>
    v = torch.randn(T, H, D, device=device)
    with torch.no_grad():
        step = rotary(x + v, pos, table, interleaved=interleaved).double() - y.double()
    lhs, rhs = float((dy.double() * step).sum()), float((dx.double() * v.double()).sum())
    n = T * H * D
    assert abs(lhs - rhs) <= 2.0 ** -20 * math.sqrt(n) * 4 * float(dy.abs().max() * (x.detach().abs().max() + v.abs().max()))
    # a broadcast gradient, a strided input, and the gradient of the gradient
    wide = torch.randn(T, H, 2 * D, device=device, requires_grad=True)
    rotary(wide[..., ::1][..., :D], pos, table, interleaved=interleaved).sum().backward()
    one = torch.ones(T, H, D, device=device)
    check(wide.grad[..., :D], one, pos, table, interleaved, transpose=True)
    assert not wide.grad[..., D:].any()
    w = dy.clone().requires_grad_()
    (gx,) = torch.autograd.grad(rotary(x, pos, table, interleaved=interleaved), x, w, create_graph=True)
    (gw,) = torch.autograd.grad(gx, w, v)
    check(gw, v, pos, table, interleaved)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    table = rotary_table(64, 10, device=device)
    x = torch.randn(4, 2, 64, device=device)
    pos = torch.zeros(4, dtype=torch.int32, device=device)
    bad = [
        (x[0], pos, table, {}),  # two dimensions
        (x.double(), pos, table, {}),
        (x.transpose(1, 2), pos, table, {}),  # last dimension not contiguous
        (x, pos[:3], table, {}),
        (x, pos.long(), table, {}),
        (x, torch.zeros(8, dtype=torch.int32, device=device)[::2], table, {}),
        (x[..., :32], pos, table, {}),  # the table is wider than the head
        (torch.randn(4, 2, 65, device=device), pos, table, {}),  # an odd head
        (x, pos, table.double(), {}),
        (x, pos, table[:, :, :1], {}),
        (x, pos, table[:0], {}),
        (x, pos, table, {"out": torch.empty(4, 2, 64, device=device, dtype=torch.bfloat16)}),
        (x, pos, table, {"out": torch.empty(4, 3, 64, device=device)}),
        (x, pos, table, {"out": torch.empty(1, 2, 64, device=device).expand(4, 2, 64)}),
        (x, pos, table, {"error": torch.zeros(1, device=device)}),
        (x.clone().requires_grad_(), pos, table, {"out": torch.empty(4, 2, 64, device=device)}),
    ]
    buf = torch.randn(6, 2, 64, device=device)
    bad.append((buf[:4], pos, table, {"out": buf[1:5]}))  # a shifted overlap
    for a, p, t, kw in bad:
        with pytest.raises(ValueError):
            rotary(a, p, t, **kw)
    assert rotary(x[:0], pos[:0], table).shape == (0, 2, 64)
    for args in ((3, 10), (0, 10), (64, 0)):
        with pytest.raises(ValueError):
            rotary_table(*args, device="cpu")
    for sc in ({"type": "spiral", "factor": 2.0}, {"type": "linear", "factor": 0.5}, {"type": "yarn", "factor": 2.0},
               {"type": "llama3", "factor": 2.0, "original_max_pos": 8, "low_freq_factor": 4, "high_freq_factor": 1}):
        with pytest.raises(ValueError):
            rotary_inv_freq(64, scaling=sc)


def test_scaled_frequencies():
    R, theta, n = 128, 5e5, 8192
    base, _ = rotary_inv_freq(R, theta)
    for i in (0, 1, 31, 63):
        assert float(base[i]) == pytest.approx(theta ** (-2 * i / R), rel=1e-14)
    lin, m = rotary_inv_freq(R, theta, {"type": "linear", "factor": 4.0})
    assert m == 1.0 and torch.equal(lin, base / 4)
    ntk, _ = rotary_inv_freq(R, theta, {"type": "ntk", "factor": 4.0})
    assert float(ntk[0]) == 1.0 and float(ntk[-1]) == pytest.approx(float(base[-1]) / 4, rel=1e-12)
    l3, _ = rotary_inv_freq(R, theta, {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                                       "high_freq_factor": 4.0, "original_max_pos": n})
    yarn, my = rotary_inv_freq(R, theta, {"type": "yarn", "factor": 8.0, "original_max_pos": n})
    for i in range(R // 2):
        turns = n * float(base[i]) / (2 * math.pi)
        want = float(base[i]) if turns > 4 else float(base[i]) / 8 if turns < 1 else \
            float(base[i]) * ((turns - 1) / 3 + (1 - (turns - 1) / 3) / 8)
        assert float(l3[i]) == pytest.approx(want, rel=1e-12)
        if turns > 40:
            assert float(yarn[i]) == float(base[i])
        if turns < 0.8:
            assert float(yarn[i]) == pytest.approx(float(base[i]) / 8, rel=1e-12)
        assert float(base[i]) / 8 * (1 - 1e-12) <= float(yarn[i]) <= float(base[i])
    assert my == pytest.approx(0.1 * math.log(8) + 1)
    # far positions keep their phase: the angle is formed in 64 bits
    t = rotary_table(R, 131072, theta, device="cpu")
    assert float(t[131071, 1, 1]) == pytest.approx(math.sin(131071 * theta ** (-2 / R)), abs=1e-6)


@pytest.mark.gpu
def test_large_offsets_streams_and_capture(dev):
    """Row offsets beyond 2^31 elements, a side stream, a captured and replayed call."""
    table = rotary_table(64, 64, device=dev)
    # two rows 2^31 + 2^8 elements apart (a strided view of one 4.3 GB buffer)
    far = torch.zeros(2 ** 31 + 2 ** 9, device=dev, dtype=torch.bfloat16)
    x = far.as_strided((2, 2, 64), (2 ** 31 + 2 ** 8, 64, 1))
    x.copy_(torch.randn(2, 2, 64, device=dev))
    pos = torch.tensor([5, 63], dtype=torch.int32, device=dev)
    check(rotary(x, pos, table), x, pos, table)
    del far, x
    x = torch.randn(300, 4, 64, device=dev).bfloat16()
    pos = torch.randint(0, 64, (300,), dtype=torch.int32, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = rotary(x, pos, table)
        g = torch.cuda.CUDAGraph()
        out = torch.empty_like(x)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            rotary(x, pos, table, out=out)
    torch.cuda.current_stream().wait_stream(s)
    check(y, x, pos, table)
    x.copy_(torch.randn(300, 4, 64, device=dev))
    g.replay()
    check(out, x, pos, table)


@pytest.mark.gpu
def test_forward_and_backward_in_a_graph(dev):
    """A captured forward and backward, replayed on new values; an eager pass over the same leaf afterwards."""
    table = rotary_table(64, 64, device=dev)
    x = torch.randn(50, 4, 64, device=dev).bfloat16().requires_grad_()
    dy = torch.randn(50, 4, 64, device=dev).bfloat16()
    pos = torch.randint(0, 64, (50,), dtype=torch.int32, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(rotary(x, pos, table), x, dy)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = rotary(x, pos, table)
        (dx,) = torch.autograd.grad(y, x, dy)
    with torch.no_grad():
        x.copy_(torch.randn(50, 4, 64, device=dev))
        dy.copy_(torch.randn(50, 4, 64, device=dev))
        pos.copy_(torch.randint(0, 64, (50,), dtype=torch.int32, device=dev))
    g.replay()
    check(y.detach(), x.detach(), pos, table)
    check(dx, dy, pos, table, transpose=True)
    (again,) = torch.autograd.grad(rotary(x, pos, table), x, dy)
    assert torch.equal(again, dx)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,R", [(7, 3, 128, 64), (5, 2, 80, 20), (4, 2, 10, 6), (9, 1, 256, 32), (6, 4, 64, 64),
                                     (5003, 9, 128, 32), (26003, 3, 128, 64)])
def test_positions_out_of_range_in_place(T, H, D, R, interleaved, dtype, device):
    """In place on part of the head: a row past the table becomes NaN in all its dimensions, the others and what lies
    between the rows stay as a new output has them."""
    if device == "cpu" and T > 1000:
        pytest.skip("the same math on the host, whatever the number of rows")
    g = torch.Generator().manual_seed(T + R)
    table = rotary_table(R, 50, device=device)
    buf = torch.randn(T, H * D + 16, generator=g).to(dtype).to(device)
    x = buf[:, 8:8 + H * D].view(T, H, D)
    pos = torch.randint(-1, 50, (T,), generator=g, dtype=torch.int32)
    pos[::3] = torch.randint(50, 2 ** 31 - 1, (len(pos[::3]),), generator=g, dtype=torch.int32)
    pos = pos.to(device)
    before, bad = buf.clone(), pos >= 50
    want = rotary(x, pos, table, interleaved=interleaved)
    err = torch.zeros(1, dtype=torch.int32, device=device)
    assert rotary(x, pos, table, interleaved=interleaved, out=x, error=err) is x
    assert int(err) == 1 and x[bad].isnan().all() and want[bad].isnan().all()
    assert torch.equal(x[~bad], want[~bad])
    assert torch.equal(buf[:, :8], before[:, :8]) and torch.equal(buf[:, 8 + H * D:], before[:, 8 + H * D:])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_mode(interleaved, device):
    """A tangent is rotated like the value, with or without a gradient switch; where it would get lost, it is refused."""
    fw = torch.autograd.forward_ad
    T, H, D, R = 9, 3, 64, 32
    table = rotary_table(R, 40, device=device)
    pos = torch.randint(0, 40, (T,), dtype=torch.int32, device=device)
    pos[3] = -1
    x = torch.randn(T, H, D, device=device)
    with fw.dual_level():
        for t in (torch.randn(T, H, D, device=device), torch.randn(1, 1, 1, device=device).expand(T, H, D),
                  torch.randn(D, H, T, device=device).permute(2, 1, 0)):
            with torch.no_grad():
                y, dy = fw.unpack_dual(rotary(fw.make_dual(x, t), pos, table, interleaved=interleaved))
            check(y, x, pos, table, interleaved)
            check(dy, t, pos, table, interleaved)
            y, dy = fw.unpack_dual(rotary(fw.make_dual(x, t), pos, table, interleaved=interleaved, transpose=True))
            check(dy, t, pos, table, interleaved, transpose=True)
        assert fw.unpack_dual(rotary(x, pos, table)).tangent is None
        dual = fw.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="forward-mode"):
            rotary(dual, pos, table, out=torch.empty_like(x))
        with pytest.raises((RuntimeError, NotImplementedError)):  # both modes at once
            rotary(fw.make_dual(x.clone().requires_grad_(), torch.ones_like(x)), pos, table)


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_of_the_table_are_refused(device):
    """The table's gradient would be dropped without a word: refused, with and without a gradient of x."""
    x, pos = torch.randn(3, 2, 64, device=device), torch.arange(3, dtype=torch.int32, device=device)
    table = rotary_table(64, 8, device=device).requires_grad_()
    for a in (x, x.clone().requires_grad_()):
        with pytest.raises(ValueError, match="table"):
            rotary(a, pos, table)
        with torch.no_grad():
            check(rotary(a, pos, table), x, pos, table.detach())
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match="table"):
            rotary(x, pos, torch.autograd.forward_ad.make_dual(table.detach(), torch.ones_like(table)))


@pytest.mark.gpu
def test_rows_up_to_31_bits(dev):
    """2^31 - 1 rows: the number of blocks does not overflow."""
    T = 2 ** 31 - 1
    table = rotary_table(2, 4, device=dev)
    pos = torch.ones(T, dtype=torch.int32, device=dev)
    pos[-1] = 3
    x = torch.tensor([[[1.0, 0.5]]], dtype=torch.bfloat16, device=dev).expand(T, 1, 2)
    y = rotary(x, pos, table)
    for rows in (slice(0, 300), slice(T // 2, T // 2 + 300), slice(T - 300, T)):
        check(y[rows], x[rows], pos[rows], table)


def test_scalings_out_of_range_are_refused():
    """Numbers for which a scaling has no meaning: a ramp that runs backwards, turns over no positions, log(theta) <= 0."""
    yarn = {"type": "yarn", "factor": 2.0, "original_max_pos": 64}
    l3 = {"type": "llama3", "factor": 2.0, "original_max_pos": 64}
    for sc, theta in ((yarn, 1.0), (yarn, 0.5), ({**yarn, "beta_fast": 1.0, "beta_slow": 2.0}, 1e4),
                      ({**yarn, "beta_slow": 0.0}, 1e4), ({**yarn, "original_max_pos": -4}, 1e4),
                      ({**l3, "original_max_pos": -4}, 1e4)):
        with pytest.raises(ValueError, match="rotary"):
            rotary_inv_freq(64, theta, sc)
    for sc in (yarn, l3, {**yarn, "beta_fast": 4.0, "beta_slow": 4.0}, {**l3, "low_freq_factor": 0.0}):
        inv, _ = rotary_inv_freq(64, 1e4, sc)
        assert torch.isfinite(inv).all()
