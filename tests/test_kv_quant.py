"""The 8-bit paged KV cache: written, read back, attended to, against plain 64-bit math."""
import math

import pytest
import torch

from turbol_b200.ops import reference as ref
from turbol_b200.ops.kv_cache import decode_attention_quant, kv_quant_read, kv_quant_write, quant_kv_cache
from turbol_b200.ops.rotary import rotary, rotary_table

F8 = torch.float8_e4m3fn
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def pages(lens, bs, device, spare=2, seed=0):
    """A block table over a shuffled pool that is larger than needed."""
    per = max(1, max(-(-n // bs) for n in lens))
    n = len(lens) * per + spare
    perm = torch.randperm(n, generator=torch.Generator().manual_seed(seed))[: len(lens) * per]
    return perm.view(len(lens), per).to(torch.int32).to(device), n


def tokens_of(lens, device):
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)]).to(torch.int32).to(device)
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).to(device)
    return seq, pos


def where(seq, pos, table, bs):
    return table[seq.long(), (pos // bs).long()].long(), (pos % bs).long()


def bits(c):
    return c.view(torch.uint8)


# ------------------------------------------------------------------ write
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lens,Hk,D,bs", [([1], 1, 64, 16), ([5, 0, 17], 2, 128, 16), ([33, 1, 40], 8, 128, 7),
                                          ([130], 3, 256, 64), ([9, 3], 1, 64, 1), ([300, 2, 77], 2, 128, 24)])
def test_write_codes_and_scales(lens, Hk, D, bs, dtype, device):
    """Unrotated rows: the scale's and the code's roundings are IEEE ones, so both equal the formula's bits; slots that
    no token names stay as they were."""
    g = torch.Generator().manual_seed(len(lens) + D)
    table, nb = pages(lens, bs, device)
    seq, pos = tokens_of(lens, device)
    T = seq.numel()
    k = (torch.randn(T, Hk, D, generator=g) * 5).to(dtype).to(device)
    v = (torch.randn(T, Hk, D, generator=g) * 0.01).to(dtype).to(device)
    k[0, 0] = 0  # a row of zeros
    v[T // 2, Hk - 1, 3] = 900.0  # one loud channel
    c = quant_kv_cache(nb, Hk, bs, D, device)
    for t in c[:2]:
        bits(t).fill_(77)
    for t in c[2:]:
        t.fill_(-5.0)
    assert kv_quant_write(k, v, seq, pos, table, *c) is None
    blk, slot = where(seq, pos, table, bs)
    seen = torch.zeros(nb, bs, dtype=torch.bool, device=device)
    seen[blk, slot] = True
    for x, code, scale in ((k, c.kc, c.ks), (v, c.vc, c.vs)):
        amax = x.float().abs().amax(-1).clamp_min(2.0 ** -90)
        top = torch.full_like(amax, 448.0)  # tensor by tensor: torch turns a scalar operand into a reciprocal product
        assert torch.equal(scale[blk, :, slot], amax / top)
        assert torch.equal(bits(code)[blk, :, slot], bits((x.float() * (top / amax)[..., None]).to(F8)))
        assert (bits(code).transpose(1, 2)[~seen] == 77).all() and (scale.transpose(1, 2)[~seen] == -5.0).all()
        # what the codes stand for is within half a step: 2^-4 of the value, or half of the smallest code (2^-10)
        back = bits(code)[blk, :, slot].view(F8).double() * scale[blk, :, slot].double()[..., None]
        tol = x.double().abs() * (2.0 ** -4 + 2.0 ** -20) + scale[blk, :, slot].double()[..., None] * 2.0 ** -10
        assert ((back - x.double()).abs() <= tol).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("Hq,Hk,D,R", [(12, 2, 128, 128), (4, 4, 64, 32), (3, 1, 256, 64), (8, 2, 128, 120),
                                       (2, 2, 64, 8)])
def test_write_with_rotary(Hq, Hk, D, R, interleaved, dtype, device):
    lens, bs = [19, 1, 6], 16
    table, nb = pages(lens, bs, device)
    seq, pos = tokens_of(lens, device)
    T = seq.numel()
    rt = rotary_table(R, 19, 1e4, device=device)
    rows = torch.randn(T, (Hq + 2 * Hk) * D + 8, device=device).to(dtype)[:, :(Hq + 2 * Hk) * D].view(T, Hq + 2 * Hk, D)
    q, k, v = rows[:, :Hq], rows[:, Hq:Hq + Hk], rows[:, Hq + Hk:]
    before = rows.clone()
    c = quant_kv_cache(nb, Hk, bs, D, device)
    out = kv_quant_write(k, v, seq, pos, table, *c, q=q, table=rt, interleaved=interleaved)
    assert torch.equal(rows, before)
    t64 = rt.double()
    eq, ek = (ref.rotary(x.double(), pos, t64, interleaved) for x in (q, k))
    mq = (q.double().abs().amax(-1, keepdim=True) * 2)
    assert ((out.double() - eq).abs() <= HALF_STEP[dtype] * eq.abs() * 1.001 + 3 * 2.0 ** -24 * mq).all()
    blk, slot = where(seq, pos, table, bs)
    scale = c.ks[blk, :, slot].double()
    amax = ek.abs().amax(-1)
    # rotated values are off by 3 * 2^-24 of the products, the scale by one rounding more
    big = k.double().abs().amax(-1) * 2
    assert ((scale * 448 - amax).abs() <= amax * 2.0 ** -23 + 3 * 2.0 ** -24 * big).all()
    back = bits(c.kc)[blk, :, slot].view(F8).double() * scale[..., None]
    tol = ek.abs() * (2.0 ** -4 + 2.0 ** -20) + scale[..., None] * 2.0 ** -10 + 4 * 2.0 ** -24 * big[..., None]
    assert ((back - ek).abs() <= tol).all()
    # v is not rotated
    av = v.float().abs().amax(-1)
    assert torch.equal(bits(c.vc)[blk, :, slot], bits((v.float() * (torch.full_like(av, 448.0) / av)[..., None]).to(F8)))
    # in place, and without q: the same
    c2 = quant_kv_cache(nb, Hk, bs, D, device)
    assert kv_quant_write(k, v, seq, pos, table, *c2, q=q, table=rt, interleaved=interleaved, q_out=q) is q
    assert torch.equal(q, out) and torch.equal(rows[:, Hq:], before[:, Hq:])
    c3 = quant_kv_cache(nb, Hk, bs, D, device)
    kv_quant_write(k, v, seq, pos, table, *c3, table=rt, interleaved=interleaved)
    for a, b, d in zip(c, c2, c3):
        assert torch.equal(bits(a), bits(b)) and torch.equal(bits(a), bits(d))


@pytest.mark.parametrize("device", DEVICES)
def test_write_strides_and_alignment(device):
    """Rows at odd offsets, expanded rows, heads before tokens: the same codes as from contiguous rows."""
    lens, bs, Hk, D = [37], 16, 2, 64
    table, nb = pages(lens, bs, device)
    seq, pos = tokens_of(lens, device)
    buf = torch.randn(37, Hk * D + 9, device=device).bfloat16()
    heads_first = torch.randn(Hk, 37, D, device=device).bfloat16()
    for k in (buf[:, 1:1 + Hk * D].view(37, Hk, D), buf[:, :D].view(37, 1, D).expand(37, Hk, D),
              heads_first.transpose(0, 1), buf[:1, :Hk * D].view(1, Hk, D).expand(37, Hk, D)):
        a, b = quant_kv_cache(nb, Hk, bs, D, device), quant_kv_cache(nb, Hk, bs, D, device)
        kv_quant_write(k, k, seq, pos, table, *a)
        kv_quant_write(k.contiguous(), k.contiguous(), seq, pos, table, *b)
        for x, y in zip(a, b):
            assert torch.equal(bits(x), bits(y))


@pytest.mark.parametrize("device", DEVICES)
def test_write_padding_bad_indexes_and_extremes(device):
    Hk, D, bs, nb = 2, 64, 4, 5
    table = torch.tensor([[0, 4], [3, 99], [-2, 1]], dtype=torch.int32, device=device)
    #              fine padding padding fine | block 99, block -2, position past the table, sequence past it
    seq = torch.tensor([0, 0, -1, 0, 1, 2, 0, 3], dtype=torch.int32, device=device)
    pos = torch.tensor([3, -1, 0, 7, 4, 1, 8, 0], dtype=torch.int32, device=device)
    k = torch.randn(8, Hk, D, device=device)
    q = torch.randn(8, 3, D, device=device)
    rt = rotary_table(64, 8, device=device)
    c = quant_kv_cache(nb, Hk, bs, D, device)
    err = torch.zeros(1, dtype=torch.int32, device=device)
    kv_quant_write(k[:4], k[:4], seq[:4].contiguous(), pos[:4].contiguous(), table, *c, error=err)
    assert int(err) == 0
    written = c.ks.transpose(1, 2).ne(0).any(-1).nonzero().tolist()
    assert written == [[0, 3], [4, 3]]
    for i in range(4, 8):
        err.zero_()
        kv_quant_write(k[i:i + 1], k[i:i + 1], seq[i:i + 1].contiguous(), pos[i:i + 1].contiguous(), table, *c, error=err)
        assert int(err) == 1
    assert c.ks.transpose(1, 2).ne(0).any(-1).nonzero().tolist() == written
    # with a table of 8 positions, position 8 has no angle: its q row is NaN; padding rows are copied
    err.zero_()
    out = kv_quant_write(k, k, seq, pos, table, *c, q=q, table=rt, error=err)
    assert int(err) == 1 and out[6].isnan().all() and torch.equal(out[1], q[1])
    # a row of denormals, the largest finite values, infinities and NaN
    x = torch.zeros(4, Hk, D, device=device)
    x[0] = 1e-40
    x[1] = 3.4e38
    x[2, :, 5] = float("inf")
    x[3, :, 5] = float("nan")
    s4, p4 = torch.zeros(4, dtype=torch.int32, device=device), torch.arange(4, dtype=torch.int32, device=device)
    kv_quant_write(x, -x, s4, p4, table, *c)
    kk, vv = kv_quant_read(*c, s4, p4, table, dtype=torch.float32)
    assert (kk[0] == 0).all() and torch.isfinite(kk[1]).all() and ((kk[1] - 3.4e38).abs() <= 3.4e38 * 2.0 ** -20).all()
    assert torch.equal(vv[1], -kk[1])
    assert not torch.isfinite(kk[2]).any() and kk[3].isnan().all()


# ------------------------------------------------------------------ read
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lens,Hk,D,bs", [([1], 1, 64, 16), ([5, 0, 17], 2, 128, 16), ([33, 1, 40], 8, 128, 7),
                                          ([130], 3, 256, 64)])
def test_read_back(lens, Hk, D, bs, dtype, device):
    """One fp32 product and one rounding: equal to the same in plain operations; untouched rows stay."""
    g = torch.Generator().manual_seed(3)
    table, nb = pages(lens, bs, device)
    seq, pos = tokens_of(lens, device)
    c = random_cache(nb, Hk, bs, D, device, g)
    order = torch.randperm(seq.numel(), generator=g).to(device)
    seq, pos = seq[order], pos[order]
    pad = torch.tensor([-1], dtype=torch.int32, device=device)
    seq, pos = torch.cat([seq, pad.abs(), seq[:1]]), torch.cat([pos, pad, pos[:1]])  # padding, and a row named twice
    out = tuple(torch.full((seq.numel(), Hk + 1, D + 3), 7.0, device=device, dtype=dtype)[:, :Hk, :D] for _ in range(2))
    r = kv_quant_read(*c, seq, pos, table, out=out)
    assert r[0] is out[0] and r[1] is out[1]
    live = pos >= 0
    blk, slot = where(seq[live], pos[live], table, bs)
    for o, code, scale in ((out[0], c.kc, c.ks), (out[1], c.vc, c.vs)):
        want = (bits(code)[blk, :, slot].view(F8).float() * scale[blk, :, slot][..., None]).to(dtype)
        assert torch.equal(o[live], want) and (o[~live] == 7.0).all()
    new = kv_quant_read(*c, seq, pos, table, dtype=dtype)
    assert torch.equal(new[0][live], out[0][live]) and (new[1][~live] == 0).all()


def random_cache(nb, Hk, bs, D, device, g, k_amp=1.0, v_amp=1.0):
    c = quant_kv_cache(nb, Hk, bs, D, device)
    for code, scale, amp in ((c.kc, c.ks, k_amp), (c.vc, c.vs, v_amp)):
        x = torch.randn(nb, Hk, bs, D, generator=g) * torch.exp(torch.randn(nb, Hk, bs, 1, generator=g)) * amp
        cc, ss = ref.kv_quantise(x)
        bits(code).copy_(bits(cc))
        scale.copy_(ss)
    return c


# ------------------------------------------------------------------ attention
def check_attention(out, q, c, table, lens, scale):
    """Against 64 bits.  The kernel's errors: scores, fp32 sums of D products (half of D roundings each way, 2^-24 of the
    sum of absolute products) and an exponential of relative error 2^-20; weights rounded to fp16 (2^-11, and below
    2^-14 of the largest an absolute 2^-25); fp32 sums over the context; the output's rounding."""
    B, Hq, D = q.shape
    nb, Hk, bs, _ = c.kc.shape
    G = Hq // Hk
    for b, n in enumerate(lens):
        if n <= 0:
            assert (out[b] == 0).all()
            continue
        blk, slot = where(torch.full((n,), b, device=q.device), torch.arange(n, device=q.device), table, bs)
        k, v = ((bits(x)[blk, :, slot].view(F8).double() * s[blk, :, slot].double()[..., None]).transpose(0, 1)
                for x, s in ((c.kc, c.ks), (c.vc, c.vs)))
        vs = c.vs[blk, :, slot].double().t()
        qq = q[b].double().view(Hk, G, D)
        a = qq @ k.transpose(1, 2) * scale
        p = torch.softmax(a, -1)
        e = p @ v
        mag = (qq.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
        ds = 2.0 ** -24 * (D / 2 + 8) * mag + 2.0 ** -20
        tol = (HALF_STEP[q.dtype] * e.abs() * 1.01 + (2.0 ** -11 + 3 * ds + n * 2.0 ** -24) * (p @ v.abs()) +
               n * 2.0 ** -24 * 448 * (p * vs[:, None]).amax(-1, keepdim=True) + (2.0 ** -25 if q.dtype == torch.float16 else 0))
        got = out[b].double().view(Hk, G, D)
        over = (got - e).abs() - tol
        assert not (over > 0).any(), (b, n, float(over.max()), float(tol.max()))
        assert torch.isfinite(got).all()


LENS = [[1], [33], [0, 1, 2, 15], [16, 17, 31, 0, 32, 129], [500, 3, 0, 257], [2049, 1]]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cap", [0, 64, 4096])
def test_attention_all_empty(cap, device):
    """Nothing but empty contexts, in tables without a column, short and long: zeros over what out held."""
    c = quant_kv_cache(3, 2, 16, 128, device)
    q = torch.randn(700, 6, 128, device=device).bfloat16()
    out = torch.full_like(q, float("nan"))
    table = torch.zeros(700, cap // 16, dtype=torch.int32, device=device)
    ctx = torch.zeros(700, dtype=torch.int32, device=device)
    ctx[5] = -3
    decode_attention_quant(q, *c, table, ctx, out=out)
    assert (out == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hk,D,bs", [(12, 2, 128, 16), (32, 8, 128, 16), (4, 4, 64, 1), (8, 1, 256, 64),
                                        (9, 3, 128, 7), (16, 1, 64, 24), (20, 1, 128, 16), (34, 2, 256, 16),
                                        (1, 1, 128, 8), (64, 1, 64, 32)])
def test_attention(Hq, Hk, D, bs, dtype, device):
    for i, lens in enumerate(LENS):
        g = torch.Generator().manual_seed(17 * i + Hq)
        table, nb = pages(lens, bs, device, seed=i)
        c = random_cache(nb, Hk, bs, D, device, g)
        q = (torch.randn(len(lens), Hq, D, generator=g) * 2).to(dtype).to(device)
        ctx = torch.tensor(lens, dtype=torch.int32, device=device)
        out = torch.full_like(q, float("nan"))
        assert decode_attention_quant(q, *c, table, ctx, out=out) is out
        check_attention(out, q, c, table, lens, D ** -0.5)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_ignores_what_lies_behind_a_context(device):
    """NaN, infinities and wild block numbers behind the contexts change no bit; neither do the strides of q and out."""
    lens, Hq, Hk, D, bs = [5, 0, 40, 129], 12, 2, 128, 16
    table, nb = pages(lens, bs, device)
    g = torch.Generator().manual_seed(5)
    c = random_cache(nb, Hk, bs, D, device, g)
    q = torch.randn(4, Hq, D, generator=g).bfloat16().to(device)
    ctx = torch.tensor(lens, dtype=torch.int32, device=device)
    want = decode_attention_quant(q, *c, table, ctx, scale=0.3)
    seq, pos = tokens_of(lens, device)
    blk, slot = where(seq, pos, table, bs)
    seen = torch.zeros(nb, bs, dtype=torch.bool, device=device)
    seen[blk, slot] = True
    for t in c[:2]:
        bits(t).transpose(1, 2)[~seen] = 0x7F
    c.ks.transpose(1, 2)[~seen] = float("inf")
    c.vs.transpose(1, 2)[~seen] = float("nan")
    wild = table.clone()
    for b, n in enumerate(lens):
        wild[b, -(-n // bs):] = 2 ** 31 - 1
    err = torch.zeros(1, dtype=torch.int32, device=device)
    assert torch.equal(decode_attention_quant(q, *c, wild, ctx, scale=0.3, error=err), want) and int(err) == 0
    neg = torch.where(ctx == 0, -7, ctx)
    assert torch.equal(decode_attention_quant(q, *c, table, neg, scale=0.3), want)
    row = torch.randn(4, (Hq + 2) * D + 1, device=device).bfloat16()
    qs = row[:, 1:1 + Hq * D].view(4, Hq, D)
    qs.copy_(q)
    out = torch.full((Hq, 4, D), 3.0, device=device, dtype=torch.bfloat16).transpose(0, 1)
    assert decode_attention_quant(qs, *c, table, ctx, scale=0.3, out=out) is out
    assert torch.equal(out, want)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_bad_blocks_and_lengths(device):
    """A block out of range inside a context, and a context longer than its table: left out, and told."""
    Hq, Hk, D, bs, nb = 4, 2, 64, 4, 8
    g = torch.Generator().manual_seed(9)
    c = random_cache(nb, Hk, bs, D, device, g)
    q = torch.randn(2, Hq, D, generator=g).bfloat16().to(device)
    table = torch.tensor([[1, 50, 3], [4, 5, 6]], dtype=torch.int32, device=device)
    fine = torch.tensor([[1, 3], [4, 5]], dtype=torch.int32, device=device)
    err = torch.zeros(1, dtype=torch.int32, device=device)
    out = decode_attention_quant(q, *c, table, torch.tensor([12, 8], dtype=torch.int32, device=device), error=err)
    assert int(err) == 1
    check_attention(out, q, c, fine, [8, 8], D ** -0.5)
    for n in (13, 2 ** 31 - 1):
        err.zero_()
        out = decode_attention_quant(q[1:], *c, table[1:].contiguous(),
                                     torch.tensor([n], dtype=torch.int32, device=device), error=err)
        assert int(err) == 1
        check_attention(out, q[1:], c, table[1:], [12], D ** -0.5)
        if device == "cpu":
            break  # the reference walks every token
    err.zero_()
    none = torch.full((2, 3), -1, dtype=torch.int32, device=device)
    out = decode_attention_quant(q, *c, none, torch.tensor([12, 1], dtype=torch.int32, device=device), error=err)
    assert (out == 0).all() and int(err) == 1


@pytest.mark.parametrize("device", DEVICES)
def test_attention_wide_ranges(device):
    """Scales that differ by many powers of two between tokens, zero rows, loud and faint queries."""
    lens, Hq, Hk, D, bs = [70], 8, 1, 128, 16
    table, nb = pages(lens, bs, device)
    for i, (ka, va, qa) in enumerate([(1e-6, 1e6, 1e6), (1e6, 1e-6, 1e-6), (1.0, 1e20, 1.0), (1.0, 1e-20, 1.0),
                                      (3e4, 1.0, 1e-4)]):
        g = torch.Generator().manual_seed(i)
        c = random_cache(nb, Hk, bs, D, device, g, ka, va)
        blk, slot = where(torch.zeros(70, device=device), torch.arange(70, device=device), table, bs)
        c.vs[blk[::3], :, slot[::3]] *= 2.0 ** 30  # every third value far louder
        bits(c.vc)[blk[1::3], :, slot[1::3]] = 0  # zero rows with the smallest scale
        c.vs[blk[1::3], :, slot[1::3]] = 2.0 ** -90 / 448
        q = (torch.randn(1, Hq, D, generator=g) * qa).bfloat16().to(device)
        out = decode_attention_quant(q, *c, table, torch.tensor(lens, dtype=torch.int32, device=device))
        check_attention(out, q, c, table, lens, D ** -0.5)
    # a NaN or infinite score inside the context is not hidden
    c.ks[blk[5], 0, slot[5]] = float("nan")
    out = decode_attention_quant(q, *c, table, torch.tensor(lens, dtype=torch.int32, device=device))
    assert out.isnan().all()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    Hk, D, bs, nb, T = 2, 64, 4, 6, 3
    c = quant_kv_cache(nb, Hk, bs, D, device)
    i32 = dict(dtype=torch.int32, device=device)
    table, seq, pos, ctx = torch.zeros(T, 2, **i32), torch.zeros(T, **i32), torch.arange(T, **i32), torch.ones(T, **i32)
    k, q = torch.randn(T, Hk, D, device=device).bfloat16(), torch.randn(T, 4, D, device=device).bfloat16()
    rt = rotary_table(D, 8, device=device)
    odd = quant_kv_cache(nb, Hk, bs, D, device)
    bad_caches = [
        (bits(c.kc), c.vc, c.ks, c.vs), (c.kc, c.vc, c.ks.double(), c.vs), (c.kc, c.vc[:, :1], c.ks, c.vs),
        (c.kc, c.vc, c.ks[:5], c.vs[:5]), (c.kc, c.vc, c.ks, c.vs.transpose(0, 1).contiguous().transpose(0, 1)),
        (c.kc[..., :32], c.vc[..., :32], c.ks, c.vs),
    ]
    for cc in bad_caches:
        with pytest.raises(ValueError):
            kv_quant_write(k, k, seq, pos, table, *cc)
        with pytest.raises(ValueError):
            kv_quant_read(*cc, seq, pos, table)
        with pytest.raises(ValueError):
            decode_attention_quant(q, *cc, table, ctx)
    W = dict(k=k, v=k, seq_of_token=seq, pos=pos, block_table=table, kc=c.kc, vc=c.vc, ks=c.ks, vs=c.vs)
    for change in (dict(k=k.float()), dict(k=k[:2]), dict(k=k[..., :32]), dict(k=k[:, :1], v=k[:, :1]), dict(k=k[0]),
                   dict(k=k.double(), v=k.double()), dict(seq_of_token=seq.long()), dict(pos=pos[:2]),
                   dict(block_table=table.long()), dict(block_table=table[0]), dict(block_table=table.t()),
                   dict(vc=c.kc), dict(vs=c.ks), dict(q=q), dict(table=rt[:, :-1].contiguous()), dict(table=rt.double()),
                   dict(q=q.float(), table=rt), dict(q=q[:2], table=rt), dict(q=q, table=rt, q_out=q[:, :2]),
                   dict(q=q, table=rt, q_out=torch.empty(1, 4, D, device=device, dtype=k.dtype).expand(T, 4, D)),
                   dict(q=q[:, :2], table=rt, q_out=k), dict(error=torch.zeros(1, device=device)),
                   dict(k=k.transpose(1, 2)), dict(q_out=q)):
        with pytest.raises(ValueError):
            kv_quant_write(**{**W, **change})
    wide = torch.randn(T, 8, D, device=device).bfloat16()
    with pytest.raises(ValueError):  # the rotated q would overwrite k
        kv_quant_write(wide[:, 3:5], wide[:, 6:], seq, pos, table, *c, q=wide[:, :4], table=rt, q_out=wide[:, 2:6])
    out = torch.zeros(T, Hk, D, device=device)
    for o in ((out, out), (out, out.clone().bfloat16()), (out[:2], out[:2].clone()),
              (out.double(), out.double().clone()), (out, out[:1].clone().expand(T, Hk, D))):
        with pytest.raises(ValueError):
            kv_quant_read(*c, seq, pos, table, out=o)
    for change in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[0]), dict(q=q[..., :32]), dict(ctx_len=ctx.long()),
                   dict(ctx_len=ctx[:2]), dict(block_table=table[:2]), dict(out=q), dict(out=q.half()),
                   dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(ValueError):
            decode_attention_quant(**{**dict(q=q, kc=c.kc, vc=c.vc, ks=c.ks, vs=c.vs, block_table=table, ctx_len=ctx),
                                      **change})
    for args in ((6, 2, 4, 96), (0, 2, 4, 64), (6, 0, 4, 64), (6, 2, 0, 64)):
        with pytest.raises(ValueError):
            quant_kv_cache(*args, device="cpu")
    # nothing to do
    kv_quant_write(k[:0], k[:0], seq[:0], pos[:0], table, *c)
    assert kv_quant_read(*c, seq[:0], pos[:0], table)[0].shape == (0, Hk, D)
    assert decode_attention_quant(q[:0], *c, table[:0], ctx[:0]).shape == (0, 4, D)
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(c, odd))


@pytest.mark.parametrize("device", DEVICES)
def test_write_attend_read_in_a_row(device):
    """A decode loop: each step rotates, writes one token per sequence and attends; the prompt comes first; at the end
    the whole cache reads back."""
    B, Hq, Hk, D, bs, Lp, steps = 3, 6, 2, 64, 8, 13, 9
    g = torch.Generator().manual_seed(1)
    lens = [Lp + steps] * B
    table, nb = pages(lens, bs, device)
    c = quant_kv_cache(nb, Hk, bs, D, device)
    rt = rotary_table(D, Lp + steps, device=device)
    seq, pos = tokens_of([Lp] * B, device)
    k = torch.randn(B * Lp, Hk, D, generator=g).bfloat16().to(device)
    v = torch.randn(B * Lp, Hk, D, generator=g).bfloat16().to(device)
    kv_quant_write(k, v, seq, pos, table, *c, table=rt)
    err = torch.zeros(1, dtype=torch.int32, device=device)
    seq1 = torch.arange(B, dtype=torch.int32, device=device)
    ks, vs = [ref.rotary(k.double(), pos, rt.double()).view(B, Lp, Hk, D)], [v.double().view(B, Lp, Hk, D)]
    for i in range(steps):
        qkv = torch.randn(B, Hq + 2 * Hk, D, generator=g).bfloat16().to(device)
        p = torch.full((B,), Lp + i, dtype=torch.int32, device=device)
        q = kv_quant_write(qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], seq1, p, table, *c, q=qkv[:, :Hq], table=rt, error=err)
        out = decode_attention_quant(q, *c, table, p + 1, error=err)
        check_attention(out, q, c, table, [Lp + i + 1] * B, D ** -0.5)
        ks.append(ref.rotary(qkv[:, Hq:Hq + Hk].double(), p, rt.double())[:, None])
        vs.append(qkv[:, Hq + Hk:].double()[:, None])
    seq, pos = tokens_of(lens, device)
    rk, rv = kv_quant_read(*c, seq, pos, table, dtype=torch.float32)
    for got, want in ((rk, torch.cat(ks, 1)), (rv, torch.cat(vs, 1))):
        want = want.reshape(-1, Hk, D)
        amax = want.abs().amax(-1, keepdim=True)
        # half a step of e4m3, or half of its smallest code at the row's scale; the read's and the rotation's roundings
        tol = want.abs() * (2.0 ** -4 + 2.0 ** -20) + amax * (2.0 ** -10 / 448 + 2.0 ** -20)
        assert ((got.double() - want).abs() <= tol).all()
    assert int(err) == 0


# ------------------------------------------------------------------ GPU only
@pytest.mark.gpu
@pytest.mark.parametrize("lens,Hq,Hk,D,bs", [([40000, 7], 8, 2, 128, 16), ([9000], 32, 1, 64, 64), ([20000], 2, 2, 256, 16),
                                             ([768] * 300, 12, 2, 128, 16), ([0, 5, 900] * 100, 20, 1, 128, 16),
                                                ([60000, 0, 2000], 16, 1, 256, 16), ([100000], 1, 1, 128, 64),
                                                ([30000, 30000], 12, 1, 64, 7), ([3000] * 40, 16, 1, 256, 64)])
def test_attention_split_and_joined(lens, Hq, Hk, D, bs, dev):
    g = torch.Generator().manual_seed(2)
    table, nb = pages(lens, bs, dev)
    c = random_cache(nb, Hk, bs, D, dev, g)
    q = torch.randn(len(lens), Hq, D, generator=g).bfloat16().to(dev)
    ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = decode_attention_quant(q, *c, table, ctx, out=torch.full_like(q, float("nan")))
    some = list(range(0, len(lens), max(1, len(lens) // 12)))
    check_attention(out[some], q[some], c, table[some], [lens[i] for i in some], D ** -0.5)
    for _ in range(3):  # the joins have a fixed order
        assert torch.equal(decode_attention_quant(q, *c, table, ctx, out=torch.full_like(q, float("nan"))), out)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_read_at_every_alignment(D, dtype, device):
    """Rows that start on multiples of 32, 16 and fewer bytes: code * scale rounded once, and the gaps as they were."""
    lens, Hk, bs = [37, 5], 3, 8
    table, nb = pages(lens, bs, device)
    c = random_cache(nb, Hk, bs, D, device, torch.Generator().manual_seed(6))
    seq, pos = tokens_of(lens, device)
    blk, slot = where(seq, pos, table, bs)
    want = [(bits(x)[blk, :, slot].view(F8).double() * s[blk, :, slot].double()[..., None]).float().to(dtype)
            for x, s in ((c.kc, c.ks), (c.vc, c.vs))]
    T, pad = pos.numel(), 32
    for shift in (0, 1, 2, 4, 8, 12, 16):
        buf = [torch.full((T * Hk * (D + pad) + shift,), 7.0, dtype=dtype, device=device) for _ in range(2)]
        rows = [b[shift:].view(T, Hk, D + pad) for b in buf]
        kv_quant_read(*c, seq, pos, table, out=(rows[0][..., :D], rows[1][..., :D]))
        for b, r, w in zip(buf, rows, want):
            assert torch.equal(r[..., :D], w)
            assert (r[..., D:] == 7).all() and (b[:shift] == 7).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_write_at_every_alignment(D, dtype, device):
    """Rows that start on multiples of 32, 16 and fewer bytes: the formula's bits, with 1 to 9 KV heads in flight."""
    for Hk, shift in ((1, 0), (2, 1), (3, 2), (5, 4), (9, 8), (4, 12), (2, 16)):
        lens, bs = [37, 1, 5], 8
        table, nb = pages(lens, bs, device)
        seq, pos = tokens_of(lens, device)
        T, pad = pos.numel(), 32
        g = torch.Generator().manual_seed(D + shift)
        rows = [torch.randn(T * Hk * (D + pad) + shift, generator=g).to(dtype).to(device)[shift:].view(T, Hk, D + pad)
                for _ in range(2)]
        c = quant_kv_cache(nb, Hk, bs, D, device)
        kv_quant_write(rows[0][..., :D], rows[1][..., :D], seq, pos, table, *c)
        blk, slot = where(seq, pos, table, bs)
        for r, code, scale in ((rows[0], c.kc, c.ks), (rows[1], c.vc, c.vs)):
            cc, ss = ref.kv_quantise(r[..., :D].cpu())
            assert torch.equal(bits(code)[blk, :, slot].cpu(), bits(cc)) and torch.equal(scale[blk, :, slot].cpu(), ss)


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_are_refused(device):
    """No silent break in an autograd graph: outside no_grad, what requires a gradient raises, and inside it runs."""
    i32 = dict(dtype=torch.int32, device=device)
    c = quant_kv_cache(2, 1, 16, 64, device)
    table, seq, pos, ctx = torch.zeros(2, 1, **i32), torch.zeros(2, **i32), torch.arange(2, **i32), torch.ones(2, **i32)
    x, q = torch.ones(2, 1, 64, device=device).bfloat16(), torch.ones(2, 4, 64, device=device).bfloat16()
    rt, leaf = rotary_table(64, 8, device=device), lambda t: t.clone().requires_grad_()
    calls = [lambda: kv_quant_write(leaf(x), x, seq, pos, table, *c), lambda: kv_quant_write(x, leaf(x), seq, pos, table, *c),
             lambda: kv_quant_write(x, x, seq, pos, table, *c, q=leaf(q), table=rt),
             lambda: kv_quant_write(x, x, seq, pos, table, *c, q=q, q_out=leaf(q), table=rt),
             lambda: kv_quant_read(*c, seq, pos, table, out=(leaf(x), x.clone())),
             lambda: decode_attention_quant(leaf(q), *c, table, ctx),
             lambda: decode_attention_quant(q, *c, table, ctx, out=leaf(q))]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("device", DEVICES)
def test_sizes_past_31_bits_are_refused(device):
    """Views and empty tensors of sizes that the kernels do not count to; nothing of them is in memory."""
    i32 = dict(dtype=torch.int32, device=device)
    c = quant_kv_cache(2, 1, 16, 64, device)
    one, table = torch.zeros(1, **i32), torch.zeros(1, 2, **i32)
    many = torch.zeros(1, 1, 64, device=device).bfloat16().expand(1, 1 << 25, 64)
    with pytest.raises(ValueError, match="2\\^31"):
        decode_attention_quant(many, *c, table, one)
    with pytest.raises(ValueError, match="2\\^31"):
        rotary(torch.zeros(1, 1, 2, device=device).expand(1, 1 << 30, 2), one, rotary_table(2, 4, device=device))
    none = torch.zeros(0, device=device)
    for shape in ((0, 1 << 32, 16, 64), (0, 1 << 25, 16, 64), (0, 1, 1 << 31, 64)):
        kc, ks = none.to(F8).expand(0).reshape(shape), none.reshape(shape[:3])
        with pytest.raises(ValueError, match="2\\^31"):
            decode_attention_quant(torch.zeros(1, 2, 64, device=device).bfloat16(), kc, kc.clone(), ks, ks.clone(), table, one)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,Hq,Hk,D,bs", [([0, 1, 17, 900, 31] * 60, 16, 1, 128, 16), ([0, 1, 17, 900, 31] * 60, 40, 2, 64, 7),
                                             ([0, 3, 400] * 120, 33, 1, 256, 64), ([50000, 3, 0], 32, 1, 128, 16),
                                             ([70000], 9, 1, 64, 8), ([20000, 20000], 17, 1, 256, 24),
                                             ([90000], 24, 1, 64, 64), ([5000] * 30, 128, 2, 128, 128)])
def test_attention_many_heads_on_one(lens, Hq, Hk, D, bs, dtype, dev):
    """9 and more query heads on a KV head, with fewer than eight for some of the warps that share its pages."""
    g = torch.Generator().manual_seed(3)
    table, nb = pages(lens, bs, dev)
    c = random_cache(nb, Hk, bs, D, dev, g)
    q = torch.randn(len(lens), Hq, D, generator=g).to(dtype).to(dev)
    ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = decode_attention_quant(q, *c, table, ctx, out=torch.full_like(q, float("nan")))
    some = list(range(0, len(lens), max(1, len(lens) // 12)))
    check_attention(out[some], q[some], c, table[some], [lens[i] for i in some], D ** -0.5)
    assert torch.isfinite(out).all()
    # the same bits again, and from rows without alignment
    row = torch.zeros(len(lens), Hq * D + 1, dtype=dtype, device=dev)
    row[:, 1:] = q.view(len(lens), -1)
    for x in (q, row[:, 1:].view(len(lens), Hq, D)):
        assert torch.equal(decode_attention_quant(x, *c, table, ctx, out=torch.full_like(q, float("nan"))), out)


@pytest.mark.gpu
def test_streams_and_two_captured_graphs(dev):
    """Two graphs of the same call on different data, replayed in turn and at once on two streams; contexts that grow
    between replays are read from the device."""
    Hq, Hk, D, bs = 12, 2, 128, 16
    lens = [3000, 100, 1, 777]
    table, nb = pages([3100] * 4, bs, dev)
    g = torch.Generator().manual_seed(4)
    sets = []
    for _ in range(2):
        c = random_cache(nb, Hk, bs, D, dev, g)
        q = torch.randn(4, Hq, D, generator=g).bfloat16().to(dev)
        ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
        out = torch.empty_like(q)
        decode_attention_quant(q, *c, table, ctx, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            decode_attention_quant(q, *c, table, ctx, out=out)
        sets.append((c, q, ctx, out, graph, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for extra in (0, 1, 50):
        for c, q, ctx, out, graph, s in sets:
            ctx.copy_(torch.tensor(lens, dtype=torch.int32) + extra)
            out.zero_()
        torch.cuda.synchronize()
        for c, q, ctx, out, graph, s in sets:
            with torch.cuda.stream(s):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for c, q, ctx, out, graph, s in sets:
            check_attention(out, q, c, table, [n + extra for n in lens], D ** -0.5)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(dev):
    """Codes further than 2^32 bytes into the pool."""
    Hq, Hk, D, bs = 8, 8, 128, 64
    nb = 2 ** 32 // (Hk * bs * D) + 40
    c = quant_kv_cache(nb, Hk, bs, D, dev)
    n = 200
    table = torch.arange(nb - 4, nb, dtype=torch.int32, device=dev).view(1, 4)
    seq, pos = tokens_of([n], dev)
    k = torch.randn(n, Hk, D, device=dev).bfloat16()
    v = torch.randn(n, Hk, D, device=dev).bfloat16()
    kv_quant_write(k, v, seq, pos, table, *c)
    kk, vv = kv_quant_read(*c, seq, pos, table)
    for got, x in ((kk, k), (vv, v)):
        codes, s = ref.kv_quantise(x)
        assert torch.equal(got, (codes.float() * s[..., None]).bfloat16())
    q = torch.randn(1, Hq, D, device=dev).bfloat16()
    out = decode_attention_quant(q, *c, table, torch.tensor([n], dtype=torch.int32, device=dev))
    check_attention(out, q, c, table, [n], D ** -0.5)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("Hq,Hk,D,R", [(5, 2, 128, 128), (3, 1, 64, 24), (2, 2, 256, 128)])
def test_write_with_rotary_at_every_alignment(Hq, Hk, D, R, interleaved, dtype, device):
    """A table on any multiple of 8 bytes, rows on any multiple of their elements, in every combination: the bits that
    aligned ones give."""
    lens, bs = [19, 1, 6], 16
    table, nb = pages(lens, bs, device)
    seq, pos = tokens_of(lens, device)
    T, H = seq.numel(), Hq + 2 * Hk
    g = torch.Generator().manual_seed(R)
    rt = rotary_table(R, 19, 1e4, device=device)
    x = torch.randn(T, H, D, generator=g).to(dtype).to(device)
    c = quant_kv_cache(nb, Hk, bs, D, device)
    want = kv_quant_write(x[:, Hq:Hq + Hk], x[:, Hq + Hk:], seq, pos, table, *c, q=x[:, :Hq], table=rt,
                          interleaved=interleaved)
    for floats, shift in ((2, 0), (4, 0), (6, 0), (0, 1), (2, 1), (2, 4), (0, 3)):
        t = torch.zeros(rt.numel() + 8, device=device)[floats:floats + rt.numel()].view(rt.shape)
        t.copy_(rt)
        assert t.data_ptr() % 16 == floats * 4 % 16
        row = torch.zeros(T * H * D + shift, dtype=dtype, device=device)[shift:].view(T, H, D)
        row.copy_(x)
        d = quant_kv_cache(nb, Hk, bs, D, device)
        q = kv_quant_write(row[:, Hq:Hq + Hk], row[:, Hq + Hk:], seq, pos, table, *d, q=row[:, :Hq], table=t,
                           interleaved=interleaved)
        assert torch.equal(q, want) and all(torch.equal(bits(a), bits(b)) for a, b in zip(c, d))
        # rotary takes other vectors then, whose products may be fused with the other sum: two results, each within three
        # roundings of 2^-24 of the two products (2 amax at most) and half a step of the exact one
        a, b = (rotary(y, pos, z, interleaved=interleaved).double() for y, z in ((row[:, :Hq], t), (x[:, :Hq], rt)))
        amax = x[:, :Hq].double().abs().amax(-1, keepdim=True)
        assert ((a - b).abs() <= 2 * (HALF_STEP[dtype] * 1.01 * a.abs().maximum(b.abs()) + 6 * 2.0 ** -24 * amax)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("max_pos", [64, 8])
def test_write_padding_by_sequence(max_pos, interleaved, device):
    """A negative sequence is padding whatever its position, even one past the table: its q row is copied, nothing is
    written, and it is no error."""
    Hq, Hk, D, bs, nb = 3, 2, 64, 16, 4
    g = torch.Generator().manual_seed(max_pos)
    seq = torch.tensor([0, -1, 0, -1, -2 ** 31, -1], dtype=torch.int32, device=device)
    pos = torch.tensor([3, 5, 7, 20, 63, 2 ** 31 - 1], dtype=torch.int32, device=device)
    table = torch.tensor([[2, 1]], dtype=torch.int32, device=device)
    q, k, v = (torch.randn(6, h, D, generator=g).bfloat16().to(device) for h in (Hq, Hk, Hk))
    rt = rotary_table(D, max_pos, device=device)
    c, err = quant_kv_cache(nb, Hk, bs, D, device), torch.zeros(1, dtype=torch.int32, device=device)
    out = kv_quant_write(k, v, seq, pos, table, *c, q=q, table=rt, interleaved=interleaved, error=err)
    pad = seq < 0
    assert torch.equal(out[pad], q[pad]) and int(err) == 0
    assert torch.equal(out[~pad], rotary(q, pos.clamp_max(7), rt, interleaved=interleaved)[~pad])
    assert not torch.equal(out[~pad], q[~pad])
    for s in (c.ks, c.vs):
        assert s.transpose(1, 2).ne(0).any(-1).nonzero().tolist() == [[2, 3], [2, 7]]
    # in place
    assert kv_quant_write(k, v, seq, pos, table, *c, q=q, table=rt, interleaved=interleaved, q_out=q, error=err) is q
    assert torch.equal(q, out) and int(err) == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("Hq,D,n", [(4, 64, 4000), (8, 128, 700), (20, 128, 4000), (3, 256, 2000)])
@pytest.mark.parametrize("B,v_scale", [(1, 1 / 448), (600, 1 / 448), (1, 128.0), (600, 128.0)])
def test_attention_huge_scores(B, v_scale, Hq, D, n, device):
    """Scores near 2^27, where neighbouring fp32 numbers are 16 apart, that creep up from tile to tile: the weights stay
    finite, so equal values average to themselves."""
    if device == "cpu" and B > 1:
        pytest.skip("the host's plain math, sequence by sequence")
    Hk, bs = 1, 16
    nb = -(-n // bs)
    c = quant_kv_cache(nb, Hk, bs, D, device)
    bits(c.kc).fill_(0x7E), bits(c.vc).fill_(0x7E)  # 448
    step = torch.arange(nb, device=device, dtype=torch.float64)[:, None, None] * 2.0 ** -23
    c.ks.copy_(((1 + step) / 512).expand_as(c.ks))
    c.vs.fill_(v_scale)
    table = torch.arange(nb, dtype=torch.int32, device=device).repeat(B, 1)
    ctx = torch.full((B,), n, dtype=torch.int32, device=device)
    for dtype in (torch.bfloat16, torch.float16):
        q = torch.ones(B, Hq, D, dtype=dtype, device=device)
        for top in (1.0, 1.37, 1.9):  # several places between two powers of two
            scale = top * 2.0 ** 27 / math.log2(math.e) / (448 / 512 * D)
            out = decode_attention_quant(q, *c, table, ctx, scale=scale)
            # values 448 * fl(1 / 448), off by 2^-24; rounded weights over their unrounded sum, and the output's rounding
            assert ((out.double() / (448 * v_scale) - 1).abs() <= HALF_STEP[dtype] * 1.01 + 2.0 ** -11 + n * 2.0 ** -22).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,D", [(1, 64), (12, 64), (2, 128)])
def test_attention_keeps_a_long_faint_tail(Hq, D, dev):
    """One loud token, whose value is zero but in dimension 0, and 2^18 faint ones, each 2^-25 of it: they make up the
    other dimensions.  Every sequence reads the same pages, and there are as many as warps, so that the loud token and
    nearly all of its tail are one warp's."""
    n, bs, Hk = 1 << 18, 64, 1
    B = 2368 if D == 64 else 1776
    nb = n // bs
    g = torch.Generator().manual_seed(D)
    c = quant_kv_cache(nb, Hk, bs, D, dev)
    tail = math.log(2.0) * (25.02 + 0.2 * torch.rand(nb, Hk, bs, generator=g))  # how far below the loud token's score
    bits(c.kc).fill_(0xFE)  # -448
    c.ks.copy_(tail / 448)
    c.ks[0, 0, 0] = 0.0
    v = 1.5 + torch.rand(nb, Hk, bs, D, generator=g) / 2
    v[0, 0, 0] = 0.0
    v[..., 0] = 2.0  # one scale for all
    cc, ss = ref.kv_quantise(v)
    bits(c.vc).copy_(bits(cc))
    c.vs.copy_(ss)
    table = torch.arange(nb, dtype=torch.int32, device=dev).repeat(B, 1)
    ctx = torch.full((B,), n, dtype=torch.int32, device=dev)
    q = torch.ones(B, Hq, D, dtype=torch.float16, device=dev)
    out = decode_attention_quant(q, *c, table, ctx, scale=1.0 / D).double()
    p = torch.softmax(-448 * c.ks.double().view(-1), 0)
    e = p @ (bits(c.vc).view(F8).double().view(n, D) * c.vs.double().view(n, 1))
    # The output's rounding and the weights' to fp16: 2^-11 relative, or where they are below 2^-14 absolute, 2^-25 for a
    # largest weight of at least 2^7, so n * 2^-32 in all for values up to 2.  Scores near 18, off by 2^-24 (D / 2 + 8)
    # of that.  Sums in fp32 of n / 16 steps: 16 products are added to the numerator in one, each perhaps cut off at 2^-24
    # of the sum, and two weights to a denominator in two roundings of 2^-24.
    tol = e * (2.0 ** -11 * 2.01 + 3 * 2.0 ** -24 * (D / 2 + 8) * 18 + n / 16 * (17 + 2) * 2.0 ** -24) + n * 2.0 ** -32 * 2
    assert (e[1:] > 20 * tol[1:]).all()  # a lost tail would be seen
    over = (out - e).abs() - tol
    assert not (over > 0).any(), (float(over.max()), float(tol.max()))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("Hq,Hk,D,bs", [(12, 2, 128, 16), (4, 4, 64, 7), (8, 1, 256, 64), (20, 1, 128, 16)])
def test_attention_infinite_scores(Hq, Hk, D, bs, device):
    """Scores of -inf: a token of weight zero beside finite ones; NaN, as the formula's 0 / 0, where a context has no
    other; and zeros still for contexts without a token that counts."""
    for lens in ([1], [40, 0, 1], [5000, 3], [300] * 160 if device != "cpu" else [300, 2]):
        table, nb = pages(lens, bs, device)
        g = torch.Generator().manual_seed(len(lens))
        c = random_cache(nb, Hk, bs, D, device, g)
        q = (torch.randn(len(lens), Hq, D, generator=g).abs() + 0.01).bfloat16().to(device)
        ctx = torch.tensor(lens, dtype=torch.int32, device=device)
        loud = quant_kv_cache(nb, Hk, bs, D, device)
        for a, b in zip(loud, c):
            bits(a).copy_(bits(b))
        # the keys of every context but its last token: all dimensions negative, times infinity
        seq, pos = tokens_of(lens, device)
        first = pos < ctx[seq.long()] - 1
        blk, slot = where(seq, pos, table, bs)
        code = bits(loud.kc).transpose(1, 2)[blk, slot]
        bits(loud.kc).transpose(1, 2)[blk, slot] = torch.where(code & 0x7F == 0, 0x81, code | 0x80).to(torch.uint8)
        loud.ks.transpose(1, 2)[blk[first], slot[first]] = float("inf")
        out = decode_attention_quant(q, *loud, table, ctx)
        last = (ctx - 1).clamp_min(0)
        lb, ls = where(torch.arange(len(lens), device=device), last, table, bs)
        v = bits(loud.vc)[lb, :, ls].view(F8).double() * loud.vs[lb, :, ls].double()[..., None]
        v = v.repeat_interleave(Hq // Hk, 1)
        # one weight, exact but for its rounding to fp16 and the output's
        tol = v.abs() * (2.0 ** -8 * 1.01 + 2.0 ** -11 + 2.0 ** -20)
        assert ((out.double() - v).abs() <= tol)[ctx > 0].all() and (out[ctx == 0] == 0).all()
        loud.ks.transpose(1, 2)[blk, slot] = float("inf")
        out = decode_attention_quant(q, *loud, table, ctx)
        assert out[ctx > 0].isnan().all() and (out[ctx == 0] == 0).all()
        err = torch.zeros(1, dtype=torch.int32, device=device)
        out = decode_attention_quant(q, *loud, torch.full_like(table, -1), ctx, error=err)
        assert (out == 0).all() and int(err) == 1


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_is_refused(device):
    """A tangent would get lost, and torch.no_grad() leaves forward mode on: refused, inside it too."""
    fw = torch.autograd.forward_ad
    i32 = dict(dtype=torch.int32, device=device)
    c = quant_kv_cache(2, 1, 16, 64, device)
    table, seq, pos, ctx = torch.zeros(2, 1, **i32), torch.zeros(2, **i32), torch.arange(2, **i32), torch.ones(2, **i32)
    x, q = torch.ones(2, 1, 64, device=device).bfloat16(), torch.ones(2, 4, 64, device=device).bfloat16()
    rt = rotary_table(64, 8, device=device)
    with fw.dual_level(), torch.no_grad():
        def dual(t):
            return fw.make_dual(t.clone(), torch.ones_like(t))

        for call in (lambda: kv_quant_write(dual(x), x, seq, pos, table, *c),
                     lambda: kv_quant_write(x, dual(x), seq, pos, table, *c),
                     lambda: kv_quant_write(x, x, seq, pos, table, *c, q=dual(q), table=rt),
                     lambda: kv_quant_read(*c, seq, pos, table, out=(dual(x), x.clone())),
                     lambda: decode_attention_quant(dual(q), *c, table, ctx),
                     lambda: decode_attention_quant(q, *c, table, ctx, out=dual(q))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_of_scales_and_table_are_refused(device):
    i32 = dict(dtype=torch.int32, device=device)
    c = quant_kv_cache(2, 1, 16, 64, device)
    table, seq, pos, ctx = torch.zeros(2, 1, **i32), torch.zeros(2, **i32), torch.arange(2, **i32), torch.ones(2, **i32)
    x, q = torch.ones(2, 1, 64, device=device).bfloat16(), torch.ones(2, 4, 64, device=device).bfloat16()
    rt = rotary_table(64, 8, device=device).requires_grad_()
    scales = [(c.kc, c.vc, c.ks.clone().requires_grad_(), c.vs), (c.kc, c.vc, c.ks, c.vs.clone().requires_grad_())]
    for call in [lambda: kv_quant_write(x, x, seq, pos, table, *c, q=q, table=rt)] + \
            [f for s in scales for f in (lambda s=s: kv_quant_write(x, x, seq, pos, table, *s),
                                         lambda s=s: kv_quant_read(*s, seq, pos, table),
                                         lambda s=s: decode_attention_quant(q, *s, table, ctx))]:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("device", DEVICES)
def test_scales_past_fp32_are_refused(device):
    """A scale that is finite in 64 bits and infinite in the kernel's 32."""
    i32 = dict(dtype=torch.int32, device=device)
    c = quant_kv_cache(1, 1, 16, 64, device)
    q = torch.zeros(1, 1, 64, device=device).bfloat16()
    args = (q, *c, torch.zeros(1, 1, **i32), torch.ones(1, **i32))
    for scale in (1e39, -1e300, 3e38):  # (3e38 overflows with the factor log2(e))
        with pytest.raises(ValueError, match="scale"):
            decode_attention_quant(*args, scale=scale)
    for scale in (2e38, -2e38, 0.0, 1e-300):
        assert (decode_attention_quant(*args, scale=scale) == 0).all()


def test_attention_far_behind_its_table_on_the_host():
    """A context of 2^31 - 1 tokens over a table of 12: the host does not walk (or hold) the missing ones."""
    Hq, Hk, D, bs, nb = 4, 2, 64, 4, 8
    g = torch.Generator().manual_seed(9)
    c = random_cache(nb, Hk, bs, D, "cpu", g)
    q = torch.randn(2, Hq, D, generator=g).bfloat16()
    table = torch.tensor([[4, 5, 6], [1, 2, 3]], dtype=torch.int32)
    err = torch.zeros(1, dtype=torch.int32)
    out = decode_attention_quant(q, *c, table, torch.tensor([2 ** 31 - 1, 12], dtype=torch.int32), error=err)
    assert int(err) == 1
    check_attention(out, q, c, table, [12, 12], D ** -0.5)
    err.zero_()
    decode_attention_quant(q, *c, table, torch.tensor([12, 12], dtype=torch.int32), error=err)
    assert int(err) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_writes_are_told_to_autograd(device):
    """A backward pass over what a call has overwritten raises, as after torch's own in-place operations."""
    i32 = dict(dtype=torch.int32, device=device)
    c = quant_kv_cache(2, 1, 16, 64, device)
    table, seq, pos, ctx = torch.zeros(2, 1, **i32), torch.zeros(2, **i32), torch.arange(2, **i32), torch.ones(2, **i32)
    x, q = torch.ones(2, 1, 64, device=device), torch.ones(2, 4, 64, device=device)
    rt, half = rotary_table(64, 8, device=device), torch.ones(2, 4, 64, device=device).bfloat16()
    w = torch.ones(1, device=device, requires_grad=True)
    out = (torch.zeros_like(x), torch.zeros_like(x))
    for call, changed in ((lambda: rotary(q, pos, rt, out=q), [q]),
                          (lambda: kv_quant_write(x, x, seq, pos, table, *c), [c.ks, c.vs]),
                          (lambda: kv_quant_write(x, x, seq, pos, table, *c, q=q, table=rt, q_out=q), [c.ks, c.vs, q]),
                          (lambda: kv_quant_read(*c, seq, pos, table, out=out), list(out)),
                          (lambda: decode_attention_quant(half.clone(), *c, table, ctx, out=half), [half])):
        losses = [(t * w).sum() for t in changed]
        codes = [t._version for t in c[:2]]
        call()
        for loss in losses:
            with pytest.raises(RuntimeError, match="inplace operation"):
                loss.backward()
        if changed[0] is c.ks:
            assert all(t._version > v for t, v in zip(c[:2], codes))
    with torch.inference_mode():
        z = torch.ones(2, 4, 64, device=device)
    with torch.inference_mode():
        rotary(z, pos, rt, out=z)
