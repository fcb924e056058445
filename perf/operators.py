"""Workloads of the 8-bit rollout path: rotary positions, the quantised paged KV cache (written, read back) and the
attention of one new token over it.

Each case names one operator, its sizes and its types.  ``run`` computes it in plain torch operations (32-bit
arithmetic, one rounding at the end) or, with ``own``, through the package's entry points; ``exact`` computes it in
64 bits, written apart from the plain form.

Cache layout: codes float8 e4m3 [num_blocks, Hk, block_size, D] and one fp32 scale for each (block, KV head, slot);
a value is code * scale with scale = max(amax, 2^-90) / 448 over the row's D values.
"""
import math

import torch

own = False

F8 = torch.float8_e4m3fn
F8_MAX = 448.0
AMAX_MIN = 2.0 ** -90
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step of 64 sequences, 12 query and 2 key heads: latency
        dict(name="rotary_decode", op="rotary", T=64, H=14, D=128, rot=128, interleaved=False, dtype="bf16",
             scaled=True, grad=False, max_pos=4096),
        # forward and backward of a training micro-batch (8 x 768 rows), half of each head rotated in pairs
        dict(name="rotary_micro_batch", op="rotary", T=6144, H=14, D=128, rot=64, interleaved=True, dtype="bf16",
             scaled=False, grad=True, max_pos=4096),
        # forward and backward of long sequences, 32 query and 8 key heads, an odd number of rows, scaled angles
        dict(name="rotary_long_train", op="rotary", T=16383, H=40, D=128, rot=128, interleaved=False, dtype="bf16",
             scaled=True, grad=True, max_pos=16384),
        # a decode step of 512 sequences: rotates q and k, quantises k and v into the pages
        dict(name="kv_write_decode", op="kv_write", seqs=512, max_len=1, ragged=False, at=700, Hq=12, Hk=2, D=128,
             bs=16, rot=128, interleaved=False, dtype="bf16"),
        # the prompts of one rollout (64 x 256 tokens, rows of the fused projection)
        dict(name="kv_write_prompts", op="kv_write", seqs=64, max_len=256, ragged=False, at=0, Hq=12, Hk=2, D=128,
             bs=16, rot=0, interleaved=False, dtype="bf16"),
        # ragged prompts padded to 1536 tokens, 8 KV heads; the padding is not written
        dict(name="kv_write_ragged", op="kv_write", seqs=32, max_len=1536, ragged=True, at=0, Hq=32, Hk=8, D=128,
             bs=16, rot=0, interleaved=False, dtype="bf16"),
        # a short shared prefix read back before its prompt is continued
        dict(name="kv_read_prefix", op="kv_read", seqs=5, max_len=77, ragged=False, Hk=2, D=128, bs=16, dtype="bf16"),
        # long ragged prefixes read back, 8 KV heads
        dict(name="kv_read_long", op="kv_read", seqs=4, max_len=32768, ragged=True, Hk=8, D=128, bs=16, dtype="bf16"),
        # one sequence at the start of its answer: latency
        dict(name="attn_one_short", op="attn", B=1, Hq=12, Hk=2, D=128, bs=16, max_len=33, ragged=False,
             dtype="bf16"),
        # a decode step of a whole rollout batch, contexts up to 768 tokens
        dict(name="attn_rollout", op="attn", B=512, Hq=12, Hk=2, D=128, bs=16, max_len=768, ragged=True,
             dtype="bf16"),
        # few sequences of very different lengths, some of them empty
        dict(name="attn_ragged", op="attn", B=37, Hq=32, Hk=8, D=128, bs=16, max_len=1536, ragged=True,
             dtype="bf16"),
        # two long contexts: the split over the cache's length has to fill the machine
        dict(name="attn_long", op="attn", B=2, Hq=32, Hk=8, D=128, bs=64, max_len=131072, ragged=False,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "kv_write", "kv_write", "kv_read", "attn", "attn", "attn"])
    if op == "rotary":
        D = rng.choice([64, 80, 96, 128, 256])
        H = rng.choice([1, 3, 8, 14, 16, 40])
        rot = rng.choice([D, D, D // 2, D // 4])
        T = _log(rng, 1, min(32768, 16383 * 40 * 128 // (H * D) // 2))
        return dict(op=op, T=T, H=H, D=D, rot=rot, interleaved=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), scaled=rng.random() < 0.5,
                    grad=rng.random() < 0.6, max_pos=_log(rng, 64, 16384))
    D = rng.choice([64, 128, 128, 256])
    bs = rng.choice([8, 16, 16, 32, 64])
    Hk = rng.choice([1, 2, 4, 8])
    if op == "attn":
        Hq = Hk * rng.choice([1, 2, 4, 6, 8, 16])
        B = _log(rng, 1, 512)
        most = 2 * 131072 * 8 * 128 // (B * Hk * D) // max(1, Hq // (4 * Hk))
        return dict(op=op, B=B, Hq=Hq, Hk=Hk, D=D, bs=bs, max_len=_log(rng, 1, max(2, min(131072, most))),
                    ragged=rng.random() < 0.6, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    seqs = _log(rng, 1, 512)
    if op == "kv_read":
        most = 32768 * 2 * 8 * 128 // (seqs * Hk * D) // 2
        return dict(op=op, seqs=seqs, max_len=_log(rng, 1, max(2, min(32768, most))), ragged=rng.random() < 0.6,
                    Hk=Hk, D=D, bs=bs, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    Hq = Hk * rng.choice([1, 4, 6])
    rot = rng.choice([0, D, D // 2])
    most = 32 * 768 * 8 * 128 // (seqs * Hk * D) // (4 if rot else 1)
    return dict(op=op, seqs=seqs, max_len=_log(rng, 1, max(2, min(4096, most))), ragged=rng.random() < 0.6,
                at=_log(rng, 1, max(2, min(2048, (1 << 26) // (seqs * Hk * D)))), Hq=Hq, Hk=Hk, D=D, bs=bs, rot=rot, interleaved=rng.random() < 0.5,
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


# ------------------------------------------------------------------ inputs
def _lengths(n, most, ragged):
    """The multiset of lengths: all `most`, or spread over [0, most] (about one in nine empty where there are many)."""
    if not ragged:
        return [most] * n
    out = [1 + int((most - 1) * ((i + 1) * 0.6180339887498949 % 1.0)) for i in range(n)]
    for i in range(4, n, 9):
        out[i] = 0
    out[0] = most
    return out


def _shuffled(case, n, seed):
    L = torch.tensor(_lengths(n, case["max_len"], case["ragged"]), dtype=torch.int64)
    return L[torch.randperm(n, generator=torch.Generator().manual_seed(seed))]


def _table(rot, max_pos, scaled):
    """fp32 [max_pos, rot / 2, 2] of (cos, sin); `scaled`: low frequencies stretched 8-fold for long contexts."""
    inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    if scaled:
        turns = 8192.0 * inv / (2 * math.pi)
        mix = ((turns - 1.0) / 3.0).clamp(0, 1)
        inv = inv * (mix + (1 - mix) / 8.0)
    ang = torch.arange(max_pos, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()


def _pages(lens, at, bs, gen):
    """A block table over a shuffled pool, and the pool's size."""
    per = max(1, -(-int(lens.max().item() + at) // bs))
    n = lens.numel()
    perm = torch.randperm(n * per + 3, generator=gen, device="cuda")[: n * per]
    return perm.view(n, per).to(torch.int32).contiguous(), n * per + 3


def _normal(shape, gen, dtype):
    """Activations: normal, a few channels some times larger."""
    x = torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32 if dtype == torch.float32 else dtype)
    loud = torch.rand(shape[-1], device="cuda", generator=gen) < 0.03
    return x * torch.where(loud, 6.0, 1.0).to(x.dtype)


def _filled(rows, D, gen):
    """Codes and scales of `rows` quantised rows, a slab at a time."""
    codes = torch.empty(rows, D, device="cuda", dtype=F8)
    scale = torch.empty(rows, device="cuda")
    for lo in range(0, rows, 1 << 20):
        x = _normal((min(1 << 20, rows - lo), D), gen, torch.bfloat16).float()
        a = x.abs().amax(-1).clamp_min(AMAX_MIN)
        codes[lo:lo + x.shape[0]] = (x * (F8_MAX / a)[:, None]).to(F8)
        scale[lo:lo + x.shape[0]] = a / F8_MAX
    return codes, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    op, dt, D = case["op"], TYPES[case["dtype"]], case["D"]
    s = dict(case)
    if op == "rotary":
        s["x"] = _normal((case["T"], case["H"], D), gen, dt).requires_grad_(case["grad"])
        s["pos"] = torch.randint(0, case["max_pos"], (case["T"],), generator=gen, device="cuda", dtype=torch.int32)
        s["table"] = _table(case["rot"], case["max_pos"], case["scaled"])
        if case["grad"]:
            s["dy"] = torch.randn((case["T"], case["H"], D), device="cuda", generator=gen, dtype=dt)
        return s
    Hk, bs = case["Hk"], case["bs"]
    if op == "attn":
        B = case["B"]
        lens = _shuffled(case, B, seed)
        s["block_table"], n = _pages(lens, 0, bs, gen)
        s["ctx_len"] = lens.to(torch.int32).cuda()
        s["q"] = _normal((B, case["Hq"], D), gen, dt)
    else:
        at = case.get("at", 0)
        lens = _shuffled(case, case["seqs"], seed)
        s["block_table"], n = _pages(lens, at, bs, gen)
        # every sequence's rows are padded to max_len; padding has position -1
        p = torch.arange(case["max_len"])[None, :] + at
        p = torch.where(p < lens[:, None] + at, p, -1)
        s["pos"] = p.reshape(-1).to(torch.int32).cuda()
        s["seq_of_token"] = torch.arange(case["seqs"]).repeat_interleave(case["max_len"]).to(torch.int32).cuda()
        T = s["pos"].numel()
    if op == "kv_write":
        Hq = case["Hq"]
        qkv = _normal((T, (Hq + 2 * Hk), D), gen, dt)
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:]
        for c in ("kc", "vc"):
            s[c] = torch.zeros(n, Hk, bs, D, device="cuda", dtype=torch.uint8).view(F8)
        for c in ("ks", "vs"):
            s[c] = torch.zeros(n, Hk, bs, device="cuda")
        s["table"] = _table(case["rot"], case["max_len"] + at, False) if case["rot"] else None
        return s
    for c, z in (("kc", "ks"), ("vc", "vs")):
        codes, scale = _filled(n * Hk * bs, D, gen)
        s[c], s[z] = codes.view(n, Hk, bs, D), scale.view(n, Hk, bs)
    if op == "kv_read":
        s["out"] = tuple(torch.zeros(T, Hk, D, device="cuda", dtype=dt) for _ in range(2))
    return s


# ------------------------------------------------------------------ plain forms
def _rotate(x, pos, table, interleaved):
    """fp32 rotation of x [T, H, D] by the table's rows."""
    x = x.float()
    rot = 2 * table.shape[1]
    cs = table[pos.long()][:, None]
    c, s = cs[..., 0], cs[..., 1]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, x[..., rot:]], -1) if rot < x.shape[-1] else y


def _plain_rotary(s):
    y = _rotate(s["x"], s["pos"], s["table"], s["interleaved"]).to(s["x"].dtype)
    if not s["grad"]:
        return {"y": y}
    dx, = torch.autograd.grad(y, s["x"], s["dy"])
    return {"y": y.detach(), "dx": dx}


def _rows(s):
    """Tokens that count, and their cache rows [tokens, Hk]."""
    keep = torch.nonzero(s["pos"] >= 0).squeeze(1)
    p, bs, Hk = s["pos"][keep].long(), s["bs"], s["Hk"]
    blk = s["block_table"][s["seq_of_token"][keep].long(), p // bs].long()
    return keep, (blk[:, None] * Hk + torch.arange(Hk, device="cuda")) * bs + (p % bs)[:, None]


def _plain_write(s):
    k, v, D = s["k"], s["v"], s["D"]
    out = {}
    if s["table"] is not None:
        p = s["pos"].clamp_min(0)
        out["q"] = torch.where((s["pos"] >= 0)[:, None, None], _rotate(s["q"], p, s["table"], s["interleaved"]),
                               s["q"].float()).to(s["q"].dtype)
        k = _rotate(k, p, s["table"], s["interleaved"])
    keep, rows = _rows(s)
    for x, c, z in ((k, "kc", "ks"), (v, "vc", "vs")):
        x = x[keep].float()
        a = x.abs().amax(-1).clamp_min(AMAX_MIN)
        s[c].view(torch.uint8).view(-1, D)[rows] = (x * (F8_MAX / a)[..., None]).to(F8).view(torch.uint8)
        s[z].view(-1)[rows] = a / F8_MAX
        out[c], out[z] = s[c], s[z]
    return out


def _plain_read(s):
    keep, rows = _rows(s)
    for c, z, o in (("kc", "ks", 0), ("vc", "vs", 1)):
        x = s[c].view(torch.uint8).view(-1, s["D"])[rows].view(F8).float() * s[z].view(-1)[rows][..., None]
        s["out"][o][keep] = x.to(s["out"][o].dtype)
    return s["out"]


def _plain_attn(s):
    q, Hk, D, bs = s["q"], s["Hk"], s["D"], s["bs"]
    B, Hq = q.shape[:2]
    idx = torch.arange(s["max_len"], device="cuda")
    blk, slot = s["block_table"][:, idx // bs].long(), idx % bs
    rows = (blk[:, None, :] * Hk + torch.arange(Hk, device="cuda")[None, :, None]) * bs + slot  # [B, Hk, L]
    k, v = (s[c].view(torch.uint8).view(-1, D)[rows].view(F8).float() * s[z].view(-1)[rows][..., None]
            for c, z in (("kc", "ks"), ("vc", "vs")))
    w = q.float().view(B, Hk, Hq // Hk, D) @ k.transpose(2, 3) / math.sqrt(D)
    w = w.masked_fill((idx >= s["ctx_len"][:, None])[:, None, None], float("-inf"))
    top = w.amax(-1, keepdim=True).clamp_min(-1e30)
    w = torch.exp(w - top)
    o = (w @ v) / w.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.view(B, Hq, D).to(q.dtype)


def run(state):
    s = state
    if not own:
        return {"rotary": _plain_rotary, "kv_write": _plain_write, "kv_read": _plain_read,
                "attn": _plain_attn}[s["op"]](s)
    if s["op"] == "rotary":
        from turbol_b200.ops.rotary import rotary

        y = rotary(s["x"], s["pos"], s["table"], interleaved=s["interleaved"])
        if not s["grad"]:
            return {"y": y}
        dx, = torch.autograd.grad(y, s["x"], s["dy"])
        return {"y": y.detach(), "dx": dx}
    from turbol_b200.ops.kv_cache import decode_attention_quant, kv_quant_read, kv_quant_write

    if s["op"] == "kv_write":
        out = {"kc": s["kc"], "ks": s["ks"], "vc": s["vc"], "vs": s["vs"]}
        if s["table"] is None:
            kv_quant_write(s["k"], s["v"], s["seq_of_token"], s["pos"], s["block_table"], s["kc"], s["vc"], s["ks"],
                           s["vs"])
        else:
            out["q"] = kv_quant_write(s["k"], s["v"], s["seq_of_token"], s["pos"], s["block_table"], s["kc"], s["vc"],
                                      s["ks"], s["vs"], q=s["q"], table=s["table"], interleaved=s["interleaved"])
        return out
    if s["op"] == "kv_read":
        return kv_quant_read(s["kc"], s["vc"], s["ks"], s["vs"], s["seq_of_token"], s["pos"], s["block_table"],
                             out=s["out"])
    return decode_attention_quant(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["block_table"], s["ctx_len"])


# ------------------------------------------------------------------ work
def work(case):
    op, D, e = case["op"], case["D"], BYTES[case["dtype"]]
    if op == "rotary":
        n = case["T"] * case["H"]
        passes = 2 if case["grad"] else 1
        rows = min(case["T"], case["max_pos"])
        return {"bytes": passes * 2 * n * D * e + 4 * case["T"] + rows * case["rot"] * 4,
                "flops": passes * 3 * n * case["rot"]}
    Hk = case["Hk"]
    if op == "attn":
        ctx = sum(_lengths(case["B"], case["max_len"], case["ragged"]))
        return {"bytes": ctx * Hk * 2 * (D + 4) + 2 * case["B"] * case["Hq"] * D * e + -(-ctx // case["bs"]) * 4,
                "flops": 4 * ctx * case["Hq"] * D}
    T = sum(_lengths(case["seqs"], case["max_len"], case["ragged"]))
    cells = case["seqs"] * case["max_len"]
    b = T * Hk * 2 * (D * e + D + 4) + cells * 8
    if op == "kv_write" and case["rot"]:
        b += 2 * cells * case["Hq"] * D * e + min(T, case["max_len"]) * case["rot"] * 4
    return {"bytes": b, "flops": T * Hk * 4 * D}


# ------------------------------------------------------------------ 64 bits
def _turn(x, pos, table, interleaved, back=False):
    """The rotation as complex products in 64 bits."""
    rot = 2 * table.shape[1]
    f = torch.view_as_complex(table.double()[pos.long()].contiguous())[:, None]
    x = x.double()
    z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else \
        torch.complex(x[..., :rot // 2], x[..., rot // 2:rot])
    z = z * (f.conj() if back else f)
    out = x.clone()
    if interleaved:
        out[..., 0:rot:2], out[..., 1:rot:2] = z.real, z.imag
    else:
        out[..., :rot // 2], out[..., rot // 2:rot] = z.real, z.imag
    return out


def _e4m3(y):
    """Nearest e4m3 value (ties to even) of 64-bit numbers within +-448."""
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -30))).clamp_min(-6)
    step = torch.exp2(e - 3)
    return (torch.round(y / step) * step).clamp(-F8_MAX, F8_MAX)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        out = {"y": _turn(s["x"], s["pos"], s["table"], s["interleaved"])}
        if case["grad"]:
            out["dx"] = _turn(s["dy"], s["pos"], s["table"], s["interleaved"], back=True)
        return out
    Hk, D, bs = case["Hk"], case["D"], case["bs"]
    if op == "attn":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["ctx_len"].tolist()):
            if not n:
                continue
            blocks = s["block_table"][b, : -(-n // bs)].long()
            for h in range(Hk):
                k, v = ((s[c].view(torch.uint8)[blocks, h].view(F8).double() * s[z][blocks, h].double()[..., None])
                        .view(-1, D)[:n] for c, z in (("kc", "ks"), ("vc", "vs")))
                G = case["Hq"] // Hk
                w = torch.softmax(s["q"][b, h * G:(h + 1) * G].double() @ k.t() * D ** -0.5, -1)
                out[b, h * G:(h + 1) * G] = w @ v
        return out
    p = s["pos"].long()
    blk = s["block_table"].long()[s["seq_of_token"].long(), p.clamp_min(0) // bs]
    live = p >= 0
    if op == "kv_read":
        out = []
        for c, z in (("kc", "ks"), ("vc", "vs")):
            x = s[c].view(torch.uint8)[blk, :, p % bs].view(F8).double() * s[z][blk, :, p % bs].double()[..., None]
            out.append(x * live[:, None, None])
        return tuple(out)
    out = {}
    k = s["k"].double()
    if s["table"] is not None:
        k = _turn(s["k"], p.clamp_min(0), s["table"], s["interleaved"])
        out["q"] = torch.where(live[:, None, None], _turn(s["q"], p.clamp_min(0), s["table"], s["interleaved"]),
                               s["q"].double())
    for x, c, z in ((k, "kc", "ks"), (s["v"].double(), "vc", "vs")):
        a = x.abs().amax(-1).clamp_min(AMAX_MIN)
        codes = torch.zeros(s[c].shape, dtype=torch.float64, device="cuda")
        scale = torch.zeros(s[z].shape, dtype=torch.float64, device="cuda")
        codes[blk[live], :, (p % bs)[live]] = _e4m3(x * (F8_MAX / a)[..., None])[live]
        scale[blk[live], :, (p % bs)[live]] = (a / F8_MAX)[live]
        out[c], out[z] = codes, scale
    return out
