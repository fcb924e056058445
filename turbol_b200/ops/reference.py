"""Plain PyTorch (fp32, CPU-friendly) restatements of every kernel's math.

These are the oracles the kernel tests compare against and the code path CPU
tensors take.  They are written for clarity, not speed.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def philox4x32_10(seed: int, c0: int, c1: int, c2: int, c3: int = 0):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC'11): the four output words
    for key ``seed`` (64-bit) and counter (c0, c1, c2, c3), as the device and
    host generators compute them."""
    m0, m1, w0, w1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
    mask = 0xFFFFFFFF
    c = [c0 & mask, c1 & mask, c2 & mask, c3 & mask]
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(10):
        p0, p1 = m0 * c[0], m1 * c[2]
        c = [((p1 >> 32) ^ c[1] ^ k0) & mask, p1 & mask, ((p0 >> 32) ^ c[3] ^ k1) & mask, p0 & mask]
        k0, k1 = (k0 + w0) & mask, (k1 + w1) & mask
    return c


def gae(rewards, values, dones, gamma: float = 0.99, lam: float = 0.95):
    """GAE over [T, N] (values [T+1, N]); recurrence of the reference's
    turbol_vllm/src/cuda/gae.cu:31-44."""
    T = rewards.shape[0]
    dt = torch.promote_types(rewards.dtype, torch.float32)
    adv = torch.zeros_like(rewards, dtype=dt)
    last = torch.zeros_like(rewards[0], dtype=dt)
    for t in range(T - 1, -1, -1):
        nd = 1.0 - dones[t].float()
        delta = rewards[t] + gamma * nd * values[t + 1] - values[t]
        last = delta + gamma * lam * nd * last
        adv[t] = last
    return adv, adv + values[:T]


def grpo_advantage(rewards, group_size: int, eps: float = 1e-4, scale_by_std: bool = True):
    r = rewards.float().view(-1, group_size)
    mean = r.mean(1, keepdim=True)
    std = r.std(1, keepdim=True, unbiased=True) if group_size > 1 else torch.zeros_like(mean)
    a = r - mean
    if scale_by_std:
        a = a / (std + eps)
    return a.reshape(-1)


def ppo_categorical_loss(logits, value, act, old_logp, adv, ret, clip=0.2, vf_coef=0.5, ent_coef=0.0,
                         old_value=None, vclip=0.0):
    """Returns (loss, stats) for the clipped-surrogate PPO objective."""
    logp_all = F.log_softmax(logits.float(), -1)
    logp = logp_all.gather(1, act.long().view(-1, 1)).squeeze(1)
    ratio = torch.exp(logp - old_logp)
    pg = -torch.min(ratio * adv, ratio.clamp(1 - clip, 1 + clip) * adv)
    if vclip > 0 and old_value is not None:
        vc = old_value + (value - old_value).clamp(-vclip, vclip)
        vl = 0.5 * torch.max((value - ret) ** 2, (vc - ret) ** 2)
    else:
        vl = 0.5 * (value - ret) ** 2
    ent = -(logp_all.exp() * logp_all).sum(-1)
    loss = pg.mean() + vf_coef * vl.mean() - ent_coef * ent.mean()
    with torch.no_grad():
        stats = torch.stack([pg.sum(), vl.sum(), ent.sum(), ((ratio - 1) - (logp - old_logp)).sum(),
                             ((ratio - 1).abs() > clip).float().sum(), torch.tensor(float(len(act)))])
    return loss, stats


def adam_step(p, g, m, v, step, lr=3e-4, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, grad_scale=1.0):
    g = g * grad_scale
    m.mul_(b1).add_(g, alpha=1 - b1)
    v.mul_(b2).addcmul_(g, g, value=1 - b2)
    bc1, bc2 = 1 - b1 ** step, 1 - b2 ** step
    p.sub_(lr * ((m / bc1) / ((v / bc2).sqrt() + eps) + wd * p))
    return p


def fnv1a_reward(ids, lengths=None):
    out = []
    ids = ids.to(torch.int64).cpu()
    for i in range(ids.shape[0]):
        L = int(lengths[i]) if lengths is not None else ids.shape[1]
        h = 0xcbf29ce484222325
        for t in range(min(L, ids.shape[1])):
            w = int(ids[i, t]) & 0xFFFFFFFF
            for _ in range(4):
                h ^= w & 0xFF
                h = (h * 0x100000001b3) & 0xFFFFFFFFFFFFFFFF
                w >>= 8
        out.append((h % 1000) / 1000.0)
    return torch.tensor(out, dtype=torch.float32)


def cartpole_step(state, action, gravity=9.8, masscart=1.0, masspole=0.1, length=0.5, force_mag=10.0, tau=0.02,
                  x_threshold=2.4, theta_threshold=12 * 2 * math.pi / 360):
    """One Euler step of the cart-pole equations; returns (next_state, terminated)."""
    x, x_dot, th, th_dot = state.unbind(-1)
    total = masscart + masspole
    pml = masspole * length
    force = torch.where(action == 1, torch.full_like(x, force_mag), torch.full_like(x, -force_mag))
    c, s = torch.cos(th), torch.sin(th)
    temp = (force + pml * th_dot ** 2 * s) / total
    th_acc = (gravity * s - c * temp) / (length * (4.0 / 3.0 - masspole * c ** 2 / total))
    x_acc = temp - pml * th_acc * c / total
    nx = torch.stack([x + tau * x_dot, x_dot + tau * x_acc, th + tau * th_dot, th_dot + tau * th_acc], -1)
    term = (nx[..., 0].abs() > x_threshold) | (nx[..., 2].abs() > theta_threshold)
    return nx, term


def rmsnorm(x, w, eps=1e-6):
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float())


def rope(x, pos, theta=1e4):
    """Rotate-half RoPE on the last dim of x [..., S, H, D] with positions [S]."""
    D = x.shape[-1]
    inv = 1.0 / (theta ** (torch.arange(0, D, 2, dtype=torch.float64, device=x.device) / D))
    ang = pos.to(torch.float64)[:, None] * inv[None, :]
    cos = torch.cos(ang).float()[:, None, :]
    sin = torch.sin(ang).float()[:, None, :]
    x1, x2 = x.float()[..., : D // 2], x.float()[..., D // 2:]
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)


def causal_attention(q, k, v, scale=None):
    """q [B, S, Hq, D], k/v [B, S, Hk, D] (GQA) -> [B, S, Hq, D] fp32."""
    B, S, Hq, D = q.shape
    Hk = k.shape[2]
    rep = Hq // Hk
    qf, kf, vf = q.float(), k.float().repeat_interleave(rep, 2), v.float().repeat_interleave(rep, 2)
    s = torch.einsum("bqhd,bkhd->bhqk", qf, kf) * (scale or 1.0 / math.sqrt(D))
    mask = torch.ones(S, S, dtype=torch.bool, device=q.device).tril()
    s = s.masked_fill(~mask, float("-inf"))
    p = s.softmax(-1)
    return torch.einsum("bhqk,bkhd->bqhd", p, vf)


def lm_forward_ref(model, ids, params=None):
    """fp32 forward of a DecoderLM (all layers, embed and head) from its bf16
    weights; returns logits [B, T, V].  ``params`` (name -> tensor) overrides the
    weights, e.g. with leaf tensors for autograd."""
    cfg = model.cfg
    P = params if params is not None else {n: model.s[n].float() for n in model.offsets}
    if params is None and model.flat is not None:
        for n in P:
            if n.endswith(("ln1", "ln2", "norm", "bqkv")):
                P[n] = model.p[n].float()
    B, T = ids.shape
    H, D, F = cfg.hidden, cfg.head_dim, cfg.ffn
    x = P["embed"][ids.long()] * cfg.embed_scale
    pos = torch.arange(T, device=ids.device)
    for i in model.layers:
        p = f"l{i}."
        h = rmsnorm(x, P[p + "ln1"], cfg.rms_eps)
        qkv = h @ P[p + "wqkv"].t()
        if cfg.qkv_bias:
            qkv = qkv + P[p + "bqkv"]
        q = qkv[..., : cfg.q_dim].view(B, T, cfg.n_heads, D)
        k = qkv[..., cfg.q_dim:cfg.q_dim + cfg.kv_dim].view(B, T, cfg.n_kv_heads, D)
        v = qkv[..., cfg.q_dim + cfg.kv_dim:].view(B, T, cfg.n_kv_heads, D)
        if cfg.rope_default:
            q, k = rope(q, pos, cfg.rope_theta), rope(k, pos, cfg.rope_theta)
        else:
            flat_pos = pos.repeat(B)
            q, k = (rotary(x.reshape(B * T, -1, D), flat_pos, model.table, cfg.rope_interleaved).view(x.shape)
                    for x in (q, k))
        a = causal_attention(q, k, v).reshape(B, T, cfg.q_dim)
        x = x + a @ P[p + "wo"].t()
        h = rmsnorm(x, P[p + "ln2"], cfg.rms_eps)
        gu = h @ P[p + "wgu"].t()
        act = torch.nn.functional.silu(gu[..., 0::2]) * gu[..., 1::2]
        x = x + act @ P[p + "wdown"].t()
    h = rmsnorm(x, P["norm"], cfg.rms_eps)
    W = P["embed"] if cfg.tie_embeddings else P["lm_head"]
    return h @ W.t()


def ppo_token_loss(lp, old_lp, adv, v, old_v, ret, clip=0.2, vclip=0.2, vf_coef=0.1, norm=1.0):
    """Clipped PPO policy loss + clipped value loss per token (the oracle of
    the ``ppo_token_loss`` kernel).  Returns (loss, d loss / d lp,
    d loss / d v, stats [pg * norm, vf * norm, clipped tokens, tokens])."""
    lp_t = lp.detach().float().clone().requires_grad_()
    v_t = v.detach().float().clone().requires_grad_()
    with torch.enable_grad():
        ratio = torch.exp(lp_t - old_lp.float())
        pg = -torch.min(ratio * adv, torch.clamp(ratio, 1 - clip, 1 + clip) * adv)
        v_clip = old_v + torch.clamp(v_t - old_v, -vclip, vclip)
        vf = 0.5 * torch.max((v_t - ret) ** 2, (v_clip - ret) ** 2)
        loss = (pg.sum() + vf_coef * vf.sum()) * norm
        loss.backward()
    stats = torch.stack([pg.detach().sum() * norm, vf.detach().sum() * norm,
                         ((ratio.detach() - 1).abs() > clip).float().sum(),
                         torch.tensor(float(lp.numel()), device=lp.device)])
    return loss.detach(), lp_t.grad, v_t.grad, stats


def rotary(x, pos, table, interleaved=False, transpose=False, out=None, error=None):
    """Rotary positions of x [T, H, D], general form (the math of the ``rotary``
    kernel, computed in table's type)."""
    R = 2 * table.shape[1]
    p = pos.long()
    bad, pad = p >= table.shape[0], p < 0
    cs = table[p.clamp(0, table.shape[0] - 1)][:, None]
    c, s = cs[..., 0], -cs[..., 1] if transpose else cs[..., 1]
    xf = x.to(table.dtype)
    a, b = (xf[..., 0:R:2], xf[..., 1:R:2]) if interleaved else (xf[..., : R // 2], xf[..., R // 2: R])
    ya, yb = a * c - b * s, b * c + a * s
    y = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    y = torch.cat([y, xf[..., R:]], -1)
    y = torch.where(pad[:, None, None], xf, y).masked_fill(bad[:, None, None], float("nan")).to(x.dtype)
    if error is not None and bool(bad.any()):
        error[0] = 1
    if out is None:
        return y
    out.copy_(y)
    return out


KV_AMAX_MIN = 2.0 ** -90  # keeps 448 / amax finite for rows of zeros


def kv_quantise(x):
    """(e4m3 codes, fp32 scales) of the rows x [..., D]."""
    xf = x.float()
    amax = xf.abs().amax(-1).clamp_min(KV_AMAX_MIN)
    top = torch.full_like(amax, 448.0)  # tensor / tensor: IEEE division (a scalar operand becomes a reciprocal product)
    return (xf * (top / amax)[..., None]).to(torch.float8_e4m3fn), amax / top


def _slots(seq_of_token, pos, block_table, num_blocks, bs, error):
    """(tokens that name a slot, their blocks, their places in the block)."""
    live = (seq_of_token >= 0) & (pos >= 0)
    ok = live & (seq_of_token < block_table.shape[0]) & (pos // bs < block_table.shape[1])
    t = torch.nonzero(ok).squeeze(1)
    blk = block_table[seq_of_token[t].long(), (pos[t] // bs).long()].long()
    fine = (blk >= 0) & (blk < num_blocks)
    if error is not None and (int(live.sum()) != int(ok.sum()) or not bool(fine.all())):
        error[0] = 1
    t, blk = t[fine], blk[fine]
    return t, blk, (pos[t] % bs).long()


def kv_quant_write(k, v, seq_of_token, pos, block_table, kc, vc, ks, vs, q=None, table=None, interleaved=False,
                   q_out=None, error=None):
    p = pos = torch.where(seq_of_token < 0, -1, pos)  # a negative sequence is padding, whatever its position
    if table is not None:
        if q is not None:
            rotary(q, pos, table, interleaved, out=q_out, error=error)
        k = rotary(k.float(), pos, table, interleaved, error=error)
        p = torch.where(pos < table.shape[0], pos, -1)
    t, blk, slot = _slots(seq_of_token, p, block_table, kc.shape[0], kc.shape[2], error)
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        codes, scale = kv_quantise(x[t])
        c.view(torch.uint8)[blk, :, slot] = codes.view(torch.uint8)
        s[blk, :, slot] = scale


def kv_quant_read(kc, vc, ks, vs, seq_of_token, pos, block_table, out, error=None):
    t, blk, slot = _slots(seq_of_token, pos, block_table, kc.shape[0], kc.shape[2], error)
    for c, s, o in ((kc, ks, out[0]), (vc, vs, out[1])):
        codes = c.view(torch.uint8)[blk, :, slot].view(torch.float8_e4m3fn)
        o[t] = (codes.float() * s[blk, :, slot][..., None]).to(o.dtype)
    return out


def decode_attention_quant(q, kc, vc, ks, vs, block_table, ctx_len, scale, out=None, error=None, dtype=torch.float32):
    """One-token attention over the 8-bit paged cache, sequence by sequence, in
    ``dtype``; out (if given) receives it rounded."""
    B, Hq, D = q.shape
    num_blocks, Hk, bs, _ = kc.shape
    y = torch.zeros(B, Hq, D, dtype=dtype, device=q.device)
    for b, n in enumerate(ctx_len.tolist()):
        # (one token behind the table is enough to tell of all)
        idx = torch.arange(min(max(n, 0), block_table.shape[1] * bs + 1), device=q.device)
        t, blk, slot = _slots(torch.full_like(idx, b), idx, block_table, num_blocks, bs, error)
        if t.numel() == 0:
            continue
        k, v = ((c.view(torch.uint8)[blk, :, slot].view(torch.float8_e4m3fn).to(dtype) *
                 s[blk, :, slot].to(dtype)[..., None]).transpose(0, 1) for c, s in ((kc, ks), (vc, vs)))
        w = torch.softmax(q[b].to(dtype).view(Hk, Hq // Hk, D) @ k.transpose(1, 2) * scale, -1)
        y[b] = (w @ v).reshape(Hq, D)
    if out is None:
        return y
    out.copy_(y)
    return out


# ------------------------------------------------------------------ distillation
def topk_logprobs(logits, k, temperature=1.0, dtype=torch.float32):
    """(log-probabilities, ids int32, log-sum-exps) of each row's k largest logits; the numbers in ``dtype``."""
    z = logits.double()
    # NaN ranks as -inf, equal values (+-0 too) by the lowest id
    key = torch.where(z.isnan(), torch.full_like(z, -math.inf), z) + 0.0
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    lse = torch.logsumexp(z / temperature, 1)
    top = key.amax(1, keepdim=True)
    top = torch.where(top.isinf(), 0.0, top)  # (differences first: next to the type's lowest value lse loses log V)
    logp = (z.gather(1, ids) - top) / temperature - torch.logsumexp((z - top) / temperature, 1, keepdim=True)
    logp = torch.where(lse[:, None].isneginf(), lse[:, None], logp)
    logp = torch.where(lse[:, None].isnan(), lse[:, None], logp)
    return logp.to(dtype), ids.to(torch.int32), lse.to(dtype)


DISTILL_REST_MIN = 2.0 ** -20


def distill(logits, ids, logprobs, weight=None, kind="forward", rest=True, temperature=1.0, target=None,
            target_weight=None, error=None, dtype=None, out_kl=None):
    """(loss fp32 [R], gradient in ``dtype``, default logits') of the distillation loss, computed in 64 bits; the KLs
    alone into ``out_kl``."""
    R, V = logits.shape
    f64 = dict(dtype=torch.float64, device=logits.device)
    w = torch.ones(R, **f64) if weight is None else weight.double()
    c = torch.zeros(R, **f64) if target is None else torch.ones(R, **f64) if target_weight is None else \
        target_weight.double()
    y = torch.full((R,), -1, device=logits.device) if target is None else target.long()
    live = (w != 0) | ((c != 0) & (y >= 0))
    bad = ((ids >= V) & ~logprobs.isneginf() & (w != 0)[:, None]).any() | ((y >= V) & live).any()
    if error is not None and bool(bad):
        error[0] = 1
    c = torch.where((y >= 0) & (y < V), c, 0.0)
    live = (w != 0) | (c != 0)
    y = y.clamp(0, V - 1)[:, None]
    z = torch.where(live[:, None], logits.double(), 0.0)
    top = z.amax(1, keepdim=True)
    # (differences first: next to the type's lowest value the sum's logarithm would be lost)
    z = (z - torch.where(top.isfinite(), top, 0.0)) / temperature
    lse = torch.logsumexp(z, 1, keepdim=True)
    lse = torch.where(lse.isinf(), math.nan, lse)
    logp = z - lse
    p = logp.exp()
    here = (ids >= 0) & (ids < V) & ~logprobs.isneginf()
    at = torch.where(here, ids.long(), V)  # (what is left out: a column behind the last)
    l = torch.where(here, logprobs.double(), -math.inf)
    top = torch.full((R, V + 1), -math.inf, **f64).scatter_reduce_(1, at, l, "amax")
    lt = torch.zeros(R, V + 1, **f64).scatter_add_(1, at, torch.where(here, (l - top.gather(1, at)).exp(), 0.0))
    lt = (top + lt.log())[:, :V]  # the classes' log-masses: of faint ones nothing else is left
    t = torch.where(lt.isneginf(), 0.0, lt.exp())
    inside = torch.zeros(R, V + 1, dtype=torch.bool, device=logits.device).scatter_(1, at, True)[:, :V]
    total = torch.where(here, l.exp(), 0.0).sum(1, keepdim=True)

    def plogq(a, la, b, on):  # a (la - log b) where it counts
        return torch.where(on & (a > 0), a * (la - b), 0.0).sum(1, keepdim=True) + \
            torch.where(on & a.isnan(), a, 0.0).sum(1, keepdim=True)

    if not rest:
        some = here.any(1, keepdim=True)
        lt = lt - torch.where(some, torch.logsumexp(l, 1, keepdim=True), 0.0)
        t = torch.where(lt.isneginf(), 0.0, lt.exp())
        kl = plogq(t, lt, logp, inside)
        d = torch.where(some, p - t, 0.0)
    else:
        outside = torch.where(inside, -math.inf, logp)
        most = outside.amax(1, keepdim=True)
        empty = most.isneginf()
        q = (outside - torch.where(empty, 0.0, most)).exp()  # (differences first here, too)
        share = q.sum(1, keepdim=True)
        lr, q = most + share.log(), torch.where(empty, 0.0, q / share)
        pr = lr.exp()
        if kind == "forward":
            tr = (1 - total).clamp_min(0)
            kl = plogq(t, lt, logp, inside) + torch.where(empty | (tr == 0), 0.0, tr * (tr.clamp_min(1e-300).log() - lr))
            a = total + torch.where(empty, 0.0, tr)  # 1, but for a student without mass outside (or a list with more than 1)
            d = torch.where(inside, a * p - t, (a * pr - tr) * q)
        else:
            f = torch.where(inside & (p > 0), logp - lt, 0.0)
            fr = torch.where(empty, 0.0, lr - (1 - total).clamp_min(DISTILL_REST_MIN).log())
            kl = (p * f).sum(1, keepdim=True) + pr * fr
            d = torch.where(inside, p * (f - kl), pr * q * (fr - kl))
    kl, d = torch.where(lse.isnan(), math.nan, kl), torch.where(lse.isnan(), math.nan, d)  # (whatever the list is)
    on, c = (w != 0)[:, None], c[:, None]
    if out_kl is not None:
        out_kl.copy_(torch.where(on, kl, 0.0).squeeze(1))
    loss = torch.where(on, w[:, None] * kl, 0.0) + torch.where(c != 0, -c * logp.gather(1, y), 0.0)
    d = torch.where(on, w[:, None] * d, 0.0) + torch.where(c != 0, c * p, 0.0)
    d.scatter_add_(1, y, -c)
    return loss.squeeze(1).float(), (d / temperature).to(logits.dtype if dtype is None else dtype)


# ------------------------------------------------------------------ embedding
def embedding(ids, weight, scale=1.0, out=None, error=None, first_row=False):
    """scale * weight[ids], padding (negative ids) zero, ids past the table NaN (or both row 0)."""
    i = ids.long()
    bad = i >= weight.shape[0]
    if first_row:
        outside = bad | (i < 0)
        if error is not None and bool(outside.any()):
            error[0] = 1
        return embedding(i.masked_fill(outside, 0), weight, scale, out)
    if error is not None and bool(bad.any()):
        error[0] = 1
    y = weight[i.clamp(0, weight.shape[0] - 1)].double() * scale
    y = y.masked_fill((i < 0)[..., None], 0.0).masked_fill(bad[..., None], math.nan).to(weight.dtype)
    if out is None:
        return y
    out.copy_(y)
    return out


def embedding_grad(ids, dy, grad, scale=1.0, accumulate=True, error=None):
    """grad[v] (+)= scale * sum of dy over the tokens v, summed in fp32 in token order."""
    i = ids.reshape(-1).long()
    if error is not None and bool((i >= grad.shape[0]).any()):
        error[0] = 1
    t = torch.nonzero((i >= 0) & (i < grad.shape[0])).squeeze(1)
    rows, at = torch.unique(i[t], return_inverse=True)
    s = torch.zeros(rows.numel(), grad.shape[1], device=grad.device)
    s.index_add_(0, at, dy.reshape(i.numel(), grad.shape[1])[t].float())
    if not accumulate:
        grad.zero_()
    grad[rows] = (grad[rows].float() + s * scale).to(grad.dtype)
    return grad
