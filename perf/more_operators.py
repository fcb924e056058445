"""Workloads at both ends of a training step, where the whole vocabulary counts: a teacher's top log-probabilities,
the distillation loss on them with its gradient, and the embedding with its gradient summed by sorted tokens.

Each case names one operator, its sizes and its types.  ``run`` computes it in plain torch operations (32-bit
arithmetic, one rounding at the end) or, with ``own``, through the package's entry points; ``exact`` computes it in
64 bits, written apart from the plain form.

Distillation: p = softmax(z / T) of the student's row z; the teacher's list has ids a_k and log-probabilities l_k,
t_k = exp(l_k).  What is outside the list is one more class (``rest``) with t_R = 1 - sum t_k and the student's mass
p_R there, or the list is renormalised.  forward: sum t log(t / p), reverse: sum p log(p / t); a row counts `weight`
times that, plus `target_weight` times -log p of its label.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
REST_MIN = 2.0 ** -20  # below this fp32 log-probabilities cannot tell the mass outside the list from none


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one sampled token's alternatives: latency
        dict(name="topk_one_row", op="topk", R=1, V=151936, pad=0, k=20, temp=1.0, dtype="bf16"),
        # the alternatives of a decode step of 512 sequences
        dict(name="topk_decode", op="topk", R=512, V=151936, pad=0, k=20, temp=1.0, dtype="bf16"),
        # the teacher's list for a micro-batch (8 x 512 response tokens)
        dict(name="topk_teacher", op="topk", R=4096, V=151936, pad=0, k=64, temp=1.0, dtype="bf16"),
        # an odd vocabulary, rows of a padded head, fp32 logits, a long list
        dict(name="topk_odd", op="topk", R=333, V=50001, pad=7, k=100, temp=0.7, dtype="fp32"),
        # a tiny model's rows, loss and gradient through autograd: latency
        dict(name="distill_tiny", op="distill", R=64, V=1024, pad=0, K=16, temp=1.0, kind="forward", rest=True,
             label=False, fused=False, dtype="bf16"),
        # a micro-batch of the student, with the policy-gradient term on the sampled tokens, loss and gradient at once
        dict(name="distill_micro_batch", op="distill", R=4096, V=151936, pad=0, K=64, temp=1.0, kind="forward",
             rest=True, label=True, fused=True, dtype="bf16"),
        # the student's own samples (reverse), rows of padding among them, through autograd
        dict(name="distill_reverse", op="distill", R=2048, V=128256, pad=0, K=32, temp=1.0, kind="reverse", rest=True,
             label=False, fused=False, dtype="bf16"),
        # an odd vocabulary, softened, the list renormalised
        dict(name="distill_odd", op="distill", R=777, V=32003, pad=0, K=50, temp=2.0, kind="forward", rest=False,
             label=False, fused=True, dtype="fp16"),
        # a decode step's lookup: latency
        dict(name="embed_decode", op="embed", N=64, H=1536, V=151936, scale=1.0, hot=0.0, grad="none", dtype="bf16"),
        # a training micro-batch (8 x 768 tokens), the gradient added to what the tied head left
        dict(name="embed_micro_batch", op="embed", N=6144, H=1536, V=151936, scale=39.25, hot=0.0, grad="add",
             dtype="bf16"),
        # a long batch through autograd, the dense gradient of an 8B-shape embedding
        dict(name="embed_dense", op="embed", N=16384, H=4096, V=128256, scale=1.0, hot=0.0, grad="dense",
             dtype="bf16"),
        # a ragged batch whose filler token is a third of it, rows of an odd number of values
        dict(name="embed_filler", op="embed", N=65537, H=1025, V=32003, scale=0.5, hot=0.33, grad="add", dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["topk", "distill", "embed"])
    dt = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "embed":
        H = rng.choice([64, 100, 257, 1024, 1536, 2048, 4096])
        V = _log(rng, 16, 151936 * 1536 // max(H, 1536))
        grad = rng.choice(["none", "add", "add", "dense"])
        return dict(op=op, N=_log(rng, 1, min(131072, 65537 * 1025 // H)), H=H, V=V,
                    scale=rng.choice([1.0, 0.5, 39.25]), hot=rng.choice([0.0, 0.0, 0.33]), grad=grad, dtype=dt)
    V = _log(rng, 200, 200000)
    most = 4096 * 151936 // (2 if dt == "fp32" else 1)
    R = _log(rng, 1, max(2, min(8192, most // V)))
    pad = rng.choice([0, 0, 0, 8, 5])
    temp = rng.choice([1.0, 1.0, 0.7, 2.0])
    k = _log(rng, 1, 200)
    if op == "topk":
        return dict(op=op, R=R, V=V, pad=pad, k=k, temp=temp, dtype=dt)
    kind = rng.choice(["forward", "forward", "reverse"])
    return dict(op=op, R=max(1, R // 2), V=V, pad=pad, K=_log(rng, 4, 100), temp=temp, kind=kind,
                rest=kind == "reverse" or rng.random() < 0.6, label=rng.random() < 0.4, fused=rng.random() < 0.6,
                dtype=dt)


# ------------------------------------------------------------------ inputs
def _ids(case):
    """The multiset of token ids: frequencies fall like 1 / rank; a share of `hot` is one id (the filler token)."""
    N, V = case["N"], case["V"]
    u = (torch.arange(N, dtype=torch.float64) + 0.5) / N
    ids = (2.7 * (torch.exp(u * math.log((V + 2.7) / 2.7)) - 1)).long().clamp_max(V - 1)
    ids[: int(case["hot"] * N)] = V // 2
    return ids


def _weights(case):
    """1 for most rows, 0 for the fifth, tenth, ... (padding)."""
    return (torch.arange(case["R"]) % 5 != 4).float()


def _logits(R, V, pad, dtype, gen):
    """Rows of a head's output: from flat to peaked."""
    x = torch.randn(R, V + pad, device="cuda", generator=gen, dtype=torch.float32 if dtype == torch.float32 else dtype)
    return x.mul_((1 + 2 * torch.rand(R, 1, device="cuda", generator=gen)).to(x.dtype))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    dt, s = TYPES[case["dtype"]], dict(case)
    if case["op"] == "embed":
        N, H, V = case["N"], case["H"], case["V"]
        ids = _ids(case)[torch.randperm(N, generator=torch.Generator().manual_seed(seed))]
        s["ids"] = ids.to(torch.int32).cuda()
        s["weight"] = torch.randn(V, H, device="cuda", generator=gen, dtype=dt).mul_(0.02)
        if case["grad"] != "none":
            s["dy"] = torch.randn(N, H, device="cuda", generator=gen, dtype=dt).mul_(0.1)
        if case["grad"] == "add":
            s["sum"] = torch.randn(V, H, device="cuda", generator=gen).mul_(0.01)
        s["weight"].requires_grad_(case["grad"] == "dense")
        return s
    R, V = case["R"], case["V"]
    x = _logits(R, V, case["pad"], dt, gen)
    s["logits"] = x[:, :V]
    if case["op"] == "topk":
        return s
    # a teacher that agrees with the student on most tokens
    t = s["logits"].float()
    t = t.add(torch.randn(R, V, device="cuda", generator=gen, dtype=torch.bfloat16), alpha=1.5).div_(case["temp"])
    top, ids = torch.topk(t, case["K"], dim=1)
    s["list_logp"] = top - torch.logsumexp(t, 1, keepdim=True)
    s["list_ids"] = ids.to(torch.int32)
    s["row_weight"] = _weights(case).cuda()
    s["label_id"] = torch.randint(0, V, (R,), device="cuda", generator=gen, dtype=torch.int32)
    s["label_weight"] = torch.randn(R, device="cuda", generator=gen)
    if not case["fused"]:
        s["dloss"] = torch.rand(R, device="cuda", generator=gen) + 0.5
        s["logits"] = s["logits"].detach().requires_grad_()
    return s


# ------------------------------------------------------------------ plain forms
def _plain_topk(s):
    z = s["logits"].float()
    # unique keys: the value's bits in order of the values, then the lowest index
    bits = (z + 0.0).view(torch.int32)
    bits = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    key = (bits.long() << 32) + (0xFFFFFFFF - torch.arange(s["V"], device="cuda"))
    ids = torch.topk(key, s["k"], dim=1).indices
    z = z / s["temp"]
    top = z.amax(1, keepdim=True)
    lse = top + torch.exp(z - top).sum(1, keepdim=True).log()
    return {"logp": z.gather(1, ids) - lse, "ids": ids.to(torch.int32), "lse": lse.squeeze(1)}


def _plain_distill(s):
    w, T = s["row_weight"][:, None], s["temp"]
    c = s["label_weight"][:, None] if s["label"] else torch.zeros_like(w)
    # (sums over the vocabulary and the numbers of a row in 64 bits: the loss is a small difference of large ones)
    ids, l = s["list_ids"].long(), s["list_logp"].double()
    z = s["logits"].detach().float()
    y = s["label_id"].long()[:, None]
    top = z.amax(1, keepdim=True)
    e = torch.exp((z - top) / T)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    p = e / total.float()
    logp = (z.gather(1, ids) - top).double() / T - total.log()
    t = l.exp()
    if not s["rest"]:
        t = t / t.sum(1, keepdim=True)
        loss = (t * (t.log() - logp)).sum(1, keepdim=True)
        d = w * p
        d.scatter_add_(1, ids, (-w * t).float())
    else:
        t_rest = 1 - t.sum(1, keepdim=True)
        e.scatter_(1, ids, 0.0)  # what is outside the list
        outside = e.sum(1, keepdim=True, dtype=torch.float64)
        p_rest, logp_rest = outside / total, (outside / total).log()
        if s["kind"] == "forward":
            t_rest = t_rest.clamp_min(0.0)
            loss = (t * (l - logp)).sum(1, keepdim=True) + t_rest * (t_rest.clamp_min(1e-30).log() - logp_rest)
            d = e / outside.float() * (w * (p_rest - t_rest)).float()
            d.scatter_(1, ids, (w * (logp.exp() - t)).float())
        else:
            f, f_rest = logp - l, logp_rest - t_rest.clamp_min(REST_MIN).log()
            loss = (logp.exp() * f).sum(1, keepdim=True) + p_rest * f_rest
            d = p * (w * (f_rest - loss)).float()
            d.scatter_(1, ids, (w * logp.exp() * (f - loss)).float())
    if s["label"]:
        d.addcmul_(p, c)
        d.scatter_add_(1, y, -c)
    loss = (w * loss + c * (total.log() - (z.gather(1, y) - top).double() / T)).float()
    d = d / T if s["fused"] else d * (s["dloss"][:, None] / T)
    return {"loss": loss.squeeze(1), "dlogits": d.to(s["logits"].dtype)}


def _plain_embed(s):
    ids = s["ids"].long()
    W = s["weight"].detach()
    out = {"y": (W[ids].float() * s["scale"]).to(W.dtype)}
    if s["grad"] == "add":
        out["sum"] = s["sum"].index_add_(0, ids, s["dy"].float() * s["scale"])
    elif s["grad"] == "dense":
        d = torch.zeros(W.shape, device="cuda").index_add_(0, ids, s["dy"].float() * s["scale"])
        out["dweight"] = d.to(W.dtype)
    return out


def run(state):
    s = state
    if not own:
        return {"topk": _plain_topk, "distill": _plain_distill, "embed": _plain_embed}[s["op"]](s)
    if s["op"] == "topk":
        from turbol_b200.ops.distill import topk_logprobs

        logp, ids, lse = topk_logprobs(s["logits"], s["k"], temperature=s["temp"])
        return {"logp": logp, "ids": ids, "lse": lse}
    if s["op"] == "distill":
        from turbol_b200.ops.distill import distill_loss, distill_loss_grad

        label = dict(target=s["label_id"], target_weight=s["label_weight"]) if s["label"] else {}
        args = (s["logits"], s["list_ids"], s["list_logp"], s["row_weight"])
        how = dict(kind=s["kind"], rest=s["rest"], temperature=s["temp"], **label)
        if s["fused"]:
            loss, d = distill_loss_grad(*args, **how)
            return {"loss": loss, "dlogits": d}
        loss = distill_loss(*args, **how)
        d, = torch.autograd.grad(loss, s["logits"], s["dloss"])
        return {"loss": loss.detach(), "dlogits": d}
    from turbol_b200.ops.embedding import embedding, embedding_grad

    y = embedding(s["ids"], s["weight"], scale=s["scale"])
    out = {"y": y.detach()}
    if s["grad"] == "add":
        out["sum"] = embedding_grad(s["ids"], s["dy"], s["sum"], scale=s["scale"])
    elif s["grad"] == "dense":
        out["dweight"], = torch.autograd.grad(y, s["weight"], s["dy"])
    return out


# ------------------------------------------------------------------ work
def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "embed":
        N, H, V = case["N"], case["H"], case["V"]
        U = int(torch.unique(_ids(case)).numel())
        b = (U + N) * H * e + 4 * N
        if case["grad"] == "add":
            b += N * H * e + 2 * U * H * 4
        elif case["grad"] == "dense":
            b += N * H * e + V * H * e
        return {"bytes": b, "flops": N * H * (1 if case["grad"] == "none" else 3)}
    R, V = case["R"], case["V"]
    if case["op"] == "topk":
        return {"bytes": R * V * e + R * (8 * case["k"] + 4), "flops": 4 * R * V}
    live = R if case["label"] else int(_weights(case).sum())
    return {"bytes": (live + R) * V * e + R * (8 * case["K"] + 16), "flops": 8 * live * V}


# ------------------------------------------------------------------ 64 bits
def _exact_rows(s, lo, hi):
    """Loss and gradient of rows lo .. hi by differentiating the loss's definition."""
    z = s["logits"][lo:hi].detach().double().requires_grad_()
    ids, l = s["list_ids"][lo:hi].long(), s["list_logp"][lo:hi].double()
    with torch.enable_grad():
        logp = torch.log_softmax(z / s["temp"], 1)
        if not s["rest"]:
            lt = torch.log_softmax(l, 1)
            loss = (lt.exp() * (lt - logp.gather(1, ids))).sum(1)
        else:
            inside = torch.zeros(z.shape, dtype=torch.bool, device="cuda").scatter_(1, ids, True)
            r = torch.logsumexp(logp.masked_fill(inside, -math.inf), 1)
            tr = 1 - l.exp().sum(1)
            lp = logp.gather(1, ids)
            if s["kind"] == "forward":
                tr = tr.clamp_min(0)
                loss = (l.exp() * (l - lp)).sum(1) + torch.xlogy(tr, tr) - tr * r
            else:
                loss = (lp.exp() * (lp - l)).sum(1) + r.exp() * (r - tr.clamp_min(REST_MIN).log())
        loss = s["row_weight"][lo:hi].double() * loss
        if s["label"]:
            y = s["label_id"][lo:hi].long()
            loss = loss - s["label_weight"][lo:hi].double() * logp[torch.arange(hi - lo, device="cuda"), y]
        g = torch.ones_like(loss) if s["fused"] else s["dloss"][lo:hi].double()
        d, = torch.autograd.grad(loss, z, g)
    return loss.detach(), d


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        W, ids = s["weight"].detach(), s["ids"].long()
        out = {"y": W.double()[ids] * case["scale"]}
        if case["grad"] != "none":
            g = s["sum"].double() if case["grad"] == "add" else torch.zeros(W.shape, dtype=torch.float64, device="cuda")
            order = torch.argsort(ids, stable=True)
            rows, count = torch.unique_consecutive(ids[order], return_counts=True)
            ends = count.cumsum(0).tolist()
            dy, rows = s["dy"], rows.tolist()
            for v, hi, n in zip(rows, ends, count.tolist()):
                if n > 1:
                    g[v] += dy[order[hi - n:hi]].double().sum(0) * case["scale"]
            one = order[(count.cumsum(0) - 1)[count == 1]]
            g[ids[one]] += dy[one].double() * case["scale"]
            out["sum" if case["grad"] == "add" else "dweight"] = g
        return out
    R, V = case["R"], case["V"]
    step = max(1, (1 << 25) // V)
    if case["op"] == "topk":
        logp, ids, lse = [], [], []
        for lo in range(0, R, step):
            x = s["logits"][lo:lo + step].double() + 0.0
            x, order = torch.sort(x, dim=1, descending=True, stable=True)
            lse.append(torch.logsumexp(x / case["temp"], 1))
            logp.append(x[:, :case["k"]] / case["temp"] - lse[-1][:, None])
            ids.append(order[:, :case["k"]].to(torch.int32))
        return {"logp": torch.cat(logp), "ids": torch.cat(ids), "lse": torch.cat(lse)}
    parts = [_exact_rows(s, lo, min(R, lo + step)) for lo in range(0, R, step)]
    return {"loss": torch.cat([a for a, _ in parts]), "dlogits": torch.cat([b for _, b in parts])}
