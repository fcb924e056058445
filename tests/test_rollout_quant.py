"""The rollout engine on the 8-bit KV cache, and the decoder with rotary positions other than the default."""
import math

import pytest
import torch

from turbol_b200.models.llm import DecoderLM, LMConfig, apply_rope, rope_table
from turbol_b200.ops import reference as ref

ROPES = [dict(rotary_dim=64), dict(rope_interleaved=True),
         dict(rotary_dim=32, rope_interleaved=True, rope_scaling={"type": "linear", "factor": 4.0}),
         dict(rope_scaling={"type": "llama3", "factor": 8.0, "original_max_pos": 64}),
         dict(rope_scaling={"type": "yarn", "factor": 4.0, "original_max_pos": 64})]


def tiny(**kw):
    cfg = LMConfig.tiny()
    for k, v in kw.items():
        setattr(cfg, k, v)
    cfg.init_std = 0.05
    return cfg


def test_config():
    assert LMConfig().rope_default and LMConfig(rotary_dim=128).rope_default
    for kw in ROPES:
        assert not tiny(**kw).rope_default
    plain = rope_table(tiny(), "cpu")
    assert plain.shape == (1024, 64, 2)
    assert rope_table(tiny(rotary_dim=64), "cpu").shape == (1024, 32, 2)
    assert torch.equal(rope_table(tiny(rope_interleaved=True), "cpu"), plain)
    for bad in (12, 0, 136):
        with pytest.raises(ValueError):
            rope_table(tiny(rotary_dim=bad, rope_interleaved=True), "cpu")


def test_kv_dtype_refused():
    from turbol_b200.rl.grpo import GRPOConfig, GRPOTrainer
    from turbol_b200.rl.rollout import LLMGenerator

    with pytest.raises(ValueError):
        GRPOTrainer(GRPOConfig(model=tiny(), kv_dtype="int3"), "cpu")
    with pytest.raises(ValueError):
        GRPOTrainer(GRPOConfig(model=tiny(), kv_dtype="fp8"), "cpu", dp="none", tp=2, tp_mode="rollout")
    with pytest.raises(ValueError):
        LLMGenerator(DecoderLM(tiny(), "cpu", master=False), 2, 32, kv_dtype="fp4")


@pytest.mark.gpu
@pytest.mark.parametrize("kw", ROPES)
def test_decoder_with_other_rotary_positions(kw, dev):
    """Forward against the fp32 model, gradients against its autograd."""
    m = DecoderLM(tiny(**kw), dev, seed=3)
    cfg = m.cfg
    B, T = 2, 64
    ids = torch.randint(0, cfg.vocab, (B, T), device=dev, dtype=torch.int32)
    pos = torch.arange(T, device=dev, dtype=torch.int32).repeat(B)
    x, saved = m.forward(m.embed(ids), B, T, pos, save=True)
    rstd = torch.empty(B * T, device=dev)
    hf = m.final_norm(x, rstd)
    logits = m.logits(hf).float().view(B, T, -1)
    leaves = {n: m.s[n].float().requires_grad_() for n in m.offsets}
    exp = ref.lm_forward_ref(m, ids, leaves)
    assert (logits - exp).abs().max() / exp.abs().max() < 3e-2
    other = DecoderLM(tiny(), dev, seed=3)
    plain = ref.lm_forward_ref(other, ids)
    assert (exp.detach() - plain).abs().max() / plain.abs().max() > 3e-2  # the positions matter at this size
    g = (torch.randn(B * T, cfg.hidden, device=dev) * 0.01).to(torch.bfloat16)
    m.zero_grad()
    m.backward(g, saved, B, T, pos)
    h = leaves["embed"][ids.long()]
    # the reference's residual stream before the final norm, rebuilt by differentiating through the layers alone
    P = leaves
    xr = h
    posr = torch.arange(T, device=dev)
    for i in m.layers:
        p = f"l{i}."
        a = ref.rmsnorm(xr, P[p + "ln1"], cfg.rms_eps)
        qkv = a @ P[p + "wqkv"].t() + P[p + "bqkv"]
        D = cfg.head_dim
        q, k, v = qkv.split((cfg.q_dim, cfg.kv_dim, cfg.kv_dim), -1)
        q, k = (ref.rotary(t.reshape(B * T, -1, D), posr.repeat(B), m.table, cfg.rope_interleaved).view(B, T, -1, D)
                for t in (q, k))
        xr = xr + ref.causal_attention(q, k, v.view(B, T, -1, D)).reshape(B, T, -1) @ P[p + "wo"].t()
        b = ref.rmsnorm(xr, P[p + "ln2"], cfg.rms_eps) @ P[p + "wgu"].t()
        xr = xr + (torch.nn.functional.silu(b[..., 0::2]) * b[..., 1::2]) @ P[p + "wdown"].t()
    xr.backward(g.float().view(B, T, -1))
    for n in ("l0.wqkv", "l1.wqkv", "l0.wo", "l0.wgu"):
        e = leaves[n].grad
        assert (m.g[n] - e).norm() / e.norm() < 5e-2, n


@pytest.mark.gpu
def test_apply_rope_default_is_the_old_kernel(dev):
    from turbol_b200._native import ops

    cfg = tiny()
    table = rope_table(cfg, dev)
    qkv = torch.randn(33, cfg.qkv_dim, device=dev).bfloat16()
    pos = torch.arange(33, device=dev, dtype=torch.int32)
    a, b = qkv.clone(), qkv.clone()
    ops().rope(a, pos, table, 6, 128)
    apply_rope(cfg, table, b, pos, 6)
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}] + ROPES[1:3])
@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("Lp", [16, 21])
def test_generate(kv_dtype, kw, Lp, dev):
    """Greedy decoding: the cache holds what a full forward computes (its first layer exactly up to the roundings), the
    captured step decodes like the uncaptured one, and each token is the argmax of the full model's logits or close to
    it."""
    from turbol_b200.rl.rollout import LLMGenerator

    m = DecoderLM(tiny(**kw), dev, seed=3)
    cfg, P, G, new = m.cfg, 3, 2, 20
    g = torch.Generator().manual_seed(1)
    prompts = torch.randint(0, cfg.vocab, (P, Lp), generator=g, dtype=torch.int32).to(dev)
    outs = []
    for graph in (True, False):
        gen = LLMGenerator(m, P * G, 64, cuda_graph=graph, kv_dtype=kv_dtype)
        outs.append(gen.generate(prompts, G, new, temperature=0.0))
        if kv_dtype == "fp8":
            assert int(gen.kv_error) == 0
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    seqs = outs[0][0]
    n = Lp + new - 1  # the last sampled token is not in the cache
    # layer 0's keys and values come from the embeddings alone
    x = m.embed(seqs[:, :n].contiguous())
    h = torch.empty_like(x)
    from turbol_b200._native import ops

    ops().rmsnorm_fwd(x, m.f32["l0.ln1"], h, None, cfg.rms_eps)
    qkv = h.double() @ m.s["l0.wqkv"].double().t() + m.f32["l0.bqkv"].double()
    pos = torch.arange(n, device=dev).repeat(P * G)
    k = qkv[:, cfg.q_dim:cfg.q_dim + cfg.kv_dim].view(-1, cfg.n_kv_heads, cfg.head_dim)
    v = qkv[:, cfg.q_dim + cfg.kv_dim:].view(k.shape)
    # fp32 sums of `hidden` products, rounded to bf16, rotated (each element mixes two), rounded again, and quantised
    size = h.double().abs() @ m.s["l0.wqkv"].double().abs().t()
    acc = 2.0 ** -24 * cfg.hidden * size.amax()
    if cfg.rope_default:
        k = ref.rotary(k, pos, m.table.double())
    else:
        k = ref.rotary(k, pos, m.table.double(), cfg.rope_interleaved)
    step = 2.0 ** -4 if kv_dtype == "fp8" else 0.0
    for s in range(P * G):
        ck, cv = gen.cached_kv(0, s, n)
        for got, want in ((ck, k[s * n:(s + 1) * n]), (cv, v[s * n:(s + 1) * n])):
            amax = want.abs().amax(-1, keepdim=True)
            tol = want.abs() * (step + 2.0 ** -8) + amax * (2 * 2.0 ** -8 * math.sqrt(2) + step * 2.0 ** -13) + acc
            assert ((got.double() - want).abs() <= tol).all()
    # every greedy token against the full model on the same prefix
    logits = ref.lm_forward_ref(m, seqs[:, :-1].contiguous())[:, Lp - 1:]
    top, picked = logits.amax(-1), logits.gather(-1, seqs[:, Lp:, None].long()).squeeze(-1)
    spread = logits.std()
    assert ((top - picked) <= (0.5 if kv_dtype == "fp8" else 0.2) * spread).all()
    with pytest.raises(ValueError):
        gen.cached_kv(0, P * G, n)


@pytest.mark.gpu
def test_fp8_rollout_in_the_trainer_and_engine(dev):
    from turbol_b200.rl.grpo import GRPOConfig, GRPOTrainer
    from turbol_b200.rl.rollout import RolloutConfig, RolloutEngine

    cfg = GRPOConfig(model=tiny(), num_prompts=2, group_size=4, prompt_len=20, response_len=12, micro_batch=4,
                     kv_dtype="fp8")
    tr = GRPOTrainer(cfg, dev)
    assert tr.gen.kv_dtype == "fp8"
    for _ in range(2):
        st = tr.step()
        assert all(math.isfinite(st[k]) for k in ("pg_loss", "kl", "rollout_logp_mean"))
    assert int(tr.gen.kv_error) == 0
    e = RolloutEngine(RolloutConfig(max_new_tokens=6, max_batch_size=4, kv_dtype="fp8"))
    e.initialize()
    assert len(e.generate_batch(["one", "another prompt"])) == 2
    e.shutdown()


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
def test_positions_past_the_model_are_refused(kv_dtype):
    """A prompt and answer longer than the model's table of positions: refused by generate before anything runs."""
    from turbol_b200.rl.rollout import LLMGenerator, TPLLMGenerator

    m = DecoderLM(tiny(max_seq=32), "cpu", master=False)
    gen = LLMGenerator(m, 2, 64, kv_dtype=kv_dtype)
    tp = TPLLMGenerator.__new__(TPLLMGenerator)
    tp.m, tp.cfg, tp.tpm, tp.max_batch, tp.max_len = m, m.cfg, type("TP", (), {"tp": 1, "rank": 0}), 2, 64
    for g in (gen, tp):
        for Lp, new in ((33, 1), (32, 2), (16, 18), (1, 33)):
            with pytest.raises(ValueError, match="max_seq"):
                g.generate(torch.zeros(1, Lp, dtype=torch.int32), 2, new)
        with pytest.raises(ValueError, match="capacity"):
            g.generate(torch.zeros(1, 16, dtype=torch.int32), 3, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [True, False])
def test_generate_reports_cache_errors(graph, dev):
    """A block out of range in the table of one sequence: the kernels skip it, and generate says so instead of
    returning; the next call, on sound tables, runs."""
    from turbol_b200.rl.rollout import LLMGenerator

    m = DecoderLM(tiny(), dev, seed=3)
    gen = LLMGenerator(m, 4, 64, cuda_graph=graph, kv_dtype="fp8")
    prompts = torch.arange(32, dtype=torch.int32, device=dev).view(2, 16)
    want = gen.generate(prompts, 2, 12, temperature=0.0)
    tables = gen._tables

    def broken(*args):
        table, *rest = tables(*args)
        table[3, 1] = gen.num_blocks + 7  # the block of the first decoded tokens
        return (table, *rest)

    gen._tables = broken
    with pytest.raises(RuntimeError, match="out of range"):
        gen.generate(prompts, 2, 12, temperature=0.0)
    gen._tables = tables
    again = gen.generate(prompts, 2, 12, temperature=0.0)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
def test_cached_kv_before_generate(kv_dtype):
    from turbol_b200.rl.rollout import LLMGenerator

    gen = LLMGenerator(DecoderLM(tiny(), "cpu", master=False), 2, 32, kv_dtype=kv_dtype)
    for layer in (0, 99):
        with pytest.raises(ValueError):
            gen.cached_kv(layer, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
def test_cached_kv_ends_where_the_cache_does(kv_dtype, dev):
    """No rows past the tokens that were written (they would come from other sequences' blocks): the last sampled token
    is not among them, nor is what an early stop left out."""
    from turbol_b200.rl.rollout import LLMGenerator

    gen = LLMGenerator(DecoderLM(tiny(), dev, seed=3), 4, 64, kv_dtype=kv_dtype)
    prompts = torch.arange(40, dtype=torch.int32, device=dev).view(2, 20)
    for new, eos, want in ((1, -1, 20), (9, -1, 28), (30, None, None)):
        if eos is None:  # a token that every sequence samples at once: stops at the first check
            eos = int(gen.generate(prompts[:1], 1, 1, temperature=0.0)[0][0, -1])
            gen.generate(prompts[:1], 2, new, temperature=0.0, eos_id=eos, stop_check=4)
            want = 24
        else:
            gen.generate(prompts, 2, new, temperature=0.0)
        assert gen.cached == want
        assert gen.cached_kv(1, 1, want)[0].shape == (want, gen.cfg.n_kv_heads, gen.cfg.head_dim)
        for seq, n in ((0, want + 1), (0, -1), (4, 1), (-1, 1)):
            with pytest.raises(ValueError):
                gen.cached_kv(0, seq, n)


@pytest.mark.parametrize("backend", ["native", "echo", "vllm"])
def test_engine_checks_its_kv_dtype(backend):
    """Unknown caches are refused whatever the backend, and an 8-bit one where the backend would not use it."""
    from turbol_b200.rl.rollout import RolloutConfig, RolloutEngine

    with pytest.raises(ValueError, match="kv_dtype"):
        RolloutEngine(RolloutConfig(inference_backend=backend, kv_dtype="int3", device="cpu")).initialize()
    if backend == "vllm":
        with pytest.raises(ValueError, match="kv_dtype"):
            RolloutEngine(RolloutConfig(inference_backend=backend, kv_dtype="fp8", device="cpu")).initialize()
    elif backend == "echo":
        e = RolloutEngine(RolloutConfig(inference_backend=backend, kv_dtype="fp8"))
        e.initialize()
        assert e.generate("x") == "[RolloutEngine] x"
