"""The distillation and the scaled embedding where the framework uses them: GRPO with a
teacher, the decoder's embedding in training and in the rollout."""
import math
import os
import sys

import pytest
import torch

from turbol_b200.models.llm import DecoderLM, LMConfig
from turbol_b200.ops import reference as ref
from turbol_b200.rl.grpo import GRPOConfig, GRPOTrainer

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def tiny(**kw):
    cfg = LMConfig.tiny()
    for k, v in kw.items():
        setattr(cfg, k, v)
    return cfg


def config(**kw):
    return GRPOConfig(**{**dict(model=tiny(), num_prompts=2, group_size=4, prompt_len=20, response_len=12, micro_batch=4), **kw})


def test_refusals():
    for kw in (dict(distill_coef=0.1, distill_kind="both"), dict(distill_coef=0.1, distill_topk=0),
               dict(distill_coef=0.1, distill_topk=257), dict(distill_coef=-1.0), dict(distill_coef=math.nan)):
        with pytest.raises(ValueError, match="distill"):
            GRPOTrainer(config(**kw), "cpu")
    with pytest.raises(ValueError, match="tensor parallelism"):
        GRPOTrainer(config(distill_coef=0.1), "cpu", tp=2)
    teacher = DecoderLM(tiny(), "cpu", master=False)
    with pytest.raises(ValueError, match="needs distill_coef"):
        GRPOTrainer(config(), "cpu", teacher=teacher)
    for t in (DecoderLM(tiny(vocab=1000), "cpu", master=False), DecoderLM(tiny(max_seq=16), "cpu", master=False)):
        with pytest.raises(ValueError, match="teacher"):
            GRPOTrainer(config(distill_coef=0.1), "cpu", teacher=t)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["forward", "reverse"])
@pytest.mark.parametrize("tie", [True, False])
def test_gradient_of_the_training_loss(kind, tie, dev):
    """The micro-batched update's gradient (policy loss, KL penalty, distillation; scaled embedding) against autograd on
    the fp32 model."""
    cfg = config(model=tiny(embed_scale=4.0, tie_embeddings=tie), distill_coef=0.7, distill_topk=24, distill_kind=kind, kl_coef=0.1)
    tr = GRPOTrainer(cfg, dev, teacher=DecoderLM(tiny(tie_embeddings=tie), dev, seed=11, master=False))
    g = torch.Generator(device=dev).manual_seed(2)
    seqs = torch.randint(0, cfg.model.vocab, (cfg.batch, cfg.seq_len), generator=g, device=dev, dtype=torch.int32)
    adv = torch.randn(cfg.batch, generator=g, device=dev)
    lists = tr._teacher_lists(cfg.batch)
    tr._score(tr.teacher, seqs, lists=lists)
    ref_lp = tr.ref_logprobs(seqs) + 0.1 * torch.randn(cfg.batch, cfg.response_len, generator=g, device=dev)
    tr.model.zero_grad()
    tr.stats.zero_()
    tr._train(seqs, ref_lp, adv, lists)
    m = tr.model
    leaves = {n: (m.p[n] if n.endswith(("ln1", "ln2", "norm", "bqkv")) else m.s[n].float()).clone().requires_grad_()
              for n in m.offsets}
    Lp, B, L = cfg.prompt_len, cfg.batch, cfg.response_len
    logits = ref.lm_forward_ref(m, seqs, leaves)[:, Lp - 1:-1]
    lsm = torch.log_softmax(logits, -1)
    lp = lsm.gather(2, seqs[:, Lp:].long()[..., None]).squeeze(2)
    pg = -(torch.exp(lp - lp.detach()) * adv[:, None])
    k3 = torch.exp(ref_lp - lp) - (ref_lp - lp) - 1
    ids, l = lists[0].long(), lists[1]
    top = lsm.gather(2, ids)
    inside = torch.zeros_like(lsm, dtype=torch.bool).scatter_(2, ids, True)
    rest = torch.logsumexp(lsm.masked_fill(inside, -math.inf), -1)
    t_rest = 1 - l.double().exp().sum(-1).float()
    if kind == "forward":
        kl = (l.exp() * (l - top)).sum(-1) + t_rest * (t_rest.log() - rest)
    else:
        kl = (top.exp() * (top - l)).sum(-1) + rest.exp() * (rest - t_rest.log())
    (pg + cfg.kl_coef * k3 + cfg.distill_coef * kl).mean().backward()
    mean = float(kl.detach().mean())
    assert abs(float(tr.distill_kl) - mean) <= 0.03 * mean
    for n in m.offsets:
        e = leaves[n].grad
        assert (m.g[n] - e).norm() / e.norm() < 5e-2, n


@pytest.mark.gpu
def test_steps(dev):
    """The frozen reference as teacher: no distance in the first step; another teacher: some; the same seeds, the same
    gradients of the embedding."""
    tr = GRPOTrainer(config(distill_coef=0.1, distill_topk=16), dev)
    assert tr.teacher is tr.ref
    st = [tr.step() for _ in range(2)]
    assert abs(st[0]["distill_kl"]) < 1e-4 and all(math.isfinite(s["distill_kl"]) for s in st)
    tr = GRPOTrainer(config(distill_coef=0.1, distill_kind="reverse"), dev, teacher=DecoderLM(tiny(), dev, seed=5, master=False))
    st = tr.step()
    assert math.isfinite(st["pg_loss"]) and st["distill_kl"] > 1e-3
    assert "distill_kl" not in GRPOTrainer(config(), dev).step()


def test_device_names():
    """A teacher on the trainer's device under another of its names passes the checks (what comes after them needs a GPU)."""
    try:
        GRPOTrainer(config(distill_coef=0.1), "cpu", teacher=DecoderLM(tiny(), "cpu:0", master=False))
    except Exception as e:
        assert "teacher" not in str(e)


@pytest.mark.gpu
def test_device_names_on_the_gpu(dev):
    here = torch.cuda.current_device()
    for name, teachers in ((f"cuda:{here}", "cuda"), ("cuda", f"cuda:{here}")):
        tr = GRPOTrainer(config(distill_coef=0.1), name, teacher=DecoderLM(tiny(), teachers, seed=5, master=False))
        assert math.isfinite(tr.step()["distill_kl"])


@pytest.mark.gpu
def test_scaled_embedding_in_the_rollout(dev):
    """Greedy tokens of a model with scaled embeddings are those of its fp32 forward (up to its bf16 rounding)."""
    from turbol_b200.rl.rollout import LLMGenerator

    m = DecoderLM(tiny(embed_scale=16.0), dev, seed=3)
    prompts = torch.randint(0, m.cfg.vocab, (2, 21), device=dev, dtype=torch.int32)
    for graph in (True, False):
        seqs, lp = LLMGenerator(m, 4, 64, cuda_graph=graph).generate(prompts, 2, 10, temperature=0.0)
        lg = ref.lm_forward_ref(m, seqs)[:, 20:-1]
        picked = lg.gather(2, seqs[:, 21:].long()[..., None]).squeeze(2)
        spread = lg.amax(-1) - lg.mean(-1)
        assert ((lg.amax(-1) - picked) <= 0.2 * spread).all()
    x, plain = m.embed(prompts), m.s["embed"][prompts.reshape(-1).long()]
    assert torch.equal(x, plain * 16)


@pytest.mark.gpu
def test_embedding_gradient_is_reproducible(dev):
    """Many tokens of few kinds: the same bits every time, and the sums of the older kernel within rounding."""
    from turbol_b200._native import ops

    m = DecoderLM(tiny(), dev)
    ids = torch.randint(0, 9, (8, 300), device=dev, dtype=torch.int32)
    dx = torch.randn(2400, m.cfg.hidden, device=dev).bfloat16()
    got = []
    for _ in range(3):
        m.zero_grad()
        m.embed_backward(ids, dx)
        got.append(m.g["embed"].clone())
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    old = torch.zeros_like(got[0])
    ops().embed_bwd(ids.reshape(-1), dx, old)
    # two fp32 sums of some 270 terms each in different orders
    mag = torch.zeros_like(old).index_add_(0, ids.reshape(-1).long(), dx.float().abs())
    assert ((old - got[0]).abs() <= 2 * 400 * 2.0 ** -24 * mag).all()


@pytest.mark.gpu
def test_example(tmp_path, dev):
    import grpo_example

    tr = grpo_example.main(["--num-prompts", "2", "--group-size", "4", "--prompt-len", "16", "--max-tokens", "16",
                            "--num-steps", "2", "--print-every", "1", "--micro-batch", "4", "--distill-coef", "0.2",
                            "--distill-topk", "20", "--distill-kind", "reverse", "--log-dir", str(tmp_path)])
    assert tr.step_count == 2 and math.isfinite(float(tr.distill_kl))


@pytest.mark.gpu
def test_resume_with_the_same_teacher(tmp_path, dev):
    """A run that distils towards a given model goes on with that model alone; the frozen reference is saved with the
    run; states without the entry load as they did."""
    from turbol_b200.utils.checkpoint import load_checkpoint, save_checkpoint

    def trainer(seed=None):
        teacher = None if seed is None else DecoderLM(tiny(), dev, seed=seed, master=False)
        return GRPOTrainer(config(distill_coef=0.1, distill_topk=16), dev, teacher=teacher)

    given, own = trainer(5), trainer()
    given.step()
    save_checkpoint(str(tmp_path / "given"), 1, given)
    save_checkpoint(str(tmp_path / "own"), 1, own)
    again = trainer(5)
    load_checkpoint(str(tmp_path / "given"), trainer=again)
    assert torch.equal(again.model.flat, given.model.flat) and again.step_count == 1
    for where, seed in (("given", None), ("given", 6), ("own", 5)):
        tr = trainer(seed)
        before = tr.model.flat.clone()
        with pytest.raises(ValueError, match="teacher"):
            load_checkpoint(str(tmp_path / where), trainer=tr)
        assert torch.equal(tr.model.flat, before)
        load_checkpoint(str(tmp_path / where), trainer=tr, strict_config=False)
        assert torch.equal(tr.model.flat, (given if where == "given" else own).model.flat)
    load_checkpoint(str(tmp_path / "own"), trainer=trainer())
    sd = given.state_dict()
    del sd["teacher"]
    trainer(6).load_state_dict(sd)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, 16.0])
def test_ids_outside_the_table_do_not_depend_on_the_scale(scale, dev):
    """The decoder's embedding reads row 0 for them and gives them no gradient."""
    m = DecoderLM(tiny(embed_scale=scale), dev, seed=3)
    ids = torch.tensor([[5, -1, m.cfg.vocab, m.cfg.vocab - 1]], dtype=torch.int32, device=dev)
    want = m.s["embed"][torch.tensor([5, 0, 0, m.cfg.vocab - 1], device=dev)] * scale
    assert torch.equal(m.embed(ids), want)
    m.zero_grad()
    m.embed_backward(ids, torch.ones(4, m.cfg.hidden, device=dev, dtype=torch.bfloat16))
    rows = m.g["embed"].abs().sum(1).nonzero().squeeze(1).tolist()
    assert rows == [5, m.cfg.vocab - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["forward", "reverse"])
def test_the_distance_does_not_depend_on_its_weight(kind, dev):
    """distill_kl beside a policy loss of ordinary size: the same for a coefficient of 1e-7 (the logits are the same;
    sums of 96 numbers in one order, so the same bits)."""
    got = []
    for coef in (1.0, 1e-7):
        tr = GRPOTrainer(config(distill_coef=coef, distill_topk=16, distill_kind=kind), dev,
                         teacher=DecoderLM(tiny(), dev, seed=11, master=False))
        g = torch.Generator(device=dev).manual_seed(2)
        n = tr.cfg.batch
        seqs = torch.randint(0, tr.cfg.model.vocab, (n, tr.cfg.seq_len), generator=g, device=dev, dtype=torch.int32)
        lists = tr._teacher_lists(n)
        tr._score(tr.teacher, seqs, lists=lists)
        tr.model.zero_grad()
        tr._train(seqs, tr.ref_logprobs(seqs), torch.randn(n, generator=g, device=dev), lists)
        got.append(float(tr.distill_kl))
    assert got[0] > 1e-3 and got[0] == got[1]


@pytest.mark.gpu
def test_the_same_seeds_give_the_same_embedding_gradient(dev):
    """Two trainers of the same seeds: the same bits in the embedding's gradient after an update's backward passes
    (the head of its own: what is compared is the lookup's)."""
    got = []
    for _ in range(2):
        tr = GRPOTrainer(config(model=tiny(tie_embeddings=False), distill_coef=0.1, distill_topk=16), dev)
        g = torch.Generator(device=dev).manual_seed(2)
        seqs = torch.randint(0, 40, (tr.cfg.batch, tr.cfg.seq_len), generator=g, device=dev, dtype=torch.int32)
        lists = tr._teacher_lists(tr.cfg.batch)
        ref_lp = tr.ref_logprobs(seqs, lists)
        tr.model.zero_grad()
        tr._train(seqs, ref_lp, torch.randn(tr.cfg.batch, generator=g, device=dev), lists)
        got.append(tr.model.g["embed"].clone())
    assert got[0].abs().sum() > 0 and torch.equal(*got)
