"""Sequences that go on from one another, through the engine: every architecture's steps after a fork give the logits of sequences that were run by
themselves; replies behind a common prefix are the replies to the whole prompts; beam search finds what a search over whole sequences finds."""
import numpy as np
import pytest
import torch

from conftest import TINY_B, TINY_C, TINY_D, close
from quicknn_b200.engine import LLM, PromptError
from quicknn_b200.kernels import ops
from quicknn_b200.sampling import BeamOptions, GenerationOptions, OptionsError

pytestmark = pytest.mark.gpu

ROT = {"base": 1000.0, "dims": 8}
ATT = {"heads": 4, "kv_heads": 2, "dim": 8, "vdim": 12, "scale": 0.3, "rot": ROT}
MATT = {"heads": 4, "kv_heads": 2, "dim": 8, "vdim": 12, "scale": 0.3, "mask": {"size": 100}}
FF = {"kind": "dense", "ff": 64}
LMOE = {"kind": "moe", "expert": {"ff": 16, "limit": 0.8}, "router": {"experts": 5, "top": 2}}
CONFIGS = {
    "gemma-b": TINY_B, "gemma-c": TINY_C, "gemma-d": TINY_D,
    "fuposun": dict(architecture="Fuposun", vocab=211, width=48, residual_mult=0.8, logit_softcap=25.0, norm={"eps": 1e-5}, initializer_range=0.1, layers=[
        {"type": "gla", "mixer": {"heads": 2, "dim": 8, "vdim": 16, "tau": 6.0, "decay_rank": 4}, "mlp": FF},
        {"type": "latent_attention", "mixer": {"heads": 2, "dim": 8, "vdim": 12, "q_rank": 16, "kv_rank": 24, "scale": 0.35, "mask": {"size": 70}},
         "mlp": {"kind": "moe", "router": {"experts": 4, "top": 2}, "expert": {"ff": 24, "limit": 0.6}, "shared": {"ff": 16, "limit": 0.9}}}]),
    "tumudra": dict(architecture="Tumudra", vocab=211, width=48, embedding={"scale": 2.0}, norm={"eps": 1e-5}, initializer_range=0.1, layers=[
        {"type": "parallel", "mlp": FF, "mixer": {"left": {"heads": 2, "kv_heads": 1, "dim": 16, "vdim": 8, "scale": 0.25, "mask": {"size": 6}, "rot": dict(ROT, dims=8)},
                                                  "right": {"heads": 2, "dim": 8, "vdim": 16, "gate_cap": 8.0}}},
        {"type": "attention", "mixer": ATT, "mlp": FF},
        {"type": "retention", "mixer": {"heads": 2, "dim": 8, "vdim": 16, "decay": [0.9, 0.99], "rot": ROT}, "mlp": None},
        {"type": "attention", "mixer": dict(ATT, kv_from=1), "mlp": FF}]),
    "mubasun": dict(architecture="Mubasun", vocab=211, width=48, max_positions=512, norm={"eps": 1e-5, "groups": 3}, initializer_range=0.1, layers=[
        {"type": "attention", "mixer": MATT, "mlp": FF},
        {"type": "attention", "mixer": dict(MATT, kv_from=0, mask={"size": 300}), "mlp": {"kind": "moe", "expert": {"ff": 16}, "shared": {"ff": 24},
                                                                                         "router": {"experts": 4, "identity": 1, "top": 2, "scale": 1.5}}},
        {"type": "attention", "mixer": {"heads": 2, "kv_heads": 1, "dim": 16, "vdim": 8, "scale": 0.25}, "mlp": None}]),
    "gunirax": dict(architecture="Gunirax", vocab=211, width=48, embedding={"scale": 2.0}, norm={"eps": 1e-5}, initializer_range=0.1, loop={"start": 0, "stop": 1, "times": 2}, layers=[
        {"type": "parallel", "mixer": {"left": {"heads": 4, "kv_heads": 2, "dim": 8, "vdim": 8, "scale": 0.3, "mask": {"size": 5}, "rot": dict(ROT, dims=4)},
                                       "right": {"heads": 2, "dim": 8, "vdim": 16, "decay": [0.8, 0.99]}}, "mlp": FF},
        {"type": "hgrn2", "mixer": {"heads": 2, "dim": 8, "vdim": 12}, "mlp": FF}]),
    "linedra": dict(architecture="Linedra", vocab=211, width=48, embedding={"scale": 2.0}, norm={"eps": 1e-5}, canon={"taps": 3}, residual_mult=0.8, logit_softcap=25.0, initializer_range=0.1, layers=[
        {"type": "parallel", "mlp": LMOE, "mixer": {"left": {"heads": 4, "kv_heads": 2, "dim": 8, "vdim": 12, "scale": 0.3, "mask": {"size": 130}},
                                                  "right": {"width": 32, "blocks": 2, "conv": 4}, "left_scale": 0.7, "right_scale": 1.3}},
        {"type": "latent_attention", "mlp": None, "mixer": {"heads": 2, "dim": 8, "rot_dim": 4, "vdim": 12, "q_rank": 16, "kv_rank": 20, "scale": 0.3, "rot": dict(ROT, dims=4)}}]),
    "vonulorn": dict(architecture="Vonulorn", vocab=211, width=48, norm={"eps": 1e-5}, residual_mult=0.8, initializer_range=0.1, layers=[
        {"type": "delta", "mlp": FF, "mixer": {"heads": 4, "kv_heads": 2, "dim": 16, "vdim": 8, "conv": 4}},
        {"type": "attention", "mlp": None, "mixer": {"heads": 4, "kv_heads": 2, "dim": 8, "vdim": 12, "scale": 0.3, "softcap": 12.0, "diff": 0.4, "q_temp": {"coef": 0.2, "every": 4}}},
        {"type": "latent_attention", "mlp": FF, "mixer": {"heads": 2, "dim": 8, "rot_dim": 4, "vdim": 12, "q_rank": 16, "kv_rank": 20, "scale": 0.3, "rot": dict(ROT, dims=4)}}]),
}


def load(name, dtype="float32", **kw):
    return LLM.random(CONFIGS[name], 3, dtype=dtype, norm_std=0.15, **{**dict(max_context=448, max_batch=8), **kw})


@pytest.fixture
def shared_calls(monkeypatch):
    calls = []
    real = ops.attn_decode_shared
    monkeypatch.setattr(ops, "attn_decode_shared", lambda *a, **k: calls.append(a[0].shape[0]) or real(*a, **k))
    return calls


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", sorted(CONFIGS))
@pytest.mark.parametrize("prefix", [40, 330])
def test_steps_after_a_fork(name, dtype, prefix, shared_calls, monkeypatch):
    if prefix == 330:                                                      # common keys read once, however few they are
        monkeypatch.setattr(ops, "shared_attention_pays", lambda *a: True)
    llm = load(name, dtype)
    eng, V = llm.engine, llm.model.spec.embedding.vocab_size
    rng = np.random.default_rng(prefix)
    text = rng.integers(1, V, prefix).tolist()
    tails = rng.integers(1, V, (4, 70)).tolist()
    base = eng.new_sequence()
    eng.step([(base, text)], [()])
    a, b = eng.fork([base, base])
    rows, said = [base, a, b], [list(text) for _ in range(3)]
    fed = [0, 0, 0]

    def check(logits, seqs):
        for row, seq in zip(logits, seqs):
            ok, err, tol = close(row.cpu().numpy(), llm.evaluate_tokens(seq), dtype)
            assert ok, (len(seq), err, tol)

    def decode(n):
        for _ in range(n):
            toks = [tails[i][fed[i]] for i in range(len(rows))]
            for i, t in enumerate(toks):
                said[i].append(t)
                fed[i] += 1
            out = eng.decode(rows, torch.tensor(toks, dtype=torch.int32, device=eng.device))
        eng.check()
        eng.cache.verify_device()
        eng.cache.audit()
        check(out, said)

    decode(1)
    decode(4)
    if prefix == 330:
        assert bool(shared_calls) == (name != "gunirax")                   # (whose attention is of another kind)
    out = eng.step([(a, tails[1][:3]), (base, tails[0][5:6])], "last")     # portions onto sequences that share pages
    said[1] += tails[1][:3]
    said[0] += tails[0][5:6]
    check(out, [said[1], said[0]])
    eng.release(base)                                                      # the source goes, its successors go on
    del rows[0], said[0], fed[0]
    c, = eng.fork([b])
    rows.append(c)
    said.append(list(said[1]))
    fed.append(0)
    decode(3)
    decode(50)                                                             # over the ends of pages and rings
    for s in rows:
        eng.release(s)
    assert eng.cache.tokens_held() == 0 and all(g.pool.n_held == 0 for g in eng.cache.groups)


@pytest.mark.parametrize("name", ["gemma-b", "gemma-d", "fuposun", "linedra"])
@pytest.mark.parametrize("n,max_batch", [(1, 1), (3, 8), (8, 8), (9, 4)])
def test_replies_behind_a_prefix(name, n, max_batch):
    llm = load(name, max_batch=max_batch, max_tokens=max_batch * 448)
    V = llm.model.spec.embedding.vocab_size
    rng = np.random.default_rng(n)
    prefix = rng.integers(1, V, 300).tolist()
    prompts = [rng.integers(1, V, 1 + 3 * i).tolist() for i in range(n)]
    o = GenerationOptions.greedy(12)
    want = llm.generate([prefix + p for p in prompts], o, stop_ids=[])
    for _ in range(2):
        got = llm.generate(prompts, o, stop_ids=[], prefix=prefix)
        for g, w in zip(got, want):
            assert g.tokens == w.tokens and g.prompt_tokens == w.prompt_tokens and g.reused_tokens == 300 and w.reused_tokens == 0
            assert g.finish_reason == w.finish_reason
        assert llm.engine.cache.tokens_held() == 0
    sampled = GenerationOptions(max_new_tokens=6, temperature=0.8, top_k=10, repetition_penalty=1.2, seed=5)
    if n <= max_batch:
        assert [r.tokens for r in llm.generate(prompts, sampled, stop_ids=[], prefix=prefix)] == \
            [r.tokens for r in llm.generate([prefix + p for p in prompts], sampled, stop_ids=[])]


def test_prefix_refusals():
    llm = load("gemma-b", max_batch=1)
    with pytest.raises(PromptError):
        llm.generate([[1], []], prefix=[1, 2])
    with pytest.raises(PromptError):
        llm.generate([[1], [2]], prefix=[1, 2])                            # two batches of one, and the prefix needs a sequence too
    with pytest.raises(PromptError):
        llm.generate([[1]], prefix=list(range(1, 448)))
    with pytest.raises(PromptError):
        llm.generate([[1]], prefix=[1, 10 ** 6])
    assert llm.generate([[1, 2]], GenerationOptions.greedy(2), prefix=[])[0].prompt_tokens == 2
    assert llm.engine.cache.tokens_held() == 0


def plain_beams(llm, prompt, o, stop):
    """The search over whole sequences, their log-probabilities from a prompt step each."""
    take = o.beams * (1 + len(stop))
    norm = lambda lp, n: lp / n ** o.length_penalty  # noqa: E731
    open_, done = [([], 0.0)], []
    for length in range(1, o.max_new_tokens + 1):
        cand = []
        for b, (seq, lp) in enumerate(open_):
            z = llm.evaluate_tokens(list(prompt) + seq).astype(np.float64)
            z = z - z.max()
            z = lp + z - np.log(np.exp(z).sum())
            cand += [(-z[t], b, int(t)) for t in np.argsort(-z, kind="stable")[:take]]
        nxt = []
        for rank, (neg, b, t) in enumerate(sorted(cand)[:take]):
            if len(nxt) == o.beams:
                break
            if t in stop:
                if rank < o.beams:
                    done.append((norm(-neg, length), open_[b][0]))
            else:
                nxt.append((open_[b][0] + [t], -neg))
        done = sorted(done, key=lambda d: -d[0])[:o.beams]
        open_ = nxt
        if len(done) == o.beams and (o.early_stopping or norm(open_[0][1], length) <= done[-1][0]) and length < o.max_new_tokens:
            return done
    return sorted(done + [(norm(lp, o.max_new_tokens), seq) for seq, lp in open_], key=lambda d: -d[0])[:o.beams]


@pytest.mark.parametrize("name", sorted(CONFIGS))
@pytest.mark.parametrize("beams,n,penalty", [(3, 9, 1.0), (4, 6, 0.5)])
def test_beam_search(name, beams, n, penalty):
    llm = load(name, max_batch=9)
    V = llm.model.spec.embedding.vocab_size
    rng = np.random.default_rng(beams)
    prompts = [rng.integers(1, V, k).tolist() for k in (300, 5, 62, 130)]
    o = BeamOptions(beams=beams, max_new_tokens=n, length_penalty=penalty, replies=beams)
    first = llm.evaluate_tokens(prompts[0])
    stop = [int(np.argsort(-first)[1])]                                    # a likely token ends some replies early
    for _ in range(2):                                                     # the second time from captured graphs
        got = llm.beam_search(prompts, o, stop_ids=stop)
        llm.engine.cache.audit()
        assert llm.engine.cache.tokens_held() == 0
    for r, p in zip(got, prompts):
        want = plain_beams(llm, p, o, stop)
        assert [h.tokens for h in r.replies] == [w[1] for w in want]
        assert np.allclose([h.score for h in r.replies], [w[0] for w in want], atol=2e-3)


def test_beam_search_of_the_bfloat16_path(shared_calls):
    llm = load("gemma-d", "bfloat16", max_batch=8)
    prompt = np.random.default_rng(0).integers(1, 1280, 390).tolist()
    got, = llm.beam_search([prompt], BeamOptions(beams=8, max_new_tokens=20, replies=8), stop_ids=[])
    assert shared_calls
    for h in got.replies:
        lp, seq = 0.0, list(prompt)
        for t in h.tokens:
            z = llm.evaluate_tokens(seq).astype(np.float64)
            lp += z[t] - z.max() - np.log(np.exp(z - z.max()).sum())
            seq.append(t)
        assert abs(lp - h.logprob) < 0.5 and len(h.tokens) == 20          # twenty logits, each off by bfloat16's roundings in two paths


def test_one_beam_is_greedy():
    llm = load("gemma-c")
    prompts = [[5, 6, 7], [9] * 80]
    got = llm.beam_search(prompts, BeamOptions(beams=1, max_new_tokens=10), stop_ids=[])
    want = llm.generate(prompts, GenerationOptions.greedy(10), stop_ids=[])
    assert [r.replies[0].tokens for r in got] == [r.tokens for r in want]


def test_beam_refusals():
    llm = load("gemma-b", max_batch=4)
    with pytest.raises(PromptError):
        llm.beam_search([[1]], BeamOptions(beams=5))
    with pytest.raises(OptionsError):
        llm.beam_search([[1]], BeamOptions(beams=0))
    with pytest.raises(PromptError):
        llm.beam_search([[]], BeamOptions(beams=2))
    with pytest.raises(PromptError):
        llm.beam_search([[10 ** 6]], BeamOptions(beams=2))
    assert llm.engine.cache.tokens_held() == 0


def test_a_batch_of_some_that_share_and_some_that_do_not(shared_calls):
    llm = load("gemma-d", "bfloat16")
    eng = llm.engine
    rng = np.random.default_rng(8)
    texts = [rng.integers(1, 1280, n).tolist() for n in (310, 33, 400)]
    slots = [eng.new_sequence() for _ in texts]
    eng.step(list(zip(slots, texts)), [()] * 3)
    f = eng.fork([slots[0], slots[0], slots[2]])
    rows = [slots[0], f[0], f[1], slots[1], slots[2], f[2]]
    said = [list(texts[i]) for i in (0, 0, 0, 1, 2, 2)]
    for step in range(3):
        toks = rng.integers(1, 1280, 6).tolist()
        for s, t in zip(said, toks):
            s.append(t)
        out = eng.decode(rows, torch.tensor(toks, dtype=torch.int32, device=eng.device), pad=True)
    assert shared_calls
    for row, seq in zip(out, said):
        ok, err, tol = close(row.cpu().numpy(), llm.evaluate_tokens(seq), "bfloat16")
        assert ok, (len(seq), err, tol)
