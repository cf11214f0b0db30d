"""LLaMA over the paged cache against HF, the static-cache path and plain statements of beam search and eviction (GPU).

Tolerances as in ``test_gpu_model.py``: fp32 logits 1e-4 of their largest magnitude with identical greedy ids, bf16 2e-2.
"""

from __future__ import annotations

import numpy as np
import pytest

from helpers import hf_greedy, tiny_golden, tiny_gqa_hf_model, tiny_hf_model, tiny_program, tiny_weights
from oracle import paged as ref

pytestmark = pytest.mark.gpu


def _runner(model, prog=None):
    from backend.hal_cuda import CudaBackend, CudaBackendConfig
    from graph.llama import ModelConfig
    from runtime.program import compile_llama, load_weights
    from runtime.session import LlamaRunner

    if prog is None:
        prog = compile_llama(ModelConfig.from_hf(model.config, max_seq=48, dtype="float32"), 1, batch=1, prompt_len=16)
    runner = LlamaRunner(prog, CudaBackend(CudaBackendConfig(1, prog.arena_bytes)))
    load_weights(prog, runner.hal, tiny_weights(prog, model))
    return runner


@pytest.mark.parametrize("page_size", [8, 16, 64])
def test_greedy_matches_hf(page_size):
    from runtime.paged import PagedLlama

    model, gold = tiny_hf_model(), tiny_golden()
    gen = PagedLlama(_runner(model), rows=1, max_slots=40, page_size=page_size)
    logits = []
    out = gen.greedy(gold["prompt"][None], 8, keep_logits=logits)
    assert out[0].tolist() == gold["tokens"].tolist()
    for got, want in zip(logits, gold["step_logits"]):
        assert np.abs(got[0] - want).max() <= 1e-4 * np.abs(want).max()
    assert gen.greedy(gold["prompt"][None], 8).tolist() == out.tolist()  # pages given back and taken again


@pytest.mark.parametrize("rows", [3, 11])
def test_rows_of_a_batch_are_independent_with_shared_kv_heads(rows):
    """Eleven rows run the projections as a row batch, three as GEMVs; each row as HF decodes it alone."""
    from runtime.paged import PagedLlama

    model = tiny_gqa_hf_model()
    rng = np.random.default_rng(rows)
    prompts = rng.integers(0, 1024, (rows, 16))
    got = PagedLlama(_runner(model), rows=rows, max_slots=32, page_size=8).greedy(prompts, 6)
    for row in range(rows):
        want, logits = hf_greedy(model, prompts[row][None], 5)
        assert got[row].tolist() == want, row


def _plain_beams(model, prompt, w, steps, eos, pad):
    """Beam search by whole forward passes of the HF model, fp64 scores."""
    import torch

    beams = [(0.0, [], False)]
    for _ in range(steps):
        cand = []
        for j, (score, toks, done) in enumerate(beams):
            if done:
                cand.append((-score, j, pad))
                continue
            with torch.no_grad():
                x = model(torch.tensor([list(prompt) + toks])).logits[0, -1].double()
            lp = torch.log_softmax(x, -1)
            for t in torch.topk(lp, w).indices.tolist():
                cand.append((-(score + float(lp[t])), j, t))
        cand = sorted(cand)[:w]
        beams = [(-s, beams[j][1] + [t], beams[j][2] or t == eos) for s, j, t in cand]
    return beams


@pytest.mark.parametrize("w,steps", [(4, 9), (6, 3), (2, 17)])
def test_beam_search_matches_whole_forward_passes(w, steps):
    """Page boundaries inside the prompt's last page and behind it; `eos` is a token that the plain search meets."""
    from runtime.paged import PagedLlama

    model = tiny_gqa_hf_model()
    prompt = np.random.default_rng(w).integers(0, 1024, 16)
    runner = _runner(model)
    gen = PagedLlama(runner, rows=w, max_slots=40, page_size=8)
    free = _plain_beams(model, prompt, w, steps, -1, 0)
    for eos in (-1, free[0][1][min(2, steps - 1)]):
        want = _plain_beams(model, prompt, w, steps, eos, 7)
        got = gen.beam_search(prompt, steps, eos=eos, pad=7)
        assert got.tokens.tolist() == [t for _, t, _ in want]
        assert got.done.tolist() == [d for _, _, d in want]
        # fp32 logits within 1e-4 of their largest magnitude (about 1 here), summed over the steps
        assert np.abs(got.scores - [s for s, _, _ in want]).max() <= 2e-4 * steps
    assert gen.cache.allocator.free < gen.spec.num_pages
    gen.reset()
    assert gen.cache.allocator.free == gen.spec.num_pages


def _plain_decode(sd, cfg, prompt, steps, budget, recent, sink):
    """Greedy decoding in fp64 NumPy with a cache that each head cuts to `budget` by accumulated weight."""
    hd, hq, hkv = cfg.head_dim, cfg.num_heads, cfg.num_kv_heads
    inv = 1.0 / cfg.rope_theta ** (np.arange(0, hd, 2) / hd)
    w = {k: v.astype(np.float64) for k, v in sd.items()}
    cache = [[dict(k=[], v=[], w=[], p=[]) for _ in range(hkv)] for _ in range(cfg.num_layers)]

    def norm(x, name):
        return x / np.sqrt((x * x).mean() + cfg.rms_eps) * w[name]

    def rope(x, pos):
        c, s = np.cos(pos * inv), np.sin(pos * inv)
        a, b = x[:, :hd // 2], x[:, hd // 2:]
        return np.concatenate([a * c - b * s, b * c + a * s], 1)

    def forward(token, pos, track):
        x = w["model.embed_tokens.weight"][token]
        for l in range(cfg.num_layers):
            p = f"model.layers.{l}."
            h = norm(x, p + "input_layernorm.weight")
            q, k, v = (w[p + f"self_attn.{n}_proj.weight"] @ h for n in "qkv")
            q, k, v = rope(q.reshape(hq, hd), pos), rope(k.reshape(hkv, hd), pos), v.reshape(hkv, hd)
            out = np.zeros((hq, hd))
            for g in range(hkv):
                c = cache[l][g]
                for name, val in (("k", k[g]), ("v", v[g]), ("w", 0.0), ("p", pos)):
                    c[name].append(val)
                keys, vals = np.array(c["k"]), np.array(c["v"])
                for i in range(g * hq // hkv, (g + 1) * hq // hkv):
                    s = keys @ q[i] / np.sqrt(hd)
                    e = np.exp(s - s.max())
                    e /= e.sum()
                    out[i] = e @ vals
                    if track:
                        c["w"] = list(np.array(c["w"]) + e)
                if track:
                    n = len(c["p"])
                    src = ref.evict(n, pos + 1, np.array(c["w"]), np.array(c["p"]), budget, recent, sink)
                    for name in c:
                        c[name] = [c[name][j] for j in src[:min(n, budget)]]
            x = x + w[p + "self_attn.o_proj.weight"] @ out.reshape(-1)
            h = norm(x, p + "post_attention_layernorm.weight")
            a, b = w[p + "mlp.gate_proj.weight"] @ h, w[p + "mlp.up_proj.weight"] @ h
            x = x + w[p + "mlp.down_proj.weight"] @ (a / (1 + np.exp(-a)) * b)
        return w["lm_head.weight"] @ norm(x, "model.norm.weight")

    for i, t in enumerate(prompt):
        logits = forward(t, i, False)
    got, all_logits = [], []
    for i in range(steps):
        got.append(int(logits.argmax()))
        all_logits.append(logits)
        if i + 1 < steps:
            logits = forward(got[-1], len(prompt) + i, True)
    return got, all_logits, cache


@pytest.mark.parametrize("budget,recent,sink", [(64, 8, 2), (20, 5, 2), (16, 4, 1), (9, 3, 0)])
def test_bounded_cache_decodes_as_the_plain_statement(budget, recent, sink):
    """A budget that is never met, one met after some steps, one token over at each step, and a prompt cut down."""
    from runtime.paged import PagedLlama
    from runtime.program import hf_state_dict

    model = tiny_gqa_hf_model()
    runner = _runner(model)
    prompt = np.random.default_rng(budget).integers(0, 1024, 16)
    steps = 14
    gen = PagedLlama(runner, rows=2, max_slots=72, page_size=8, budget=budget, recent=recent, sink=sink)
    logits = []
    got = gen.greedy(np.stack([prompt, prompt]), steps, keep_logits=logits)
    want, want_logits, cache = _plain_decode(hf_state_dict(model, "float32"), runner.prog.cfg, prompt, steps, budget, recent,
                                             sink)
    assert got.tolist() == [want, want]
    for a, b in zip(logits, want_logits):
        assert np.abs(a[0] - b).max() <= 1e-4 * np.abs(b).max() and np.array_equal(a[0], a[1])
    n = min(16 + steps - 1, budget)
    assert gen.lengths.tolist() == [n, n]
    for l, heads in enumerate(cache):
        for h, c in enumerate(heads):
            assert gen.cache.slot_positions[l, 0, h, :n].tolist() == c["p"], (l, h)
            w = gen.cache.weights[l, 0, h, :n].cpu().numpy()
            assert np.abs(w - np.array(c["w"])).max() <= 1e-4 * max(1.0, np.abs(c["w"]).max())
    if budget < 16:
        assert sum(len(x) for x in gen.cache.held) == 2 * -(-budget // 8)  # pages behind the budget were given back


def test_bf16_step_matches_the_static_cache():
    """Two layers of the 7B shape: the paged step's logits against the decode plan's, fed the same tokens."""
    from backend.hal_cuda import CudaBackend, CudaBackendConfig
    from graph.llama import ModelConfig
    from runtime.executor import execute_plan, read_logits
    from runtime.paged import PagedLlama
    from runtime.program import compile_llama
    from runtime.session import LlamaRunner

    cfg = ModelConfig.llama2_7b(max_seq=128, num_layers=2)
    prog = compile_llama(cfg, 1, batch=1, prompt_len=64)
    runner = LlamaRunner(prog, CudaBackend(CudaBackendConfig(1, prog.arena_bytes)))
    runner.load_random_weights(3)
    prompt = np.random.default_rng(0).integers(0, cfg.vocab_size, (1, 64))
    gen = PagedLlama(runner, rows=2, max_slots=100)
    logits = []
    tokens = gen.greedy(np.repeat(prompt, 2, 0), 5, keep_logits=logits)
    runner.prefill(prompt)
    for i in range(4):
        execute_plan(prog.plans["decode"], runner.hal, tokens=tokens[:1, i:i + 1], pos=np.full(1, 64 + i, np.int32))
        want = np.asarray(read_logits(prog.plans["decode"], runner.hal), np.float32).reshape(-1)
        for row in (0, 1):
            assert np.abs(logits[i + 1][row] - want).max() <= 2e-2 * np.abs(want).max()


def test_refusals():
    from runtime.paged import PagedLlama

    model = tiny_hf_model()
    runner = _runner(model)
    with pytest.raises(ValueError, match="leaves no room"):
        PagedLlama(runner, rows=1, max_slots=16)
    with pytest.raises(ValueError, match="recent"):
        PagedLlama(runner, rows=1, max_slots=40, budget=8, recent=6, sink=4)
    gen = PagedLlama(runner, rows=2, max_slots=20, page_size=8, budget=18, recent=1)
    with pytest.raises(ValueError, match="shares pages"):
        gen.beam_search(np.zeros(16, np.int32), 2)
    with pytest.raises(ValueError, match="expected prompts"):
        gen.greedy(np.zeros((1, 16), np.int32), 2)
    gen = PagedLlama(runner, rows=1, max_slots=20, page_size=8)
    with pytest.raises(ValueError, match="no room"):
        gen.greedy(np.zeros((1, 16), np.int32), 12)
    with pytest.raises(ValueError, match="one rank"):
        PagedLlama(type("R", (), {"prog": tiny_program(2), "hal": None})(), rows=1, max_slots=40)


def test_a_step_behind_a_search_stays_within_its_pages():
    """The pages that a search took are all that its beams have: a further step is refused, not written elsewhere."""
    from runtime.paged import PagedLlama

    gen = PagedLlama(_runner(tiny_hf_model()), rows=2, max_slots=40, page_size=8)
    prompt = np.arange(16, dtype=np.int32)
    with pytest.raises(ValueError, match="steps must be positive"):
        gen.greedy(np.stack([prompt, prompt]), 0)
    with pytest.raises(ValueError, match="steps must be positive"):
        gen.beam_search(prompt, 0)
    first = gen.beam_search(prompt, 9)  # 24 slots, the third page full
    with pytest.raises(ValueError, match="all are in use"):
        gen.step()
    again = gen.beam_search(prompt, 9)
    assert again.tokens.tolist() == first.tokens.tolist() and again.scores.tolist() == first.scores.tolist()


def test_beam_search_needs_the_prompts_pages_once_and_a_tail_for_each_beam():
    """Ten pages are enough for eight beams over two pages of prompt and one of new tokens; nine are refused."""
    from runtime.paged import PagedLlama

    runner = _runner(tiny_gqa_hf_model())
    prompt = np.random.default_rng(3).integers(0, 1024, 16)
    want = PagedLlama(runner, rows=8, max_slots=40, page_size=8).beam_search(prompt, 9)
    gen = PagedLlama(runner, rows=8, max_slots=40, page_size=8, num_pages=10)
    for _ in range(2):
        got = gen.beam_search(prompt, 9)
        assert got.tokens.tolist() == want.tokens.tolist() and got.scores.tolist() == want.scores.tolist()
    small = PagedLlama(runner, rows=8, max_slots=40, page_size=8, num_pages=9)
    with pytest.raises(MemoryError):
        small.beam_search(prompt, 9)
    small.reset()
    assert small.cache.allocator.free == 9


def test_an_error_is_reported_once_and_the_next_run_is_judged_by_itself():
    """A token id outside the vocabulary, and lengths that every layer's operators find bad."""
    from runtime.paged import PagedLlama

    gold = tiny_golden()
    gen = PagedLlama(_runner(tiny_hf_model()), rows=1, max_slots=40, page_size=8)
    prompt = gold["prompt"][None]
    for spoil, said in ((lambda: gen.ids.fill_(10**6), "vocabulary"), (lambda: gen.lengths.fill_(-7), "pim_paged_append")):
        gen._start(prompt)
        gen.ids.fill_(1)
        spoil()
        gen.step()
        with pytest.raises(ValueError, match=said):
            gen.check()
        gen.check()
        assert gen.greedy(prompt, 8)[0].tolist() == gold["tokens"].tolist()
        gen._start(prompt)
        gen.ids.fill_(1)
        spoil()
        gen.step()
        assert gen.greedy(prompt, 8)[0].tolist() == gold["tokens"].tolist()  # (a new start: what was before is not its error)


def test_prompts_are_taken_in_by_operators_that_are_bound_once(monkeypatch):
    """A later start binds nothing and waits for nothing of its own; a bad page met on the way in is reported by ``check``."""
    import runtime.paged as module

    gold = tiny_golden()
    bound = []
    monkeypatch.setattr(module, "PagedAppend", lambda *a, _make=module.PagedAppend, **kw: bound.append(1) or _make(*a, **kw))
    gen = module.PagedLlama(_runner(tiny_hf_model()), rows=2, max_slots=40, page_size=8)
    layers = gen.cfg.num_layers
    prompts = np.stack([gold["prompt"]] * 2)
    for _ in range(3):
        assert gen.greedy(prompts, 8)[1].tolist() == gold["tokens"].tolist()
        assert len(bound) == 3 * layers  # a step's, and one for each row
    gen._start(prompts)
    gen.cache.table.fill_(10**6)
    gen._import(1)
    with pytest.raises(ValueError, match="pim_paged_append"):
        gen.check()
    assert gen.greedy(prompts, 8)[0].tolist() == gold["tokens"].tolist()


def test_a_search_that_finds_no_pages_leaves_the_rows_empty():
    """Beams that hold the prompt's pages but have no tail would write their next token into them."""
    from runtime.paged import PagedLlama

    gold = tiny_golden()
    gen = PagedLlama(_runner(tiny_hf_model()), rows=2, max_slots=40, page_size=8, num_pages=6)
    with pytest.raises(MemoryError):
        gen.beam_search(gold["prompt"], 25)
    assert gen.cache.allocator.free == 6 and not gen.slots.any() and not any(gen.cache.held)
    assert gen.greedy(np.stack([gold["prompt"]] * 2), 8)[0].tolist() == gold["tokens"].tolist()
