"""Sequences of ragged lengths over a paged cache (models/qwen.py) and drawn tokens in the decode loops."""
import json

import pytest
import torch

from tyr_b200.cli import model_runner as R
from tyr_b200.io import safetensors as st
from tyr_b200.models import qwen as Q
from tyr_b200.models.generation import SamplingStrategy, sample_from_logits
from tyr_b200.ops import sampling


def tiny(**kw):
    return Q.QwenConfig(**{**dict(vocab_size=64, hidden_size=32, intermediate_size=64, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, half_head_dim=4,
                                  eos_token_ids=(1,)), **kw})


PROMPTS = [[5, 9, 33, 2, 17], [40], [7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19]]


def test_paged_generation_is_the_uncached_one():
    lm = Q.Qwen3ForCausalLM.init(tiny())
    new = Q.generate_paged(lm, PROMPTS, 9, eos_token_ids=(), page=4, cache=torch.float32)
    for p, row in zip(PROMPTS, new):
        assert torch.tensor(p + row).equal(Q.generate_greedy_uncached(lm, torch.tensor([p]), 9, eos_token_ids=())[0])


def test_pieces_of_prompts_pages_given_back_and_places_taken_again():
    lm = Q.Qwen3ForCausalLM.init(tiny())
    s = Q.PagedQwen3Session(lm, 3, 24, page=4, pages=9, cache=torch.float32)
    whole = [lm.forward(torch.tensor([p]))[0, -1] for p in PROMPTS]
    s.extend([PROMPTS[0][:3], [], PROMPTS[2][:6]])
    last = s.extend([PROMPTS[0][3:], PROMPTS[1], PROMPTS[2][6:]])
    assert torch.allclose(last, torch.stack(whole), atol=1e-4) and s.held == [5, 1, 13] and len(s.free) == 9 - 2 - 1 - 4
    out = s.step(torch.tensor([3, 4, 6]))
    for b, t in enumerate((3, 4, 6)):
        assert torch.allclose(out[b], lm.forward(torch.tensor([PROMPTS[b] + [t]]))[0, -1], atol=1e-4)
    s.release(2)
    assert s.held == [6, 2, 0] and len(s.free) == 6
    out = s.step(torch.tensor([3, 4, 6]))
    assert s.held == [7, 3, 0] and torch.allclose(out[0], lm.forward(torch.tensor([PROMPTS[0] + [3, 3]]))[0, -1], atol=1e-4)
    logits = s.extend([[], [], [20, 21]])
    assert not logits[:2].any() and torch.allclose(logits[2], lm.forward(torch.tensor([[20, 21]]))[0, -1], atol=1e-4)
    for call in (lambda: s.extend([[1] * 20, [], []]), lambda: s.extend([[1] * 17, [1] * 10, []]), lambda: s.extend([[1]]), lambda: s.extend([[], [], []]),
                 lambda: Q.PagedQwen3Session(lm, 0, 4), lambda: Q.generate_paged(lm, [[1], []])):
        before = (s.held, list(s.free))
        with pytest.raises(ValueError):
            call()
        assert before == (s.held, s.free)


def test_finished_sequences_stop():
    lm = Q.Qwen3ForCausalLM.init(tiny())
    free = Q.generate_paged(lm, PROMPTS, 12, eos_token_ids=(), page=4, cache=torch.float32)
    eos = free[1][2]
    stopped = Q.generate_paged(lm, PROMPTS, 12, eos_token_ids=(eos,), page=4, cache=torch.float32)
    for a, b in zip(free, stopped):
        cut = next((i + 1 for i, t in enumerate(a) if t == eos), len(a))
        assert b == a[:cut]


def test_drawn_strategy_takes_its_numbers_from_the_generator():
    logits = torch.randn(5, 300)
    strategy = SamplingStrategy.drawn(0.8, 20, 0.9, 0.05)
    got = sample_from_logits(logits, strategy, torch.Generator().manual_seed(4))
    want = sampling.sample(logits, torch.rand(5, generator=torch.Generator().manual_seed(4)), temperature=0.8, top_k=20, top_p=0.9, min_p=0.05)
    assert torch.equal(got, want)
    lm = Q.Qwen3ForCausalLM.init(tiny())
    a = Q.generate(lm, torch.tensor([[3, 4]]), 5, SamplingStrategy.drawn(top_k=1), eos_token_ids=())
    assert torch.equal(a, Q.generate_greedy(lm, torch.tensor([[3, 4]]), 5, eos_token_ids=()))


def test_command_line_with_a_paged_cache(tmp_path, capsys, monkeypatch):
    lm = Q.Qwen3ForCausalLM.init(tiny(vocab_size=300), tie_word_embeddings=False)
    st.save_file({k: v.contiguous() for k, v in Q.state_dict(lm).items()}, str(tmp_path / "model.safetensors"))
    json.dump({"model_type": "qwen3", "vocab_size": 300, "hidden_size": 32, "intermediate_size": 64, "num_hidden_layers": 3, "num_attention_heads": 4, "num_key_value_heads": 2,
               "head_dim": 8, "rope_theta": 10000.0}, open(tmp_path / "config.json", "w"))

    class Bytes:
        def encode(self, s): return list(s.encode())
        def decode(self, ids, skip_special=True): return " ".join(map(str, ids))
        def token_id(self, s): return None
    monkeypatch.setattr(R.tok_hf, "load_qwen3", lambda d: Bytes())
    (tmp_path / "p.txt").write_text("one\na longer prompt\n")
    args = ["--family", "qwen3", "--source", str(tmp_path), "--prompt-file", str(tmp_path / "p.txt"), "--device", "cpu", "--max-new-tokens", "4", "--batch-size", "2"]
    assert R.main([*args, "--cache", "paged", "--bench"]) == 0
    paged = capsys.readouterr().out
    assert R.main([*args[:-2], "--batch-size", "1"]) == 0
    assert paged.split("BENCH")[0] == capsys.readouterr().out
    assert R.main([*args, "--cache", "paged8", "--temperature", "0.9", "--min-p", "0.1", "--top-k", "40"]) == 0
    assert capsys.readouterr().out.count("\n") == 4
    with pytest.raises(ValueError, match="no paged cache"):
        R.load_text_family("qwen35", str(tmp_path), "cpu", torch.float32, "paged")


@pytest.mark.gpu
@pytest.mark.parametrize("cache", (torch.bfloat16, torch.float8_e4m3fn))
def test_gpu_graph_steps_match_eager_ones(monkeypatch, cache):
    cfg = tiny(vocab_size=500, hidden_size=256, intermediate_size=512, num_attention_heads=6, half_head_dim=64)
    lm = Q.Qwen3ForCausalLM.init(cfg, device="cuda", dtype=torch.bfloat16, seed=3)
    prompts = [[i * 7 % 500 for i in range(n)] for n in (37, 1, 130, 64)]
    toks = torch.randint(0, 500, (70, 4), device="cuda")
    runs = []
    for graph in ("1", "0"):
        monkeypatch.setenv("TYR_DECODE_GRAPH", graph)
        s = Q.PagedQwen3Session(lm, 4, 256, page=32, cache=cache)
        outs = [s.extend(prompts)]
        for i, t in enumerate(toks):
            if i == 40:
                s.release(1)
                outs.append(s.extend([[], [9, 8, 7], [], []]))
            outs.append(s.step(t).clone())
        assert (s._graph is not None) == (graph == "1")
        runs.append(outs)
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    # 16-bit pages: the session over dense stores, prompt by prompt
    if cache == torch.bfloat16:
        dense = Q.Qwen3Session(lm, 1, 256)
        ref = [dense.prefill(torch.tensor([prompts[2]], device="cuda"))] + [dense.step(t[2:3]) for t in toks[:20]]
        for a, b in zip(runs[0], ref):
            assert (a[2].float() - b[0].float()).abs().max() < 0.06 * max(1.0, b.float().abs().max().item())


@pytest.mark.gpu
def test_gpu_generation_in_8_bits_with_drawn_tokens():
    cfg = tiny(vocab_size=500, hidden_size=256, intermediate_size=512, num_attention_heads=6, half_head_dim=64, eos_token_ids=())
    lm = Q.Qwen3ForCausalLM.init(cfg, device="cuda", dtype=torch.bfloat16, seed=3)
    prompts = [[i * 7 % 500 for i in range(n)] for n in (37, 1, 130)]
    draw = lambda: Q.generate_paged(lm, prompts, 30, SamplingStrategy.drawn(0.8, 50, 0.95), generator=torch.Generator("cuda").manual_seed(5))
    a, b = draw(), draw()
    assert a == b and all(len(r) == 30 for r in a)


def test_drawn_rows_with_nothing_to_choose_from():
    """Such a row's token goes into an embedding all the same: it is an index, the one that the greedy choice gives."""
    logits = torch.full((3, 40), -float("inf"))
    logits[1] = float("nan")
    logits[2, 7] = 0.0
    assert sample_from_logits(logits, SamplingStrategy.drawn(0.8, 20, 0.9)).tolist() == [0, 0, 7]


def test_a_step_takes_a_token_for_every_sequence():
    """Fewer or more are refused before anything is counted (a captured step would hand one token to all)."""
    lm = Q.Qwen3ForCausalLM.init(tiny())
    s = Q.PagedQwen3Session(lm, 3, 24, page=4, cache=torch.float32)
    s.extend(PROMPTS)
    before = (list(s.held), list(s.free), s.lengths.tolist())
    for n in (1, 2, 4):
        with pytest.raises(ValueError):
            s.step(torch.zeros(n, dtype=torch.long))
        assert before == (s.held, s.free, s.lengths.tolist())
    out = s.step(torch.tensor([[3], [4], [6]]))
    assert torch.allclose(out[1], lm.forward(torch.tensor([PROMPTS[1] + [4]]))[0, -1], atol=1e-4)


@pytest.mark.gpu
def test_a_captured_step_refuses_other_numbers_of_tokens():
    cfg = tiny(vocab_size=500, hidden_size=256, intermediate_size=512, num_attention_heads=6, half_head_dim=64)
    s = Q.PagedQwen3Session(Q.Qwen3ForCausalLM.init(cfg, device="cuda", dtype=torch.bfloat16, seed=3), 3, 128, page=32)
    s.extend([[1, 2, 3], [4], [5, 6]])
    s.step(torch.tensor([7, 8, 9], device="cuda"))
    with pytest.raises(ValueError):
        s.step(torch.tensor([7], device="cuda"))
    assert s.held == [4, 2, 3] and s.lengths.tolist() == s.held


@pytest.mark.gpu
def test_gpu_draws_from_models_in_64_bits():
    logits = torch.randn(4, 300, dtype=torch.float64, generator=torch.Generator().manual_seed(1)).cuda()
    strategy, gen = SamplingStrategy.drawn(0.8, 20, 0.9, 0.05), torch.Generator("cuda")
    got = sample_from_logits(logits, strategy, gen.manual_seed(4))
    assert torch.equal(got, sample_from_logits(logits.float(), strategy, gen.manual_seed(4)))
