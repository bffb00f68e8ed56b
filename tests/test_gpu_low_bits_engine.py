"""Models served with an 8-bit cache and 4-bit weights: through the step function and the entry point."""
import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def runner_for(model_dir, **kw):
    from cajeta_llm_b200.engine.model import load_model
    from cajeta_llm_b200.engine.step import ModelRunner
    from cajeta_llm_b200.parts.base import Runtime
    model, _ = load_model(model_dir, Runtime("bfloat16", device=DEV, **{k: kw.pop(k) for k in ("cache_dtype", "weight_dtype") if k in kw}))
    return ModelRunner(model, page_tokens=16, max_seqs=4, max_tokens_per_seq=512, **kw)


def logits_of(runner, toks, portions):
    from cajeta_llm_b200.engine.step import StepEntry
    s, at, out = runner.admit(), 0, []
    for n in portions:
        out.append(runner.step([StepEntry(s, toks[at:at + n], list(range(n)))]).clone())
        at += n
    runner.release(s)
    runner.check_waits()
    return torch.cat(out)


def apart(a, b):
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("name", ["M", "W"])
def test_an_8_bit_cache_serves_portions_and_single_tokens_alike(name, model_dirs):
    """What is cached does not depend on how a prompt is cut; what is left is the bfloat16 path's own rounding (steps of other kernels)
    and, against the bfloat16 cache, e4m3's (2^-4 of an entry, averaged over heads and keys)."""
    toks = helpers.random_tokens(helpers.CONFIGS[name]["vocab_size"], 300, seed=4)
    e4m3, full = runner_for(model_dirs[name], cache_dtype="float8_e4m3"), runner_for(model_dirs[name])
    whole = logits_of(e4m3, toks, [300])
    assert apart(logits_of(e4m3, toks, [255] + [1] * 45), whole) < 0.05
    assert apart(logits_of(e4m3, toks, [2, 129, 1, 168]), whole) < 0.05
    assert apart(whole, logits_of(full, toks, [300])) < 0.2
    assert e4m3.cache.bytes_per_token() * 2 * 64 <= full.cache.bytes_per_token() * 65


def test_steps_from_graphs_have_the_same_bits(model_dirs):
    toks = helpers.random_tokens(helpers.CONFIGS["M"]["vocab_size"], 60, seed=5)
    both = dict(cache_dtype="float8_e4m3", weight_dtype="int4")
    plain, captured = runner_for(model_dirs["M"], cuda_graphs=False, **both), runner_for(model_dirs["M"], **both)
    portions = [20, 1, 1, 1, 17, 17, 1, 1, 1]
    want = logits_of(plain, toks, portions)
    for _ in range(3):
        assert apart(logits_of(captured, toks, portions), want) < 1e-6
    assert captured.graph_replays > 0


@pytest.mark.parametrize("name", ["M", "W"])
def test_4_bit_weights_are_the_quantised_ones(name, model_dirs):
    """The bfloat16 engine with the quantised weights in its matrices' place gives the same logits, up to the order of sums."""
    from cajeta_llm_b200.csrc import kernels as K
    q4, full = runner_for(model_dirs[name], weight_dtype="int4"), runner_for(model_dirs[name])

    def rounded(w):
        codes, scales = K.Q4Weight.codes_of(w.contiguous())
        w.copy_(codes.float() * scales.repeat_interleave(64, dim=-1)[..., :w.shape[-1]])

    for block in full.model.blocks:
        ff = block.feed_forward
        for w in [block.mixer.w_qkv, block.mixer.w_o, ff.w_gate, ff.w_up, ff.w_down] + [getattr(ff, n, None) for n in ("ws_gate", "ws_up", "ws_down")]:
            if w is not None:
                rounded(w)
        if getattr(ff, "shared_chunks", 0) and ff.ws_down is not None:
            # (one matrix whose groups are the chunks' groups)
            C, I = ff.shared_chunks, ff.inter
            ff.ws_down.view(-1, C, I).copy_(ff.w_down[ff.num_experts:].permute(1, 0, 2))
    toks = helpers.random_tokens(helpers.CONFIGS[name]["vocab_size"], 150, seed=6)
    for portions in ([150], [120] + [1] * 30):
        assert apart(logits_of(q4, toks, portions), logits_of(full, toks, portions)) < 0.05
    assert q4.model.weight_bytes() < full.model.weight_bytes()


def test_generation_with_both_through_the_entry_point(model_dirs):
    from cajeta_llm_b200.engine.llm_engine import LlmEngine
    from cajeta_llm_b200.engine.options import EngineOptions
    from cajeta_llm_b200.sampling.params import SamplingParams
    prompts = [helpers.random_tokens(1000, n, seed=n) for n in (3, 40, 17, 90, 1, 60)]
    got = []
    for kw in (dict(), dict(num_blocks=24), dict(chunk=16)):
        engine = LlmEngine.load(EngineOptions(model=model_dirs["M"], dtype="bfloat16", ctx=128, max_seqs=4, cache_dtype="float8_e4m3",
                                              weight_dtype="int4", **kw))
        got.append(engine.generate(prompts, SamplingParams(max_new_tokens=8, stop_token_ids=())))
        engine.runner.check_waits()
        engine.close()
    assert all(len(t) == 8 for run in got for t in run)
    same = sum(a == b for run in got[1:] for x, y in zip(run, got[0]) for a, b in zip(x, y))
    assert same >= 0.7 * 2 * 8 * len(prompts)              # scarce pages and short portions: near ties aside, the same tokens
