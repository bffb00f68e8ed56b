"""What calls over the 8-bit cache and with 4-bit weights work out on the host, without a GPU."""
from cajeta_llm_b200.csrc import kernels as K


def test_contexts_of_one_length_in_steps_ask_for_the_blocks_of_a_row_once(monkeypatch):
    """A decoded token makes the context one longer: the rule, some 200 us of the host, is worked out once for each step of 128 keys."""
    worked_out, blocks = [], K._e4m3_blocks
    monkeypatch.setattr(K, "_e4m3_blocks", lambda *a: worked_out.append(a) or blocks(*a))
    got = {K.e4m3_splits(5, 30, 3, span, 147) for span in range(20_001, 20_097)}
    assert len(got) == 1 and len(worked_out) == 1
    K.e4m3_splits(5, 30, 3, 20_097, 147)
    assert len(worked_out) == 2


def test_models_that_scale_what_a_sublayer_adds_say_so_before_they_are_loaded():
    """4-bit products do not scale their sums, an 8-bit cache's attention takes positive scales: refused when the model is built, not in its first step."""
    import dataclasses

    import pytest

    import helpers
    from cajeta_llm_b200.config import parse_config_dict
    from cajeta_llm_b200.config.base import get_architecture
    from cajeta_llm_b200.engine.model import Model
    from cajeta_llm_b200.parts.base import Runtime
    from cajeta_llm_b200.parts.plan import PartSpec
    cfg = parse_config_dict(dict(helpers.MEDIUM, mlp_only_layers=[0, 1]))
    plan = get_architecture(cfg.architecture).build_plan(cfg)
    names = {"mixer_norm_name": "a", "feed_forward_norm_name": "b", "mixer_name": "m", "feed_forward_name": "f"}

    def built(block=None, mixer=None, **held):
        layers = [dataclasses.replace(l, block=block or l.block, mixer=mixer or l.mixer, feed_forward=None if block else l.feed_forward) for l in plan.layers]
        return Model(dataclasses.replace(plan, layers=layers), Runtime("bfloat16", "cpu", **held))

    assert all(b.mixer.takes_q4_weights for b in built(PartSpec("parallel", names), weight_dtype="int4").blocks)
    scaled = PartSpec("parallel", dict(names, residual_mult=0.5))
    built(scaled), built(scaled, cache_dtype="float8_e4m3")
    with pytest.raises(ValueError, match="4-bit weights"):
        built(scaled, weight_dtype="int4")
    upside_down = PartSpec("attention", dict(plan.layers[0].mixer.params, scale=-0.1))
    built(mixer=upside_down), built(mixer=upside_down, weight_dtype="int4")
    with pytest.raises(ValueError, match="8-bit cache"):
        built(mixer=upside_down, cache_dtype="float8_e4m3")
