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
