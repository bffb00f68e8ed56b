"""8-bit cache and 4-bit weights without a GPU: what is refused, the options, and the cache's books."""
import pytest
import torch

import helpers
from cajeta_llm_b200.csrc import kernels as K


@pytest.fixture
def anywhere(monkeypatch):
    """Tensors of the host pass for the device's; a call that is not refused would reach the library, which is not there."""
    def need(t, name, dtype=None):
        if not t.is_contiguous():
            raise K.KernelError(f"{name} must be contiguous")
        if dtype is not None and t.dtype != dtype:
            raise K.KernelError(f"{name} must be {dtype}, found {t.dtype}")

    class Reached(Exception):
        pass

    def library(name):
        raise Reached(name)

    monkeypatch.setattr(K, "_need", need)
    monkeypatch.setattr(K, "_on_device", lambda t: True)
    monkeypatch.setattr(K, "_need_same_device", lambda *a: None)
    monkeypatch.setattr(K, "_sm_count", lambda: 148)
    monkeypatch.setattr(K, "library", library)
    monkeypatch.setattr(K, "_stream", lambda: 0)
    return Reached


def cache(kv=2, hd=64, pages=3):
    k, v = (torch.zeros((pages, kv, 16, hd), dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
    return dict(k_plane=k, v_plane=v, k_exp=torch.zeros((pages, kv, 16), dtype=torch.uint8), v_exp=torch.zeros((pages, kv, 16), dtype=torch.uint8))


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def append(**kw):
    a = dict(qkv=torch.zeros(3, 512), q_off=0, k_off=256, v_off=384, q_out=torch.zeros(3, 4, 64, dtype=torch.bfloat16), **cache(), positions=i32(3),
             row_req=i32(3), table=i32(2, 4), page_tokens=16, n_heads=4, n_kv=2, head_dim=64, rotary_dim=64, inv_freq=torch.zeros(32), write_kv=True)
    a.update(kw)
    K.rope_kv_write_e4m3(**a)


def decode(**kw):
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), out=torch.zeros(3, 4, 64, dtype=torch.bfloat16), **cache(), positions=i32(3), row_req=i32(3),
             table=i32(2, 4), page_tokens=16, n_heads=4, n_kv=2, head_dim=64, window=0, scale=1.0, max_context=9)
    a.update(kw)
    K.decode_attention_e4m3(**a)


def prefill(**kw):
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), out=torch.zeros(3, 4, 64, dtype=torch.bfloat16), **cache(), req_start=i32(3), req_prior=i32(2),
             table=i32(2, 4), page_tokens=16, n_heads=4, n_kv=2, head_dim=64, window=0, scale=1.0)
    a.update(kw)
    K.prefill_attention_e4m3(**a)


def product(w=None, **kw):
    w = w if w is not None else K.Q4Weight(torch.zeros(8 * 544 * 2, dtype=torch.uint8), (70, 128), 64)
    a = dict(a=torch.zeros(3, 128, dtype=torch.bfloat16), w=w, out=torch.zeros(3, 70))
    a.update(kw)
    K.gemm_q4(**a)


@pytest.mark.parametrize("call", [append, decode, prefill, product])
def test_the_calls_themselves_are_taken(call, anywhere):
    with pytest.raises(anywhere):
        call()


EXPERTS = K.Q4Weight(torch.zeros(1, dtype=torch.uint8), (4, 70, 128), 64)


@pytest.mark.parametrize("call,kw", [
    (append, dict(qkv=torch.zeros(3, 512, dtype=torch.bfloat16))), (append, dict(qkv=torch.zeros(512, 3).T)), (append, dict(q_off=300)),
    (append, dict(v_off=385)), (append, dict(k_off=-2)), (append, dict(q_out=torch.zeros(2, 4, 64, dtype=torch.bfloat16))),
    (append, dict(q_out=torch.zeros(3, 4, 64))), (append, dict(positions=i32(2))), (append, dict(positions=torch.zeros(3, dtype=torch.int64))),
    (append, dict(row_req=i32(4))), (append, dict(inv_freq=None)), (append, dict(inv_freq=torch.zeros(31))), (append, cache(kv=1)),
    (append, dict(k_plane=torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16))), (append, dict(k_exp=torch.zeros(3, 2, 15, dtype=torch.uint8))),
    (append, dict(table=i32(8))),
    (decode, dict(q=torch.zeros(3, 4, 64))), (decode, dict(out=torch.zeros(2, 4, 64, dtype=torch.bfloat16))), (decode, dict(head_dim=96)),
    (decode, dict(n_heads=3)), (decode, dict(n_kv=3)), (decode, dict(positions=i32(2))), (decode, dict(row_req=i32(2))), (decode, dict(table=i32(8))),
    (decode, dict(page_tokens=8)), (decode, dict(v_exp=torch.zeros(3, 2, 16, dtype=torch.int8))), (decode, dict(splits=-1)), (decode, dict(window=-1)),
    (prefill, dict(req_start=i32(2))), (prefill, dict(table=i32(1, 4))), (prefill, dict(req_prior=torch.zeros(2))), (prefill, dict(window=-5)), (prefill, dict(scale=0.0)),
    (product, dict(w=torch.zeros(70, 128))), (product, dict(a=torch.zeros(3, 128))), (product, dict(a=torch.zeros(128, 3, dtype=torch.bfloat16).T)),
    (product, dict(a=torch.zeros(3, 64, dtype=torch.bfloat16))), (product, dict(a=torch.zeros(4, 128, dtype=torch.bfloat16))),
    (product, dict(out=torch.zeros(3, 71))), (product, dict(out=torch.zeros(3, 70, dtype=torch.float16))),
    (product, dict(out=torch.zeros(3, 70, dtype=torch.bfloat16), accumulate=True)), (product, dict(bias=torch.zeros(71))),
    (product, dict(group_offsets=i32(2))), (product, dict(w=EXPERTS)), (product, dict(w=EXPERTS, group_offsets=i32(4))),
    (product, dict(a_row_index=i32(2))), (product, dict(w_up=EXPERTS))])
def test_refusals(call, kw, anywhere):
    with pytest.raises(K.KernelError):
        call(**kw)


def test_weights_that_are_refused(anywhere, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    good = torch.zeros(8, 64, dtype=torch.int8), torch.ones(8, 1)
    with pytest.raises(anywhere):
        K.Q4Weight.from_codes(*good)
    for codes, scales, group in ((good[0] + 8, good[1], 64), (good[0] - 9, good[1], 64), (good[0], good[1] * 1.03125 * 1.0625, 64),
                                 (good[0], good[1] * float("inf"), 64), (good[0], torch.ones(8, 2), 64), (good[0], good[1], 48), (good[0], good[1], 0),
                                 (good[0][:, :60].contiguous(), good[1], 64), (good[0].short(), good[1], 64), (good[0][0], good[1], 64)):
        with pytest.raises(K.KernelError):
            K.Q4Weight.from_codes(codes, scales, group)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(K.KernelError, match="captured"):
        K.Q4Weight.from_codes(*good)
    with pytest.raises(K.KernelError):
        EXPERTS.first(5)


def test_options_and_models_that_do_not_take_them():
    from cajeta_llm_b200.cli import parse_run
    from cajeta_llm_b200.config import parse_config_dict
    from cajeta_llm_b200.engine.model import build_model
    from cajeta_llm_b200.engine.options import EngineOptions
    from cajeta_llm_b200.parts.base import Runtime
    o, _, _ = parse_run(["--model", "m", "--prompt", "1 2", "--cache-dtype", "float8_e4m3", "--weight-dtype", "int4"])
    o.validate()
    assert (o.cache_dtype, o.weight_dtype) == ("float8_e4m3", "int4")
    for kw in (dict(cache_dtype="int8"), dict(weight_dtype="int8"), dict(cache_dtype="float8_e4m3", dtype="float32"), dict(weight_dtype="int4", dtype="float32")):
        with pytest.raises(ValueError):
            EngineOptions(model="m", **kw).validate()
        with pytest.raises(ValueError):
            Runtime(device="cpu", **kw)
    for kw in (dict(cache_dtype="float8_e4m3"), dict(weight_dtype="int4")):
        build_model(parse_config_dict(helpers.MEDIUM), Runtime("bfloat16", "cpu", **kw))
    odd = dict(helpers.MEDIUM, head_dim=32)
    with pytest.raises(ValueError, match="8-bit cache"):
        build_model(parse_config_dict(odd), Runtime("bfloat16", "cpu", cache_dtype="float8_e4m3"))
    with pytest.raises(ValueError, match="4-bit weights"):
        build_model(parse_config_dict(dict(helpers.MEDIUM, moe_intermediate_size=100, shared_expert_intermediate_size=200)),
                    Runtime("bfloat16", "cpu", weight_dtype="int4"))


def test_the_cache_holds_codes_and_exponents():
    from cajeta_llm_b200.cache.manager import CacheManager
    from cajeta_llm_b200.parts.base import KvNeed
    need = KvNeed(2, 64, 0)
    c = CacheManager([need, need], [None, None], [None, 0], 16, 2, 64, 8, torch.float8_e4m3fn, "cpu")
    assert c.plane(0)[0].dtype == torch.float8_e4m3fn and c.exponents(0)[0].shape == c.plane(0)[0].shape[:3]
    assert c.exponents(1)[1].data_ptr() == c.exponents(0)[1].data_ptr()
    assert c.bytes_per_token() == 2 * 2 * (64 + 1)
    plain = CacheManager([need], [None], [None], 16, 2, 64, 8, torch.bfloat16, "cpu")
    assert plain.exponents(0) == (None, None) and plain.bytes_per_token() == 2 * 2 * 64 * 2


def test_blocks_a_row():
    """Few rows are dealt out to many blocks, many or short ones are not; never to more than a step of 128 keys each."""
    assert K.e4m3_splits(1, 16, 16, 576, 148) > 2
    assert K.e4m3_splits(8, 16, 16, 576, 148) == 1
    assert 20 <= K.e4m3_splits(1, 28, 4, 32768, 148) <= 64
    assert K.e4m3_splits(1, 40, 2, 1, 148) == 1
    for rows, span in ((1, 1), (3, 200), (64, 2048), (1000, 9), (1, 100_000)):
        assert 1 <= K.e4m3_splits(rows, 28, 4, span, 148) <= max(1, -(-span // 128))


def test_which_form_portions_take():
    """Many rows in tiles, few one by one with their keys shared out, a few dozen of one request in tiles."""
    assert K.e4m3_portions(33, 1, 16, 16, 4096, 148) == 0 and K.e4m3_portions(32, 1, 16, 16, 4096, 148) == 0
    assert K.e4m3_portions(2, 1, 28, 4, 4096, 148) == 8 and K.e4m3_portions(8, 1, 28, 4, 4096, 148) == 4
    assert K.e4m3_portions(36, 6, 28, 4, 4096, 148) == 1 and K.e4m3_portions(64, 7, 28, 4, 4096, 148) == 0
    assert K.e4m3_portions(30, 8, 28, 4, 4096, 148) == 1 and K.e4m3_portions(1, 1, 4, 4, 100, 148) == 1
    for rows, requests in ((1, 1), (7, 7), (20, 3), (32, 32)):
        assert 0 <= K.e4m3_portions(rows, requests, 40, 2, 50_000, 148) <= 8


def test_which_form_a_4_bit_product_takes():
    assert not K.q4_on_tcgen05(1, 151_936, 0) and not K.q4_on_tcgen05(8, 151_936, 0) and not K.q4_on_tcgen05(64, 2048, 0)
    assert K.q4_on_tcgen05(64, 6144, 0) and K.q4_on_tcgen05(2048, 512, 0)
    assert not K.q4_on_tcgen05(32, 1408, 60) and K.q4_on_tcgen05(8192, 1408, 60)
    for rows, features, groups, gated in ((2048, 3584, 0, False), (100, 70, 0, True), (8192, 1408, 60, True), (300, 9, 4, False)):
        tok = K.q4_tile_rows(rows, features, groups, gated, 148)
        assert tok % 16 == 0 and 16 <= tok <= 256


def test_what_a_call_hands_over_is_what_the_function_takes():
    """The letters of every entry point's arguments against the declaration in its source."""
    import os
    import re
    from cajeta_llm_b200.csrc import build
    with open(K.__file__) as f:
        calls = set(re.findall(r'_entry\("(\w+)", "(\w+)", "(\w+)"\)', f.read()))
    assert len(calls) >= 6
    for lib, name, signs in calls:
        with open(os.path.join(build.HERE, build.LIBRARIES[lib])) as f:
            declared = re.search(r"CJ_EXPORT int " + name + r"\(([^)]*)\)", f.read()).group(1)
        kinds = "".join("p" if "*" in a or "cudaStream_t" in a else "l" if "long long" in a else "f" if "float" in a else "i" for a in declared.split(","))
        assert kinds == signs, name
