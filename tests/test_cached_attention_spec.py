"""CPU tests of the cached attention operators' specs: bindings, refusals, round trip."""
import json

import pytest

import jade_compute_b200 as jc
from jade_compute_b200.runtime import JadeError

ROPE = {"op": "qk_norm_rope", "batch": 2, "seq": 3, "heads": 8, "kv_heads": 2, "dim": 64, "epsilon": 1e-6, "dtype": "bf16"}
GRAD = {**ROPE, "op": "qk_norm_rope_grad"}
TREE = {"op": "attention_tree", "batch": 2, "seq": 33, "heads": 8, "kv_heads": 2, "dim": 64, "capacity": 100, "dtype": "bf16"}
EVICT = {"op": "cache_evict", "batch": 2, "kv_heads": 2, "dim": 64, "capacity": 100, "keep": 10, "recent": 3, "dtype": "fp16"}
COMMIT = {"op": "cache_commit", "batch": 2, "kv_heads": 2, "dim": 64, "capacity": 100, "seq": 9, "dtype": "fp32"}


def names(spec):
    return [(b["name"], b["elements"], b["write"], b["dtype"]) for b in jc.spec_bindings(spec)]


def test_bindings():
    assert names(ROPE) == [("qkv", 2 * 3 * 12 * 64, False, "bf16"), ("q_weight", 64, False, "bf16"), ("k_weight", 64, False, "bf16"),
                           ("positions", 6, False, "i32"), ("q", 2 * 8 * 3 * 64, True, "bf16"), ("k", 2 * 2 * 3 * 64, True, "bf16"),
                           ("v", 2 * 2 * 3 * 64, True, "bf16")]
    cached = names({**ROPE, "capacity": 50, "norm": False})
    assert [n for n, *_ in cached] == ["qkv", "positions", "starts", "q", "k", "v"]
    assert cached[2] == ("starts", 2, False, "i32") and cached[4] == ("k", 2 * 2 * 50 * 64, True, "bf16")
    assert names(GRAD)[4:] == [("dq", 2 * 8 * 3 * 64, False, "bf16"), ("dk", 2 * 2 * 3 * 64, False, "bf16"), ("dv", 2 * 2 * 3 * 64, False, "bf16"),
                               ("dqkv", 2 * 3 * 12 * 64, True, "bf16"), ("dq_weight", 64, True, "fp32"), ("dk_weight", 64, True, "fp32")]
    assert names({**TREE, "weights": True}) == [
        ("q", 2 * 8 * 33 * 64, False, "bf16"), ("k", 2 * 2 * 100 * 64, False, "bf16"), ("v", 2 * 2 * 100 * 64, False, "bf16"),
        ("lengths", 2, False, "i32"), ("tree", 2 * 33 * 2, False, "i32"), ("out", 2 * 8 * 33 * 64, True, "bf16"), ("weights", 400, True, "fp32")]
    assert names(EVICT) == [("k", 25600, False, "fp16"), ("v", 25600, False, "fp16"), ("weights", 400, False, "fp32"), ("lengths", 2, False, "i32"),
                            ("k_out", 25600, True, "fp16"), ("v_out", 25600, True, "fp16"), ("weights_out", 400, True, "fp32"),
                            ("kept", 40, True, "i32"), ("lengths_out", 2, True, "i32")]
    assert [n for n, *_ in names({**COMMIT, "weights": True})] == ["path", "counts", "lengths", "k", "v", "weights", "lengths_out"]
    assert [n for n, *_ in names(COMMIT)] == ["path", "counts", "lengths", "k", "v", "lengths_out"]
    # a cache may be longer than 31 bits
    assert names({**TREE, "capacity": 1 << 30})[1][1] == 2 * 2 * (1 << 30) * 64


@pytest.mark.parametrize("spec,change,message", [
    (ROPE, {"heads": 7}, "multiple of kv_heads"), (ROPE, {"kv_heads": 0}, "kv_heads"), (ROPE, {"dim": 60}, "multiple of 8"),
    (ROPE, {"dim": 264}, "multiple of 8"), (ROPE, {"rotary": 33}, "rotary"), (ROPE, {"rotary": 66}, "rotary"),
    (ROPE, {"epsilon": 0.0}, "epsilon"), (ROPE, {"epsilon": None}, "epsilon"), (ROPE, {"base": 0.5}, "base"),
    (ROPE, {"scaling": "cubic", "factor": 2.0}, "scaling"), (ROPE, {"scaling": "linear"}, "factor"), (ROPE, {"scaling": "linear", "factor": 0.5}, "factor"),
    (ROPE, {"scaling": "ntk", "factor": 2.0, "rotary": 2}, "ntk"), (ROPE, {"scaling": "yarn", "factor": 2.0}, "original"),
    (ROPE, {"scaling": "yarn", "factor": 2.0, "original": 0}, "original"), (ROPE, {"capacity": 2}, "capacity"), (ROPE, {"capacity": 0}, "capacity"),
    (ROPE, {"seq": 0}, "sequence"), (ROPE, {"batch": 0}, "batch"), (ROPE, {"dtype": "tf32"}, "dtype"), (ROPE, {"out_dtype": "fp32"}, "input type"),
    (ROPE, {"batch": 65535, "seq": 131072}, "31-bit"), (GRAD, {"capacity": 50}, "no cache"),
    (TREE, {"seq": 129, "capacity": 1000}, "sequence"), (TREE, {"capacity": 32}, "capacity"), (TREE, {"capacity": (1 << 30) + 1}, "capacity"),
    (TREE, {"capacity": 1 << 30, "batch": 60}, "2^40"), (TREE, {"heads": 9}, "multiple of kv_heads"),
    (EVICT, {"keep": 0}, "keep"), (EVICT, {"keep": 101}, "keep"), (EVICT, {"recent": 11}, "recent"),
    (COMMIT, {"seq": 129}, "sequence"), (COMMIT, {"capacity": 8}, "capacity"),
])
def test_refusals(spec, change, message):
    jc.spec_validate(spec)
    bad = {k: v for k, v in {**spec, **change}.items() if v is not None}
    with pytest.raises(JadeError) as e:
        jc.spec_validate(bad)
    assert e.value.code == 1 and message in e.value.message


@pytest.mark.parametrize("spec", [ROPE, {**ROPE, "scaling": "yarn", "factor": 8.0, "original": 4096, "capacity": 9, "interleaved": True}, GRAD, TREE, EVICT, COMMIT])
def test_round_trip_and_no_reference_lowering(spec):
    text = jc.canonical(spec)
    again = json.loads(text)
    assert jc.canonical(again) == text and jc.spec_bindings(again) == jc.spec_bindings(spec)
    assert all(again[k] == v for k, v in spec.items() if not isinstance(v, float))
    for call in (jc.spec_launch, jc.emit, lambda s: jc.emit(s, "cuda")):
        with pytest.raises(JadeError):
            call(spec)


def test_outputs_must_not_alias():
    lengths = [b["elements"] for b in jc.spec_bindings(COMMIT)]
    jc.spec_validate_bindings(COMMIT, lengths, list(range(6)))
    with pytest.raises(JadeError, match="alias"):
        jc.spec_validate_bindings(COMMIT, lengths, [0, 1, 2, 3, 4, 2])  # lengths_out on lengths


def test_drafts_only_goes_with_weights():
    spec = {**TREE, "weights": True, "drafts_only": True}
    assert json.loads(jc.canonical(spec))["drafts_only"] is True and jc.spec_bindings(spec) == jc.spec_bindings({**TREE, "weights": True})
    assert jc.canonical({**spec, "drafts_only": False}) == jc.canonical({**TREE, "weights": True})
    with pytest.raises(JadeError, match="drafts_only"):
        jc.spec_validate({**TREE, "drafts_only": True})
