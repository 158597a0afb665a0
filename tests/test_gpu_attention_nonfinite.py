"""Prompt attention over keys that are NaN or score infinity: their rows are NaN, in every
kernel (persistent two-tile, CTA pair, FP32) and at each place of a key tile."""
import numpy as np
import pytest

import jade_compute_b200 as jc
from tests import cached_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    r = jc.Runtime(0)
    yield r
    r.close()


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,dim,seq", [("bf16", 64, 640), ("bf16", 128, 640), ("fp16", 128, 640), ("bf16", 128, 2048), ("fp32", 64, 256)])
def test_key_that_is_nan_or_scores_infinity(rt, dtype, dim, seq, causal, value):
    # head h has it at key 130 + h, which every query from there on sees
    heads = 16
    rng = np.random.default_rng(90)
    q, k, v = (R.rounded(rng.standard_normal((heads, seq, dim)), dtype) for _ in range(3))
    q[..., 0] = R.rounded(np.abs(q[..., 0]) + 0.25, dtype)
    clean = R.run(rt, spec := {"op": "attention_online", "heads": heads, "seq": seq, "dim": dim, "causal": causal, "dtype": dtype},
                  {"q": q, "k": k, "v": v})["out"].reshape(heads, seq, dim)
    for h in range(heads):
        k[h, 130 + h, 0] = value
    got = R.run(rt, spec, {"q": q, "k": k, "v": v})["out"].reshape(heads, seq, dim)
    for h in range(heads):
        first = 130 + h if causal else 0
        assert np.isnan(got[h, first:]).all(), h
        np.testing.assert_array_equal(got[h, :first], clean[h, :first])
