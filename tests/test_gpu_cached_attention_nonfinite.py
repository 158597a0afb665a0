"""attention_tree over caches that hold infinities and NaN in committed entries, and over
weights that span many powers of two: outputs and accumulated weights against the 64-bit
definition (tests/cached_reference.py; tolerances: tests/test_gpu_cached_attention.py),
in each form of the kernel: four, two and one copies of the rows, two row tiles (more
than 128 rows), FP32, and 16-bit heads above 128."""
import numpy as np
import pytest

import jade_compute_b200 as jc
from tests import cached_reference as R
from tests import test_gpu_cached_attention as base

pytestmark = pytest.mark.gpu

# (dtype, dim, rows): every kernel form
FORMS = [("bf16", 64, 4), ("fp16", 128, 32), ("bf16", 128, 40), ("fp16", 64, 64), ("bf16", 128, 72), ("fp16", 128, 128), ("bf16", 64, 132),
         ("fp16", 128, 200), ("bf16", 128, 256), ("fp16", 64, 300), ("fp32", 64, 4), ("fp32", 128, 40), ("bf16", 136, 20), ("fp16", 256, 6)]


@pytest.fixture(scope="module")
def rt():
    r = jc.Runtime(0)
    yield r
    r.close()


def inputs(dtype, dim, rows, batch, length, seed, kv_heads=2, q_sign=0):
    """seq * group = rows; q_sign: element 0 of every query is positive, so that an infinite
    element 0 of a key is an infinite score of its sign in every row."""
    seq = max(t for t in range(1, min(rows, 100) + 1) if rows % t == 0)
    case = dict(batch=batch, seq=seq, heads=rows // seq * kv_heads, kv_heads=kv_heads, dim=dim, capacity=length + seq, lengths=[length] * batch)
    x, sees = base.tree_inputs(case, dtype, seed)
    if q_sign:
        x["q"][..., 0] = R.rounded(np.abs(x["q"][..., 0]) + 0.25, dtype)
    return case, x, sees


def rows_of(got, case):
    """[batch, kv_heads, seq, group, dim]"""
    B, T, H, Hk, D = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    return got["out"].reshape(B, T, Hk, H // Hk, D).transpose(0, 2, 1, 3, 4)


@pytest.mark.parametrize("value", ["nan", "inf"])
@pytest.mark.parametrize("dtype,dim,rows", FORMS)
def test_committed_key_that_is_nan_or_scores_infinity_makes_its_head_nan(rt, dtype, dim, rows, value):
    # a NaN score is in every row's sum, an infinite one divides infinity by infinity: sequence
    # b has it at key 256 + b, so at each place of 16, and in kv head 0 alone
    case, x, sees = inputs(dtype, dim, rows, 16, 700, 70, q_sign=1)
    clean = base.tree_reference(case, x, sees)
    for b in range(16):
        x["k"][b, 0, 256 + b, 0] = float(value)
    got = R.run(rt, base.tree_spec(case, dtype), x)
    out = rows_of(got, case)
    assert np.isnan(out[:, 0]).all()
    u, exp_error = R.ROUNDOFF[dtype], 2e-5 if dtype == "fp32" else 1e-4
    ref, mag = (rows_of({"out": z}, case) for z in clean[:2])
    base.close(out[:, 1], ref[:, 1], mag[:, 1], u, exp_error + (0 if dtype == "fp32" else u))
    weights = got["weights"].reshape(16, 2, -1)
    if value == "nan":  # every weight of the row is NaN
        assert np.isnan(weights[:, 0, :700]).all()
    assert np.isnan(weights[np.arange(16), 0, 256 + np.arange(16)]).all() and np.isfinite(weights[:, 1]).all()


@pytest.mark.parametrize("rows", [4, 40, 72, 128, 132, 256])
def test_fp16_keeps_a_long_tail_of_small_weights(rt, rows):
    # One key of weight 1 and 1,023 of e^-17.5 = 2^-25.2 whose values alone are not 0: the
    # output is their sum. Two values round here: p, of at least 2^-25.2 of the largest, to the
    # type (relative error u down to 2^-25 of the largest weight, 2^-36 of it below), and the
    # output. Enough heads that a block has whole sequences.
    heads, length, dim = 160, 1023, 64
    seq = max(t for t in range(1, min(rows, 100) + 1) if rows % t == 0)
    case = dict(batch=1, seq=seq, heads=rows // seq * heads, kv_heads=heads, dim=dim, capacity=length + seq, lengths=[length])
    sees = np.zeros((1, seq, seq), bool)
    x = {"q": np.zeros((1, case["heads"], seq, dim)), "k": np.zeros((1, heads, length + seq, dim)), "v": np.zeros((1, heads, length + seq, dim)),
         "lengths": np.array([length], np.int32), "tree": R.tree_words(sees)}
    x["q"][..., 0] = 8.0
    x["k"][0, :, 0, 0] = 17.5  # score 17.5, the others 0
    x["v"][0, :, 1:length] = 1000.0
    ref, mag, _ = base.tree_reference(case, {**x, "weights": np.zeros((1, heads, length + seq))}, sees)
    got = R.run(rt, base.tree_spec(case, "fp16", False), x)["out"].reshape(ref.shape)
    u = R.ROUNDOFF["fp16"]
    small = 2.0 ** -36 * 1000.0 * length
    base.close(got, ref, mag + small / (u + 1e-4), u, u + 1e-4)


@pytest.mark.parametrize("case", [1, 3, 5])
def test_fp16_large_scores(rt, case):
    # the running maximum grows again and again, in smaller steps than in BF16
    base.test_attention_tree_large_scores(rt, case, "fp16")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows", [132, 256])
def test_visible_infinities_of_many_single_tile_sequences(rt, dtype, rows):
    # Sequences of one key tile each, several a block: whether a draft's values are infinite is
    # noted per sequence, and the two row tiles of a sequence finish apart from the next one's
    case, x, sees = inputs(dtype, 64, rows, 700, 20, 74)
    draft = np.arange(700) % case["seq"]
    odd = np.arange(700) % 3 != 1
    for b in np.nonzero(odd)[0]:
        x["v"][b, :, 20 + draft[b], b % 64] = np.inf
    out = rows_of(R.run(rt, base.tree_spec(case, dtype, False), x), case)
    for b in range(700):
        see = sees[b, :, draft[b]] if odd[b] else np.zeros(case["seq"], bool)
        assert np.isposinf(out[b][:, see, :, b % 64]).all()
        assert np.isfinite(out[b][:, ~see]).all() and np.isfinite(np.delete(out[b][:, see], b % 64, axis=-1)).all()


@pytest.mark.parametrize("dtype,dim,rows", FORMS)
def test_committed_keys_that_score_minus_infinity_weigh_nothing(rt, dtype, dim, rows):
    # single keys, whole tiles of 128 at a sequence's start, in its middle and over all its
    # committed keys but one: outputs are those of the other keys
    case, x, sees = inputs(dtype, dim, rows, 4, 700, 71, q_sign=1)
    for b, gone in enumerate(([0, 17, 130, 699], np.arange(128), np.r_[0:256, 384:512], np.delete(np.arange(700), 650))):
        x["k"][b, :, gone, 0] = -np.inf
    base.check_tree(R.run(rt, base.tree_spec(case, dtype, False), x), case, x, sees, dtype, weights=False)


@pytest.mark.parametrize("dtype,dim,rows", FORMS)
def test_weights_of_keys_that_score_minus_infinity_stay(rt, dtype, dim, rows):
    case, x, sees = inputs(dtype, dim, rows, 2, 700, 72, q_sign=1)
    x["k"][0, :, [3, 300, 699], 0] = -np.inf
    x["k"][1, :, 256:384, 0] = -np.inf
    got = R.run(rt, base.tree_spec(case, dtype), x)
    base.check_tree(got, case, x, sees, dtype)
    weights = got["weights"].reshape(x["weights"].shape)
    np.testing.assert_array_equal(weights[0][:, [3, 300, 699]], x["weights"][0][:, [3, 300, 699]])
    np.testing.assert_array_equal(weights[1][:, 256:384], x["weights"][1][:, 256:384])


@pytest.mark.parametrize("length", [1, 100, 700, 5000])
@pytest.mark.parametrize("dtype,dim,rows", FORMS)
def test_committed_infinity_in_v_reaches_its_column_as_it_is(rt, dtype, dim, rows, length):
    # p > 0 for every committed key, so p v is the infinity of v's sign in each of the head's
    # rows, in that column alone; NaN where the column holds both signs, or a NaN
    case, x, sees = inputs(dtype, dim, rows, 1, length, 73)
    clean = base.tree_reference(case, x, sees)[:2]
    places = [(5, 0, np.inf), (2, length // 2, -np.inf), (dim - 1, length - 1, np.inf), (0, length - 1, np.nan)]
    for column, key, value in places:
        x["v"][0, 0, key, column] = value
    if length > 1:
        x["v"][0, 0, 0, 3], x["v"][0, 0, length - 1, 3] = np.inf, -np.inf
    got = R.run(rt, base.tree_spec(case, dtype), x)
    out, ref, mag = (rows_of(z, case)[0] for z in (got, {"out": clean[0]}, {"out": clean[1]}))
    assert np.isposinf(out[0][..., 5]).all() and np.isneginf(out[0][..., 2]).all() and np.isposinf(out[0][..., dim - 1]).all()
    assert np.isnan(out[0][..., 0]).all() and (length == 1 or np.isnan(out[0][..., 3]).all())
    others = np.delete(np.arange(dim), [0, 2, 5, dim - 1] + ([3] if length > 1 else []))
    u = R.ROUNDOFF[dtype]
    c = 2e-5 if dtype == "fp32" else 1e-4 + u
    base.close(out[0][..., others], ref[0][..., others], mag[0][..., others], u, c)
    base.close(out[1], ref[1], mag[1], u, c)
    assert np.isfinite(got["weights"]).all()
