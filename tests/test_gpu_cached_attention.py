"""GPU parity of the cached attention operators against 64-bit numpy statements of
their formulas (tests/cached_reference.py) on the same rounded inputs.

Tolerances, per element, from where the kernels round (u: the type's unit roundoff,
2^-8 / 2^-11 / 2^-23; FP16 rounds values below 2^-14 to multiples of 2^-24, so there
its rounding is at most 2^-25 instead):
  rope        u |ref| + 4e-6 m, m = |a cos| + |b sin| of the turned pair: FP32 sum of
              squares (<= 256 terms, tree order, 1e-6), rsqrt (2^-22), sine and cosine
              (4e-7 absolute)
  gradient    u |ref| + 2e-5 m, m = r (|u| + |x r| mean|u x r|) with |u| from the turned
              pair's magnitude: the same roundings twice and two more sums; weights'
              gradients 2e-5 sum |g x r|
  attention   u |ref| + (u_p + 1e-4) m, m = sum p |v|: 16-bit types round p to the type
              before the product with v (u_p = u), FP32 does not and has no fast
              exponential in it (u_p = 0, 2e-5 in place of 1e-4); weights (sums of p)
              1e-4 of the sum, 2e-5 in FP32, and one rounding of the running total
  evict, commit  moved bits are equal
"""
import numpy as np
import pytest

import jade_compute_b200 as jc
from jade_compute_b200.runtime import JadeError
from tests import cached_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    r = jc.Runtime(0)
    yield r
    r.close()


def close(got, ref, m, u, c):
    rounding = np.maximum(u * np.abs(ref), 2.0 ** -25 if u == R.ROUNDOFF["fp16"] else 0.0)
    bad = ~(np.abs(got - ref) <= rounding + c * m)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], ref[bad][:4], m[bad][:4])


# ------------------------------------------------------------------ qk_norm_rope
ROPES = [
    dict(batch=1, seq=1, heads=1, kv_heads=1, dim=8),
    dict(batch=8, seq=1, heads=32, kv_heads=8, dim=128, capacity=40),
    dict(batch=2, seq=37, heads=6, kv_heads=2, dim=64, interleaved=True),
    dict(batch=3, seq=5, heads=7, kv_heads=1, dim=80, rotary=20, capacity=9),  # halves of 10: not whole vectors
    dict(batch=1, seq=130, heads=4, kv_heads=4, dim=96, rotary=48, scaling="yarn", factor=8.0, original=4096),
    dict(batch=2, seq=3, heads=2, kv_heads=1, dim=256, rotary=2, capacity=3),
    dict(batch=1, seq=19, heads=5, kv_heads=5, dim=24, rotary=0),
    dict(batch=2, seq=9, heads=3, kv_heads=3, dim=136, rotary=130, interleaved=True, scaling="linear", factor=4.0),
    dict(batch=2, seq=33, heads=8, kv_heads=2, dim=128, norm=False, scaling="ntk", factor=2.5, base=500000.0),
    dict(batch=1, seq=300, heads=16, kv_heads=16, dim=40, rotary=16, capacity=512),
]


def rope_inputs(spec, seed, first=0):
    rng = np.random.default_rng(seed)
    B, T, H, Hk, D, d = spec["batch"], spec["seq"], spec["heads"], spec["kv_heads"], spec["dim"], spec["dtype"]
    x = {"qkv": R.rounded(1.5 * rng.standard_normal((B, T, H + 2 * Hk, D)), d),
         "positions": (first + rng.integers(0, 200000, (B, T))).astype(np.int32)}
    if spec.get("norm", True):
        x["q_weight"] = R.rounded(1 + 0.2 * rng.standard_normal(D), d)
        x["k_weight"] = R.rounded(1 + 0.2 * rng.standard_normal(D), d)
    if "capacity" in spec:
        x["starts"] = rng.integers(0, spec["capacity"] - T + 1, B).astype(np.int32)
        x["starts"][0] = spec["capacity"] - T
        for n in "kv":
            x[n] = R.rounded(rng.standard_normal((B, Hk, spec["capacity"], D)), d)
    return x


def rope_spec(case, dtype, op="qk_norm_rope"):
    spec = {"op": op, "dtype": dtype, "epsilon": 1e-6, **case}
    if op.endswith("grad"):
        spec.pop("capacity", None)
    return spec


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", range(len(ROPES)))
def test_qk_norm_rope(rt, case, dtype):
    spec = rope_spec(ROPES[case], dtype)
    x = rope_inputs(spec, case)
    got = R.run(rt, spec, x)
    (q, mq), (k, mk), (v, _) = R.norm_rope(spec, x)
    B, T, Hk, D = spec["batch"], spec["seq"], spec["kv_heads"], spec["dim"]
    u = R.ROUNDOFF[dtype]
    close(got["q"].reshape(B, -1, T, D), q.transpose(0, 2, 1, 3), mq.transpose(0, 2, 1, 3), u, 4e-6)
    C = spec.get("capacity", T)
    for name, new, m in (("k", k, mk), ("v", v, None)):
        cache = got[name].reshape(B, Hk, C, D)
        for b in range(B):
            at = int(x["starts"][b]) if "capacity" in spec else 0
            rows = cache[b, :, at:at + T]
            if m is None:
                np.testing.assert_array_equal(rows, new[b].transpose(1, 0, 2))
            else:
                close(rows, new[b].transpose(1, 0, 2), m[b].transpose(1, 0, 2), u, 4e-6)
            if "capacity" in spec:  # every other slot keeps its bits
                old = np.delete(x[name][b], np.s_[at:at + T], axis=1)
                np.testing.assert_array_equal(np.delete(cache[b], np.s_[at:at + T], axis=1), old)


def test_rope_positions_to_the_ends_of_the_type(rt):
    # the angle is reduced exactly: negative positions and 2^31 - 1 turn as precisely as 1
    spec = rope_spec(dict(batch=1, seq=6, heads=2, kv_heads=1, dim=64), "fp32")
    x = rope_inputs(spec, 5)
    x["positions"] = np.array([[0, 1, -1, -(2 ** 31), 2 ** 31 - 1, 1 << 24]], np.int32)
    got = R.run(rt, spec, x)["q"].reshape(1, 2, 6, 64)
    # a 64-bit product of 2^31 and a frequency is itself off by 2e-7 rad
    (q, m), _, _ = R.norm_rope(spec, x)
    close(got, q.transpose(0, 2, 1, 3), m.transpose(0, 2, 1, 3), 2.0 ** -23, 4e-6)


def test_rope_carries_nan_and_infinity_in_their_own_rows_only(rt):
    spec = rope_spec(dict(batch=1, seq=4, heads=2, kv_heads=2, dim=64), "bf16")
    x = rope_inputs(spec, 6)
    clean = R.run(rt, spec, x)
    x["qkv"][0, 1, 0, 3] = np.nan  # a query
    x["qkv"][0, 2, 5, 7] = np.inf  # a value
    got = R.run(rt, spec, x)
    for name, at in (("q", (0, 1)), ("k", None), ("v", (1, 2))):
        a, b = got[name].reshape(2, 4, 64), clean[name].reshape(2, 4, 64)
        if at:
            assert not np.isfinite(a[at]).all()
            a[at] = b[at]
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("op", ["qk_norm_rope", "qk_norm_rope_grad"])
@pytest.mark.parametrize("rotary, interleaved", [(32, False), (20, False), (20, True), (32, True), (2, False), (2, True), (0, False)])
def test_rope_passes_infinities_beside_what_turns(rt, op, rotary, interleaved):
    # without norms an element that does not turn is copied, whatever it is, and reaches no other
    spec = rope_spec(dict(batch=1, seq=3, heads=2, kv_heads=1, dim=56, rotary=rotary, interleaved=interleaved, norm=False), "fp32", op)
    x = rope_inputs(spec, 7) if op == "qk_norm_rope" else grad_inputs(spec, 7)
    name, out = ("qkv", "q") if op == "qk_norm_rope" else ("dq", "dqkv")
    clean = R.run(rt, spec, x)[out].copy()
    bad = [rotary, rotary + 5, 55]
    x[name] = x[name].copy()
    rows = x[name][:, :, :2] if op == "qk_norm_rope" else x[name]  # of queries
    rows[..., bad] = [np.inf, np.nan, -np.inf]
    got = R.run(rt, spec, x)[out].copy()
    heads = (2, 3, 56) if op == "qk_norm_rope" else (3, 4, 56)
    got, clean = got.reshape(heads), clean.reshape(heads)
    queries = got if op == "qk_norm_rope" else got[:, :2]
    np.testing.assert_array_equal(queries[..., bad], np.broadcast_to(np.float32([np.inf, np.nan, -np.inf]), queries[..., bad].shape))
    queries[..., bad] = (clean if op == "qk_norm_rope" else clean[:, :2])[..., bad]
    np.testing.assert_array_equal(got, clean)


def rope_gradient(spec, x):
    """The formula's gradients and their magnitudes: dqkv, and dq_weight, dk_weight."""
    H, Hk = spec["heads"], spec["kv_heads"]
    at, out, mag, dw = x["positions"][:, :, None], [], [], {}
    for name, lo, hi in (("q", 0, H), ("k", H, H + Hk)):
        g, mg = R.turn(x["d" + name].transpose(0, 2, 1, 3), at, spec, -1.0)
        if spec.get("norm", True):
            row = x["qkv"][:, :, lo:hi]
            r = 1 / np.sqrt((row * row).mean(-1, keepdims=True) + spec["epsilon"])
            w = x[name + "_weight"]
            dw[name] = ((g * row * r).sum((0, 1, 2)), (mg * np.abs(row * r)).sum((0, 1, 2)))
            unit = row * r
            mg = r * (mg * np.abs(w) + np.abs(unit) * (mg * np.abs(w * unit)).mean(-1, keepdims=True))
            g = r * (g * w - unit * (g * w * unit).mean(-1, keepdims=True))
        out.append(g)
        mag.append(mg)
    dv = x["dv"].transpose(0, 2, 1, 3)
    return np.concatenate([*out, dv], 2), np.concatenate([*mag, 0 * dv], 2), dw


def grad_inputs(spec, seed):
    rng = np.random.default_rng(100 + seed)
    x = rope_inputs(spec, seed)
    B, T, H, Hk, D, d = spec["batch"], spec["seq"], spec["heads"], spec["kv_heads"], spec["dim"], spec["dtype"]
    for name, heads in (("dq", H), ("dk", Hk), ("dv", Hk)):
        x[name] = R.rounded(rng.standard_normal((B, heads, T, D)), d)
    return x


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", range(len(ROPES)))
def test_qk_norm_rope_grad(rt, case, dtype):
    spec = rope_spec(ROPES[case], dtype, "qk_norm_rope_grad")
    x = grad_inputs(spec, case)
    got = R.run(rt, spec, x, repeats=2)  # a second pass writes the same sums, not twice them
    ref, m, dw = rope_gradient(spec, x)
    close(got["dqkv"].reshape(ref.shape), ref, m, R.ROUNDOFF[dtype], 2e-5)
    for name, (s, ms) in dw.items():
        close(got[f"d{name}_weight"], s, ms, 0.0, 2e-5)


def test_qk_norm_rope_grad_against_differences(rt):
    # <gradient, direction> against a central difference of the forward formula in 64 bits,
    # step 1e-5: truncation 1e-10, rounding 1e-16 / 1e-5 of the sum's terms
    spec = rope_spec(dict(batch=2, seq=7, heads=4, kv_heads=2, dim=48, rotary=20, scaling="yarn", factor=4.0, original=128), "fp32",
                     "qk_norm_rope_grad")
    x = grad_inputs(spec, 3)
    got = R.run(rt, spec, x)
    rng = np.random.default_rng(9)

    def value(y):
        (q, _), (k, _), (v, _) = R.norm_rope(spec, y)
        return sum((d * z.transpose(0, 2, 1, 3)).sum() for d, z in ((x["dq"], q), (x["dk"], k), (x["dv"], v)))

    for name, grad in (("qkv", "dqkv"), ("q_weight", "dq_weight"), ("k_weight", "dk_weight")):
        step = rng.standard_normal(x[name].shape)
        ends = [value({**x, name: x[name] + h * step}) for h in (1e-5, -1e-5)]
        g = got[grad].reshape(x[name].shape)
        assert abs((ends[0] - ends[1]) / 2e-5 - (g * step).sum()) <= 2e-5 * np.abs(g * step).sum(), name


# ------------------------------------------------------------------ attention_tree
TREES = [
    dict(batch=1, seq=1, heads=1, kv_heads=1, dim=64, capacity=1, lengths=[0]),
    dict(batch=3, seq=1, heads=8, kv_heads=2, dim=128, capacity=700, lengths=[699, 0, 128]),
    dict(batch=2, seq=5, heads=6, kv_heads=6, dim=64, capacity=260, lengths=[127, 255]),  # pages end inside a tile
    dict(batch=3, seq=33, heads=4, kv_heads=1, dim=80, capacity=200, lengths=[0, 95, 167]),  # 132 rows, two mask words
    dict(batch=2, seq=128, heads=2, kv_heads=1, dim=96, capacity=900, lengths=[772, 1]),
    dict(batch=1, seq=64, heads=14, kv_heads=2, dim=128, capacity=3000, lengths=[2936]),  # 448 rows
    dict(batch=2, seq=3, heads=3, kv_heads=3, dim=8, capacity=64, lengths=[61, 20]),
    dict(batch=1, seq=7, heads=4, kv_heads=2, dim=256, capacity=333, lengths=[300]),
    dict(batch=5, seq=2, heads=4, kv_heads=4, dim=128, capacity=2100, lengths=[2098, 1000, 3, 0, 2047]),
    dict(batch=1, seq=1, heads=64, kv_heads=1, dim=128, capacity=9000, lengths=[8999]),
    dict(batch=1, seq=16, heads=8, kv_heads=8, dim=120, capacity=1500, lengths=[1400]),
    # more sequences than a warp has lanes, lengths around the tiles' ends, most items short
    dict(batch=77, seq=3, heads=4, kv_heads=2, dim=64, capacity=400, lengths=[(37 * b) % 398 if b % 5 else (0, 125, 126, 253, 397)[b // 5 % 5] for b in range(77)]),
    dict(batch=4, seq=10, heads=12, kv_heads=3, dim=72, capacity=1100, lengths=[1090, 118, 119, 500]),  # 40 rows
    dict(batch=2, seq=17, heads=6, kv_heads=2, dim=104, capacity=1300, lengths=[1283, 640]),  # 51 rows
    dict(batch=2, seq=100, heads=3, kv_heads=1, dim=64, capacity=5000, lengths=[4900, 20]),  # 300 rows: a second row block
]


def tree_spec(case, dtype, weights=True):
    return {"op": "attention_tree", "dtype": dtype, "weights": weights, **{k: v for k, v in case.items() if k != "lengths"}}


def tree_inputs(case, dtype, seed, scale=1.0):
    rng = np.random.default_rng(200 + seed)
    B, T, H, Hk, D, C = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim", "capacity"))
    sees = R.random_tree(rng, B, T)
    if T > 2:
        sees[0, -1] = False  # a token that sees no draft
    x = {"q": R.rounded(scale * rng.standard_normal((B, H, T, D)), dtype), "k": R.rounded(rng.standard_normal((B, Hk, C, D)), dtype),
         "v": R.rounded(rng.standard_normal((B, Hk, C, D)), dtype), "lengths": np.array(case["lengths"], np.int32),
         "tree": R.tree_words(sees), "weights": np.abs(rng.standard_normal((B, Hk, C))).astype(np.float32)}
    for b, n in enumerate(case["lengths"]):  # slots that nothing may read
        x["k"][b, :, n + T:] = np.nan
        x["v"][b, :, n + T:] = np.nan
    return x, sees


def tree_reference(case, x, sees):
    B, T, H, Hk, D = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    G = H // Hk
    out, mag, weights = np.zeros((B, T, H, D)), np.zeros((B, T, H, D)), x["weights"].astype(np.float64)
    for b, n in enumerate(case["lengths"]):
        mask = np.concatenate([np.ones((T, n), bool), sees[b]], 1)
        for h in range(Hk):
            o, m, p = R.attention(x["q"][b, h * G:(h + 1) * G].reshape(G * T, D), x["k"][b, h, :n + T], x["v"][b, h, :n + T],
                                  np.tile(mask, (G, 1)))
            out[b, :, h * G:(h + 1) * G] = o.reshape(G, T, D).transpose(1, 0, 2)
            mag[b, :, h * G:(h + 1) * G] = m.reshape(G, T, D).transpose(1, 0, 2)
            weights[b, h, :n + T] += p.sum(0)
    return out, mag, weights


def check_tree(got, case, x, sees, dtype, weights=True):
    out, mag, w = tree_reference(case, x, sees)
    u, exp_error = R.ROUNDOFF[dtype], 2e-5 if dtype == "fp32" else 1e-4
    close(got["out"].reshape(out.shape), out, mag, u, exp_error + (0 if dtype == "fp32" else u))
    if weights:
        added = w - x["weights"]
        close(got["weights"].reshape(w.shape), w, added, 2.0 ** -23, exp_error)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", range(len(TREES)))
def test_attention_tree(rt, case, dtype):
    x, sees = tree_inputs(TREES[case], dtype, case)
    got = R.run(rt, tree_spec(TREES[case], dtype), x)
    check_tree(got, TREES[case], x, sees, dtype)


# off the tensor core: every count of row groups and of warps that share a tile's keys, lengths
# around tiles of 16 and 32 keys, many tiles a block, heads that do not fill a warp's lanes
NARROW = [
    dict(batch=6, seq=1, heads=3, kv_heads=3, dim=136, capacity=99, lengths=[98, 0, 15, 16, 31, 32]),
    dict(batch=3, seq=5, heads=2, kv_heads=2, dim=256, capacity=400, lengths=[395, 11, 27]),  # two groups
    dict(batch=2, seq=3, heads=8, kv_heads=2, dim=200, capacity=700, lengths=[697, 30]),  # three
    dict(batch=2, seq=13, heads=1, kv_heads=1, dim=248, capacity=2500, lengths=[2400, 51]),  # four, the last with one row
    dict(batch=2, seq=19, heads=2, kv_heads=2, dim=192, capacity=300, lengths=[281, 13]),  # five: blocks of three
    dict(batch=40, seq=1, heads=16, kv_heads=16, dim=144, capacity=500, lengths=[(131 * b) % 500 for b in range(40)]),
    dict(batch=2, seq=125, heads=4, kv_heads=2, dim=160, capacity=260, lengths=[135, 0]),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", range(len(NARROW)))
def test_attention_tree_wide_heads(rt, case, dtype):
    x, sees = tree_inputs(NARROW[case], dtype, 50 + case)
    got = R.run(rt, tree_spec(NARROW[case], dtype), x)
    check_tree(got, NARROW[case], x, sees, dtype)
    again = R.run(rt, tree_spec(NARROW[case], dtype), x)
    np.testing.assert_array_equal(got["out"], again["out"])
    np.testing.assert_array_equal(got["weights"], again["weights"])


@pytest.mark.parametrize("dim", [8, 24, 64, 88, 128])
@pytest.mark.parametrize("rows", [1, 4, 6, 12, 16, 21, 35])
def test_attention_tree_fp32_rows(rt, rows, dim):
    case = dict(batch=3, seq=rows, heads=2, kv_heads=2, dim=dim, capacity=1000, lengths=[960, 31 - rows if rows < 31 else 3, 0])
    x, sees = tree_inputs(case, "fp32", 60 + rows)
    check_tree(R.run(rt, tree_spec(case, "fp32"), x), case, x, sees, "fp32")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_tree_without_weights_is_the_same(rt, dtype):
    x, _ = tree_inputs(TREES[4], dtype, 4)
    a, b = (R.run(rt, tree_spec(TREES[4], dtype, w), x) for w in (True, False))
    np.testing.assert_array_equal(a["out"], b["out"])
    assert "weights" not in b


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("case", [1, 3, 5])
def test_attention_tree_large_scores(rt, case, dtype):
    # scores of some hundreds: the softmax picks single keys, and the running maximum grows
    # again and again. An error of eps |s| in a score moves p by as much: the bound's FP32 term
    # grows with the largest score
    x, sees = tree_inputs(TREES[case], dtype, case, scale=30.0)
    got = R.run(rt, tree_spec(TREES[case], dtype), x)
    out, mag, w = tree_reference(TREES[case], x, sees)
    top = 30.0 * 6 * np.sqrt(TREES[case]["dim"])
    score_error = 2.0 ** -21 * top
    u = R.ROUNDOFF[dtype]
    close(got["out"].reshape(out.shape), out, mag, u, score_error + 1e-4 + (0 if dtype == "fp32" else u))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("case", [3, 4, 8])
def test_attention_tree_masked_nan_and_infinity_stay_away(rt, case, dtype):
    masked_nan_and_infinity(rt, TREES[case], dtype)


@pytest.mark.parametrize("case", [2, 4, 6])
def test_attention_tree_wide_heads_masked_nan_and_infinity_stay_away(rt, case):
    masked_nan_and_infinity(rt, NARROW[case], "fp16")


def masked_nan_and_infinity(rt, case, dtype):
    x, sees = tree_inputs(case, dtype, 30)
    T = case["seq"]
    hidden = T // 2  # a draft that only itself sees
    sees[:, :, hidden] = False
    sees[:, hidden, hidden] = True
    x["tree"] = R.tree_words(sees)
    for b, n in enumerate(case["lengths"]):
        x["k"][b, :, n + hidden] = np.inf
        x["v"][b, :, n + hidden] = np.nan
        x["v"][b, :, n + hidden, ::2] = -np.inf
    got = R.run(rt, tree_spec(case, dtype), x)["out"].reshape(case["batch"], T, case["heads"], -1)
    assert not np.isfinite(got[:, hidden]).any()
    clean = {n: v.copy() for n, v in x.items()}
    for b, n in enumerate(case["lengths"]):
        clean["k"][b, :, n + hidden] = clean["v"][b, :, n + hidden] = 0
    out, mag, _ = tree_reference(case, clean, sees)
    u = R.ROUNDOFF[dtype]
    others = np.arange(T) != hidden
    close(got[:, others], out[:, others], mag[:, others], u, 1e-4 + (0 if dtype == "fp32" else u))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_attention_tree_visible_infinity_reaches_exactly_its_rows(rt, dtype):
    case = TREES[3]
    x, sees = tree_inputs(case, dtype, 31)
    x["v"][1, 0, case["lengths"][1] + 2, 5] = np.inf  # draft 2 of sequence 1
    got = R.run(rt, tree_spec(case, dtype), x)["out"].reshape(3, 33, 4, 80)
    see = sees[1, :, 2]
    assert np.isposinf(got[1, see, :, 5]).all() and np.isfinite(got[1, ~see]).all()
    assert np.isfinite(np.delete(got[1, see], 5, axis=-1)).all() and np.isfinite(got[[0, 2]]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_tree_empty_rows_are_zero(rt, dtype):
    case = dict(batch=2, seq=40, heads=4, kv_heads=2, dim=64, capacity=64, lengths=[0, 10])
    x, sees = tree_inputs(case, dtype, 32)
    sees[0] = False
    sees[1, ::3] = False
    x["tree"] = R.tree_words(sees)
    got = R.run(rt, tree_spec(case, dtype), x)
    assert not got["out"].reshape(2, -1)[0].any()
    check_tree(got, case, x, sees, dtype)


def test_attention_tree_repeats_bit_for_bit_and_accumulates(rt):
    case = TREES[5]
    x, sees = tree_inputs(case, "bf16", 33)
    a, b = (R.run(rt, tree_spec(case, "bf16"), x) for _ in range(2))
    np.testing.assert_array_equal(a["out"], b["out"])
    np.testing.assert_array_equal(a["weights"], b["weights"])
    thrice = R.run(rt, tree_spec(case, "bf16"), x, repeats=3)
    _, _, w = tree_reference(case, x, sees)
    added = w - x["weights"]
    close(thrice["weights"].reshape(w.shape), x["weights"] + 3 * added, 3 * added, 2.0 ** -22, 1e-4)


class Span:
    """A buffer as torch sees device memory."""

    def __init__(self, buf):
        kind, size = {"bf16": ("<i2", 2), "i32": ("<i4", 4), "fp32": ("<f4", 4)}[buf.dtype]
        self.buf = buf
        self.__cuda_array_interface__ = {"shape": (buf.nbytes // size,), "typestr": kind, "data": (buf.ptr, False), "version": 3}


def test_caches_beyond_32_bit_offsets(rt):
    # 2 sequences of 2^24 + 8 slots of 128 elements: sequence 1 starts behind element 2^31
    # (byte 2^32); its rows come out as in a small cache
    import torch
    C, D, T, n = (1 << 24) + 8, 128, 4, 1000
    small = dict(batch=1, seq=T, heads=2, kv_heads=1, dim=D, capacity=n + T, lengths=[n])
    x, sees = tree_inputs(small, "bf16", 40)
    spec = {**tree_spec(small, "bf16", False), "batch": 2, "capacity": C}
    kernel = rt.compile(spec)
    buffers = {b["name"]: rt.alloc(b["elements"], b["dtype"]) for b in kernel.info["bindings"]}
    try:
        views = {n: torch.as_tensor(Span(b), device="cuda") for n, b in buffers.items()}
        for name in "kv":
            rows = torch.from_numpy(jc.f32_to_bf16(x[name].ravel()).view(np.int16)).cuda()
            views[name].view(2, C, D)[1, :n + T] = rows.view(n + T, D)
        torch.cuda.synchronize()
        rt.upload(buffers["q"], jc.f32_to_bf16(np.concatenate([0 * x["q"], x["q"]]).ravel().astype(np.float32)))
        rt.upload(buffers["lengths"], np.array([0, n], np.int32))
        rt.upload(buffers["tree"], np.concatenate([x["tree"]] * 2).ravel())
        rt.execute([(kernel, [buffers[b["name"]] for b in kernel.info["bindings"]])])
        got = {"out": rt.download_f32(buffers["out"]).reshape(2, -1)[1].astype(np.float64)}
        check_tree(got, small, x, sees, "bf16", weights=False)
        # the same rows appended by qk_norm_rope at the far end, and moved by cache_commit
        rope = rope_spec(dict(batch=2, seq=T, heads=2, kv_heads=1, dim=D, capacity=C), "bf16")
        y = rope_inputs({**rope, "capacity": 16}, 41)
        k_rope = rt.compile(rope)
        extra = {"starts": np.array([0, C - T], np.int32), "qkv": y["qkv"], "positions": y["positions"], "q_weight": y["q_weight"],
                 "k_weight": y["k_weight"]}
        more = {}
        for b in k_rope.info["bindings"]:
            if b["name"] in extra:
                more[b["name"]] = rt.alloc(b["elements"], b["dtype"])
                v = np.asarray(extra[b["name"]]).ravel()
                rt.upload(more[b["name"]], v if b["dtype"] == "i32" else jc.f32_to_bf16(v.astype(np.float32)))
        commit = rt.compile({"op": "cache_commit", "batch": 2, "kv_heads": 1, "dim": D, "capacity": C, "seq": T, "dtype": "bf16"})
        for name, v in (("path", np.array([[0, 1, 2, 3], [1, 3, 3, 3]], np.int32)), ("counts", np.array([0, 2], np.int32)),
                        ("lengths", np.array([0, C - T], np.int32)), ("lengths_out", np.zeros(2, np.int32))):
            more["c_" + name] = rt.alloc(v.size, "i32")
            rt.upload(more["c_" + name], v.ravel())
        rt.execute([(k_rope, [more.get(b["name"], buffers.get(b["name"])) for b in k_rope.info["bindings"]]),
                    (commit, [more["c_path"], more["c_counts"], more["c_lengths"], buffers["k"], buffers["v"], more["c_lengths_out"]])])
        _, _, (v, _) = R.norm_rope(rope, y)
        tail = views["v"].view(2, C, D)[1, C - T:].cpu().numpy().view(np.uint16)
        want = jc.f32_to_bf16(v[1, [1, 3, 2, 3], 0].astype(np.float32))
        np.testing.assert_array_equal(tail, want.reshape(T, D))
        assert rt.download(more["c_lengths_out"]).tolist() == [0, C - 2]
        for b in more.values():
            b.free()
    finally:
        views = None
        for b in buffers.values():
            b.free()


# ------------------------------------------------------------------ cache_evict, cache_commit
EVICTS = [
    dict(batch=1, kv_heads=1, dim=8, capacity=1, keep=1, recent=0, lengths=[1]),
    dict(batch=3, kv_heads=2, dim=64, capacity=700, keep=100, recent=10, lengths=[700, 0, 99]),
    dict(batch=2, kv_heads=3, dim=80, capacity=3000, keep=1025, recent=1025, lengths=[3000, 1026]),  # the newest alone
    dict(batch=4, kv_heads=1, dim=128, capacity=5000, keep=5000, recent=7, lengths=[5000, 4999, 1, 3]),  # nothing goes
    dict(batch=2, kv_heads=2, dim=96, capacity=70000, keep=4097, recent=64, lengths=[70000, 66000]),
]


def evict_reference(case, x):
    keep, recent = case["keep"], case["recent"]
    B, H, C, D = (case[n] for n in ("batch", "kv_heads", "capacity", "dim"))
    kept = np.full((B, H, keep), -1, np.int64)
    for b, n in enumerate(case["lengths"]):
        count, last = min(n, keep), max(0, n - recent)
        for h in range(H):
            w = x["weights"][b, h, :last].astype(np.float64)
            w = np.where(np.isnan(w), np.inf, w)
            nan_first = np.lexsort((np.arange(last), -w, ~np.isnan(x["weights"][b, h, :last])))
            kept[b, h, :count] = sorted(nan_first[:count - (n - last)].tolist() + list(range(last, n)))
    return kept


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind", ["spread", "ties", "strange"])
@pytest.mark.parametrize("case", range(len(EVICTS)))
def test_cache_evict(rt, case, kind, dtype):
    case = EVICTS[case]
    rng = np.random.default_rng(300)
    B, H, C, D, keep = (case[n] for n in ("batch", "kv_heads", "capacity", "dim", "keep"))
    w = np.exp(1.5 * rng.standard_normal((B, H, C))).astype(np.float32)
    if kind == "ties":  # a few values, many equal
        w = np.round(w).astype(np.float32)
    if kind == "strange":  # signs, both zeros, infinities, NaN
        w = rng.choice(np.array([0.0, -0.0, 1e-45, -3.0, np.inf, -np.inf, np.nan, 2.5, 2.5000002], np.float32), (B, H, C))
    x = {"k": R.rounded(rng.standard_normal((B, H, C, D)), dtype), "v": R.rounded(rng.standard_normal((B, H, C, D)), dtype),
         "weights": w, "lengths": np.array(case["lengths"], np.int32), "k_out": np.full((B, H, C, D), 7.0), "v_out": np.full((B, H, C, D), 7.0)}
    x["k_out"] = x["k_out"].astype(np.float32)
    x["v_out"] = x["v_out"].astype(np.float32)
    # outputs' old contents: `run` uploads them too
    spec = {"op": "cache_evict", "dtype": dtype, **{n: v for n, v in case.items() if n != "lengths"}}
    got = R.run(rt, spec, x)
    kept = evict_reference(case, x)
    np.testing.assert_array_equal(got["kept"].reshape(kept.shape), kept)
    assert got["lengths_out"].tolist() == [min(n, keep) for n in case["lengths"]]
    for b, n in enumerate(case["lengths"]):
        count = min(n, keep)
        for h in range(H):
            rows = kept[b, h, :count]
            for name in "kv":
                out = got[name + "_out"].reshape(B, H, C, D)[b, h]
                np.testing.assert_array_equal(out[:count], x[name][b, h, rows])
                assert (out[count:] == 7.0).all()
            out = got["weights_out"].reshape(B, H, C)[b, h]
            np.testing.assert_array_equal(out[:count], w[b, h, rows].astype(np.float64))
            assert not out[count:].any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("B,H,D,T,C", [(1, 1, 8, 1, 1), (3, 2, 64, 5, 20), (4, 3, 80, 128, 300), (2, 1, 256, 77, 77), (9, 8, 128, 33, 64)])
def test_cache_commit(rt, B, H, D, T, C, weights, dtype):
    rng = np.random.default_rng(400)
    lengths = rng.integers(0, C - T + 1, B).astype(np.int32)
    counts = rng.integers(0, T + 1, B).astype(np.int32)
    counts[0] = T
    path = np.stack([np.sort(rng.permutation(T)) for _ in range(B)]).astype(np.int32)
    for b in range(B):
        path[b, :counts[b]] = np.sort(rng.permutation(T)[:counts[b]])
    x = {"k": R.rounded(rng.standard_normal((B, H, C, D)), dtype), "v": R.rounded(rng.standard_normal((B, H, C, D)), dtype),
         "weights": rng.random((B, H, C)).astype(np.float32), "lengths": lengths, "counts": counts, "path": path}
    spec = {"op": "cache_commit", "batch": B, "kv_heads": H, "dim": D, "capacity": C, "seq": T, "dtype": dtype, "weights": weights}
    got = R.run(rt, spec, x)
    ref = {n: x[n].astype(np.float64).copy() for n in ("k", "v", "weights")}
    for b in range(B):
        n, a = lengths[b], counts[b]
        for name in ("k", "v", "weights"):
            moved = ref[name][b][:, n + path[b, :a]].copy()
            if name == "weights":
                ref[name][b][:, n:n + T] = 0
            ref[name][b][:, n:n + a] = moved
    for name in ("k", "v") + (("weights",) if weights else ()):
        np.testing.assert_array_equal(got[name].reshape(ref[name].shape), ref[name])
    assert got["lengths_out"].tolist() == (lengths + counts).tolist()


# ------------------------------------------------------------------ refusals that only the device can make
def test_lengths_outside_the_cache_are_reported_and_skipped(rt):
    case = dict(TREES[1])
    x, sees = tree_inputs(case, "bf16", 50)
    for bad in (-1, 700):
        x["lengths"] = np.array([699, bad, 128], np.int32)
        with pytest.raises(JadeError, match="cache length") as e:
            R.run(rt, tree_spec(case, "bf16"), x)
        assert e.value.code == 1
        with pytest.raises(JadeError, match="cache length"):
            R.run(rt, tree_spec(case, "fp32"), x)
    spec = rope_spec(ROPES[1], "bf16")
    y = rope_inputs(spec, 1)
    y["starts"][3] = spec["capacity"]
    with pytest.raises(JadeError, match="cache length"):
        R.run(rt, spec, y)
    ev = {"op": "cache_evict", "batch": 1, "kv_heads": 1, "dim": 8, "capacity": 4, "keep": 2, "dtype": "bf16"}
    with pytest.raises(JadeError, match="cache length"):
        R.run(rt, ev, {"lengths": np.array([5], np.int32)})
    # the context carries on
    x["lengths"] = np.array(case["lengths"], np.int32)
    check_tree(R.run(rt, tree_spec(case, "bf16"), x), case, x, sees, "bf16")


@pytest.mark.parametrize("path,count", [([0, 2, 1, 3], 4), ([0, 0, 1, 2], 2), ([0, 1, 2, 4], 4), ([-1, 1, 2, 3], 1), ([0, 1, 2, 3], 5), ([0, 1, 2, 3], -1)])
def test_commit_refuses_a_path_that_is_none(rt, path, count):
    spec = {"op": "cache_commit", "batch": 1, "kv_heads": 2, "dim": 8, "capacity": 9, "seq": 4, "dtype": "fp32"}
    x = {"path": np.array(path, np.int32), "counts": np.array([count], np.int32), "lengths": np.array([2], np.int32)}
    with pytest.raises(JadeError, match="path must ascend") as e:
        R.run(rt, spec, x)
    assert e.value.code == 1


# ------------------------------------------------------------------ batch times read on request
def test_batch_times_outlive_the_next_batch_and_the_runtime():
    r = jc.Runtime(0)
    k = r.compile({"op": "l2_flush", "bytes": 1 << 28})
    b = r.alloc_bytes(1 << 28)
    try:
        r.execute([(k, [b])])  # nobody holds this one
        first = r.execute([(k, [b])], repeats=20)
        second = r.execute([(k, [b])])
        third = r.execute([(k, [b])], repeats=20)
    finally:
        r.close()
    assert second.gpu_ms > 0 and first.gpu_ms > 5 * second.gpu_ms and third.gpu_ms > 5 * second.gpu_ms
    assert first.gpu_ms == first.gpu_ms


# ------------------------------------------------------------------ the runtime's ways to run a batch
def tensors(rt, spec, arrays):
    kernel, bufs = rt.compile(spec), {}
    for b in kernel.info["bindings"]:
        bufs[b["name"]] = rt.alloc(b["elements"], b["dtype"])
        if b["name"] in arrays:
            x = np.asarray(arrays[b["name"]]).ravel()
            rt.upload(bufs[b["name"]], x if b["dtype"] == "i32" else jc.f32_to_bf16(x.astype(np.float32)) if b["dtype"] == "bf16" else x)
    return kernel, bufs


@pytest.mark.parametrize("way", [{"graph": True}, {"streams": True}, {"per_job": True}])
def test_batches_of_several_operators_run_every_way(rt, way):
    # two attention kernels with their own workspaces in turn, an eviction and a gradient: each
    # is several launches, some started early; a graph, transfer streams and per-job events
    # give what single batches gave
    cases = [(tree_spec(TREES[i], "bf16"), tree_inputs(TREES[i], "bf16", i)[0]) for i in (1, 4)]
    ev = {"op": "cache_evict", "batch": 1, "kv_heads": 2, "dim": 64, "capacity": 900, "keep": 100, "recent": 5, "dtype": "bf16"}
    rng = np.random.default_rng(60)
    cases.append((ev, {"k": R.rounded(rng.standard_normal((1, 2, 900, 64)), "bf16"), "v": R.rounded(rng.standard_normal((1, 2, 900, 64)), "bf16"),
                       "weights": rng.random((1, 2, 900)).astype(np.float32), "lengths": np.array([850], np.int32)}))
    grad = rope_spec(ROPES[1], "bf16", "qk_norm_rope_grad")
    cases.append((grad, grad_inputs(grad, 1)))
    jobs = [tensors(rt, spec, x) for spec, x in cases]
    try:
        expected = [R.run(rt, spec, x) for spec, x in cases]
        batch = [(k, [bufs[b["name"]] for b in k.info["bindings"]]) for k, bufs in jobs]
        done = rt.execute(batch, **way)
        assert not way.get("per_job") or min(done.job_ms) > 0
        for (k, bufs), want in zip(jobs, expected):
            for name, values in want.items():
                got = rt.download(bufs[name]) if bufs[name].dtype == "i32" else rt.download_f32(bufs[name])
                np.testing.assert_array_equal(got.astype(values.dtype), values, err_msg=name)
        if "graph" in way:  # replays: the attention weights accumulate, everything else stays
            rt.execute(batch, repeats=3, graph=True)
            for (k, bufs), want in zip(jobs, expected):
                for name, values in want.items():
                    if name != "weights":
                        got = rt.download(bufs[name]) if bufs[name].dtype == "i32" else rt.download_f32(bufs[name])
                        np.testing.assert_array_equal(got.astype(values.dtype), values, err_msg=name)
    finally:
        for k, bufs in jobs:
            for b in bufs.values():
                b.free()


def test_weight_gradients_repeat_bit_for_bit(rt):
    spec = rope_spec(dict(batch=3, seq=700, heads=8, kv_heads=2, dim=96, rotary=32), "bf16", "qk_norm_rope_grad")
    x = grad_inputs(spec, 61)
    a, b = (R.run(rt, spec, x, repeats=n) for n in (1, 3))
    for name in a:
        np.testing.assert_array_equal(a[name], b[name])
    ref, m, dw = rope_gradient(spec, x)
    close(a["dqkv"].reshape(ref.shape), ref, m, R.ROUNDOFF["bf16"], 2e-5)
    for name, (s, ms) in dw.items():
        close(a[f"d{name}_weight"], s, ms, 0.0, 2e-5)
