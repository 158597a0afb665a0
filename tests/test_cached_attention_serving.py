"""CachedAttention's accumulated weights and its forms, against the 64-bit definition on the
buffers that the layer's attention read (tolerances: tests/test_gpu_cached_attention.py)."""
import numpy as np
import pytest

import jade_compute_b200 as jc
from jade_compute_b200.cached_attention import CachedAttention, causal_tree, tree_words
from tests import cached_reference as R
from tests import test_gpu_cached_attention as base

pytestmark = pytest.mark.gpu
B, T, WIDTH, H, HK, D, C = 2, 4, 64, 4, 2, 32, 60


@pytest.fixture(scope="module")
def rt():
    r = jc.Runtime(0)
    yield r
    r.close()


def make(rt, **options):
    layer = CachedAttention(rt, B, T, WIDTH, H, HK, D, C, **options)
    rng = np.random.default_rng(5)
    layer.load(0.2 * rng.standard_normal((WIDTH, (H + 2 * HK) * D)), 0.2 * rng.standard_normal((H * D, WIDTH)), np.ones(D), np.ones(D))
    return layer


def added_weights(rt, layer, lengths, sees, rows=None):
    """The definition's sum of weights of the layer's last step; rows [B, T]: those that count."""
    def fetch(buf, *shape):
        return rt.download_f32(buf).astype(np.float64).reshape(shape)

    q, k, v = fetch(layer.q, B, H, T, D), fetch(layer.k, B, HK, C, D), fetch(layer.v, B, HK, C, D)
    added = np.zeros((B, HK, C))
    for b in range(B):
        live = slice(0, lengths[b] + T)
        mask = np.concatenate([np.ones((T, lengths[b]), bool), sees[b]], 1)
        for h in range(HK):
            p = R.attention(q[b, h * H // HK:(h + 1) * H // HK].reshape(-1, D), k[b, h, live], v[b, h, live], np.tile(mask, (H // HK, 1)))[2]
            added[b, h, live] = (p.reshape(H // HK, T, -1) * (1 if rows is None else rows[b][:, None])).sum((0, 1))
    return added


def held_weights(rt, layer):
    return rt.download_f32(layer.weights).astype(np.float64).reshape(B, HK, C)


def near(got, ref):
    bound = 1e-4 * ref + 1e-6
    assert (np.abs(got - ref) <= bound).all(), np.max(np.abs(got - ref) - bound)


CAUSAL = np.tile(np.tril(np.ones((T, T), bool)), (B, 1, 1))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_layer_without_head_norms(rt, dtype):
    rng = np.random.default_rng(8)
    layer = CachedAttention(rt, B, T, WIDTH, H, HK, D, C, dtype=dtype, norm=False)
    wqkv = R.rounded(0.2 * rng.standard_normal((WIDTH, (H + 2 * HK) * D)), dtype)
    layer.load(wqkv, 0.2 * rng.standard_normal((H * D, WIDTH)))
    try:
        at = np.tile(np.arange(T), (B, 1))
        y = layer.step(rng.standard_normal((B, T, WIDTH)), at)
        assert np.isfinite(y).all()
        qkv = rt.download_f32(layer.qkv).astype(np.float64).reshape(B, T, H + 2 * HK, D)
        (q, m), _, _ = R.norm_rope({"heads": H, "kv_heads": HK, "dim": D, "norm": False}, {"qkv": qkv, "positions": at})
        got = rt.download_f32(layer.q).astype(np.float64).reshape(B, H, T, D)
        u, tiny = R.ROUNDOFF[dtype], 2.0 ** -25 if dtype == "fp16" else 0.0
        q, m = q.transpose(0, 2, 1, 3), m.transpose(0, 2, 1, 3)
        assert (np.abs(got - q) <= np.maximum(u * np.abs(q), tiny) + 4e-6 * m).all()
        assert layer.commit().tolist() == [T] * B
    finally:
        layer.release()


def test_load_wants_the_norm_weights_that_the_layer_has(rt):
    wqkv, wo = np.zeros((WIDTH, (H + 2 * HK) * D)), np.zeros((H * D, WIDTH))
    for options, weights in (({}, []), ({}, [np.ones(D)]), ({"norm": False}, [np.ones(D)] * 2)):
        layer = CachedAttention(rt, B, T, WIDTH, H, HK, D, C, **options)
        with pytest.raises(ValueError, match="norm weights"):
            layer.load(wqkv, wo, *weights)
        layer.release()
def test_step_that_is_not_committed_leaves_no_weight(rt):
    # a step over again, with other tokens, as a server makes it after a failed draft
    rng = np.random.default_rng(6)
    layer = make(rt, keep=16, recent=2)
    try:
        lengths, expected = np.zeros(B, int), np.zeros((B, HK, C))
        for n in range(6):
            at = lengths[:, None] + np.arange(T)
            for tries in range(1 + n % 3):
                layer.step(rng.standard_normal((B, T, WIDTH)), at, causal_tree(B, T))
            working = expected + added_weights(rt, layer, lengths, CAUSAL)
            near(held_weights(rt, layer), working)
            counts = np.array([T, T - n % 2])
            layer.commit(counts=counts)
            for b in range(B):
                working[b, :, lengths[b] + counts[b]:] = 0
            expected, lengths = working, lengths + counts
            near(held_weights(rt, layer), expected)
        layer.step(rng.standard_normal((B, T, WIDTH)), lengths[:, None] + np.arange(T))
        kept = layer.evict()  # of the committed entries by their committed weights
        for b in range(B):
            for h in range(HK):
                slots = kept[b, h][kept[b, h] >= 0]
                near(held_weights(rt, layer)[b, h, :len(slots)], expected[b, h, slots])
                older = np.delete(np.arange(lengths[b] - 2), slots[slots < lengths[b] - 2])
                assert expected[b, h, older].max() <= expected[b, h, slots[slots < lengths[b] - 2]].min() * (1 + 2e-4)
    finally:
        layer.release()


def test_places_without_a_draft_add_no_weight(rt):
    # the last piece of a prompt, a tree smaller than the step: their rows are no tokens
    rng = np.random.default_rng(7)
    layer = make(rt, keep=16, recent=2)
    try:
        layer.step(rng.standard_normal((B, T, WIDTH)), np.tile(np.arange(T), (B, 1)), causal_tree(B, T))
        expected = added_weights(rt, layer, [0] * B, CAUSAL)
        layer.commit()
        words = tree_words([[-1, 0, -2, -2], [-1, 0, 0, -2]])
        layer.step(rng.standard_normal((B, T, WIDTH)), T + np.tile(np.arange(T), (B, 1)), words)
        sees = (words[:, :, 0, None] >> np.arange(T) & 1).astype(bool)
        rows = sees.any(-1)
        assert rows.tolist() == [[True, True, False, False], [True, True, True, False]]
        near(held_weights(rt, layer), expected + added_weights(rt, layer, [T] * B, sees, rows))
    finally:
        layer.release()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", [1, 3, 4, 5, 7, 12, 13, 14])
def test_drafts_only_leaves_out_rows_that_see_no_draft(rt, case, dtype):
    case = base.TREES[case]
    x, sees = base.tree_inputs(case, dtype, 80)
    rng = np.random.default_rng(81)
    sees &= (rng.random(sees.shape[:2]) < 0.6)[:, :, None]
    sees[0, 0] = False
    words = R.tree_words(sees)
    if case["seq"] % 32:  # bits beyond the drafts are none
        words[..., -1] = (words[..., -1].view(np.uint32) | np.uint32(0xffffffff) << np.uint32(case["seq"] % 32)).view(np.int32)
    x["tree"] = words
    got = R.run(rt, {**base.tree_spec(case, dtype), "drafts_only": True}, x)
    base.check_tree(got, case, x, sees, dtype, weights=False)
    hk, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    added = np.zeros_like(x["weights"], np.float64)
    for b, n in enumerate(case["lengths"]):
        mask, live = np.concatenate([np.ones((case["seq"], n), bool), sees[b]], 1), slice(0, n + case["seq"])
        for h in range(hk):
            q = x["q"][b, h * group:(h + 1) * group].reshape(-1, case["dim"])
            p = R.attention(q, x["k"][b, h, live], x["v"][b, h, live], np.tile(mask, (group, 1)))[2]
            added[b, h, live] = p[np.tile(sees[b].any(-1), group)].sum(0)
    base.close(got["weights"].reshape(added.shape), x["weights"] + added, added, 2.0 ** -23, 2e-5 if dtype == "fp32" else 1e-4)


@pytest.mark.parametrize("path,counts", [([[1, 3, 0, 0], [2, 1, 0, 0]], [2, 2]), ([[1, 3, 0, 0], [0, 4, 0, 0]], [2, 2]), ([[1, 3, 0, 0], [-1, 1, 0, 0]], [2, 1]),
                                         ([[1, 3, 0, 0], [0, 0, 0, 0]], [2, 5]), ([[1, 3, 0, 0], [0, 0, 0, 0]], [2, -1])])
def test_commit_that_is_refused_moves_nothing(rt, path, counts):
    # a path that is none in one sequence: no other sequence's drafts move either, so that the
    # right commit that follows finds them where the step left them
    rng = np.random.default_rng(9)
    layer = make(rt, keep=16, recent=2)
    try:
        layer.step(rng.standard_normal((B, T, WIDTH)), np.tile(np.arange(T), (B, 1)))
        k = rt.download_f32(layer.k).reshape(B, HK, C, D)[:, :, :T].copy()
        weights = held_weights(rt, layer)
        with pytest.raises(jc.JadeError, match="path must ascend"):
            layer.commit(path, counts)
        np.testing.assert_array_equal(rt.download_f32(layer.k).reshape(B, HK, C, D)[:, :, :T], k)
        assert layer.commit([[1, 3, 0, 0], [1, 2, 0, 0]], [2, 2]).tolist() == [2, 2]
        for b, rows in enumerate(([1, 3], [1, 2])):
            np.testing.assert_array_equal(rt.download_f32(layer.k).reshape(B, HK, C, D)[b, :, :2], k[b][:, rows])
            np.testing.assert_array_equal(held_weights(rt, layer)[b, :, :2], weights[b][:, rows])
    finally:
        layer.release()
