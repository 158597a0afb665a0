"""CachedAttention: the tree helper on the CPU; on the GPU a run of steps as a server
would make them (prompt pieces, drafted trees, commits, an eviction), every stage
checked against 64 bits on the buffers that it read (tolerances: tests/test_gpu_cached_attention.py;
products: 2 K 2^-24 of the sum of magnitudes for FP32 accumulation, and the output's rounding)."""
import numpy as np
import pytest

import jade_compute_b200 as jc
from jade_compute_b200.cached_attention import CachedAttention, causal_tree, tree_words
from tests import cached_reference as R


def test_tree_words():
    words = tree_words([[-1, 0, 0, 1, -2, 3]])
    assert words.shape == (1, 6, 1) and words[0, :, 0].tolist() == [1, 3, 5, 11, 0, 43]
    wide = causal_tree(2, 70).view(np.uint32)
    assert wide.shape == (2, 70, 3) and wide[1, 69].tolist() == [2 ** 32 - 1, 2 ** 32 - 1, 63] and wide[0, 31].tolist() == [2 ** 32 - 1, 0, 0]
    for bad in ([[0]], [[-1, 1]], [[-3]]):
        with pytest.raises(ValueError):
            tree_words(bad)


def near(got, ref, bound):
    assert (np.abs(got - ref) <= bound).all(), np.max(np.abs(got - ref) - bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rotation", [("bf16", {}), ("fp16", {"rotary": 16, "interleaved": True, "scaling": "linear", "factor": 2.0})])
def test_serving_steps(dtype, rotation):
    B, T, width, H, Hk, D, C, keep, recent = 3, 5, 64, 6, 2, 32, 160, 60, 8
    rt = jc.Runtime(0)
    layer = CachedAttention(rt, B, T, width, H, Hk, D, C, dtype=dtype, keep=keep, recent=recent, **rotation)
    rng = np.random.default_rng(1)
    u = R.ROUNDOFF[dtype]
    w = {"wqkv": R.rounded(0.2 * rng.standard_normal((width, (H + 2 * Hk) * D)), dtype), "wo": R.rounded(0.2 * rng.standard_normal((H * D, width)), dtype),
         "q_weight": R.rounded(1 + 0.1 * rng.standard_normal(D), dtype), "k_weight": R.rounded(1 + 0.1 * rng.standard_normal(D), dtype)}
    layer.load(*w.values())
    spec = {"heads": H, "kv_heads": Hk, "dim": D, "epsilon": 1e-6, **rotation}

    def fetch(buf, *shape):
        return rt.download_f32(buf).astype(np.float64).reshape(shape)

    def product(got, a, b, more=0.0):
        k = a.shape[-1]
        near(got, a @ b + more, u * np.abs(a @ b + more) + 2 * k * 2.0 ** -24 * (np.abs(a) @ np.abs(b) + np.abs(more)))

    try:
        lengths, position, expected = np.zeros(B, int), np.zeros(B, int), np.zeros((B, Hk, C))
        for n in range(24):
            x = R.rounded(rng.standard_normal((B, T, width)), dtype)
            if n < 20:  # prompt pieces
                sees, at = np.tile(np.tril(np.ones((T, T), bool)), (B, 1, 1)), position[:, None] + np.arange(T)
                counts = np.array([T, T, T - n % 2])  # one sequence drops the last token of every other piece
                path = np.tile(np.arange(T), (B, 1))
            else:  # drafted trees
                sees = R.random_tree(rng, B, T)
                at = position[:, None] + sees.sum(-1) - 1
                counts = rng.integers(0, T + 1, B)
                path = np.stack([np.sort(rng.permutation(T)) for _ in range(B)])
                for b in range(B):
                    path[b, :counts[b]] = np.sort(rng.permutation(T)[:counts[b]])
            y = layer.step(x, at, R.tree_words(sees)).astype(np.float64)
            qkv = fetch(layer.qkv, B, T, H + 2 * Hk, D)
            product(qkv.reshape(B, T, -1), x, w["wqkv"])
            (q, mq), (k, mk), (v, _) = R.norm_rope(spec, {"qkv": qkv, "positions": at, **w})
            gq, gk, gv = fetch(layer.q, B, H, T, D), fetch(layer.k, B, Hk, C, D), fetch(layer.v, B, Hk, C, D)
            tiny = 2.0 ** -25 if dtype == "fp16" else 0.0
            near(gq, q.transpose(0, 2, 1, 3), np.maximum(u * np.abs(q), tiny).transpose(0, 2, 1, 3) + 4e-6 * mq.transpose(0, 2, 1, 3))
            out, added = fetch(layer.out, B, T, H, D), np.zeros((B, Hk, C))
            for b in range(B):
                rows = slice(lengths[b], lengths[b] + T)
                near(gk[b, :, rows], k[b].transpose(1, 0, 2), np.maximum(u * np.abs(k[b]), tiny).transpose(1, 0, 2) + 4e-6 * mk[b].transpose(1, 0, 2))
                np.testing.assert_array_equal(gv[b, :, rows], v[b].transpose(1, 0, 2))
                mask = np.concatenate([np.ones((T, lengths[b]), bool), sees[b]], 1)
                for h in range(Hk):
                    heads = slice(h * H // Hk, (h + 1) * H // Hk)
                    live = slice(0, lengths[b] + T)
                    o, m, p = R.attention(gq[b, heads].reshape(-1, D), gk[b, h, live], gv[b, h, live], np.tile(mask, (H // Hk, 1)))
                    o, m = (z.reshape(H // Hk, T, D).transpose(1, 0, 2) for z in (o, m))
                    near(out[b, :, heads], o, np.maximum(u * np.abs(o), tiny) + (u + 1e-4) * m)
                    added[b, h, live] = p.sum(0)
            product(y, out.reshape(B, T, -1), w["wo"], x)
            expected += added
            near(fetch(layer.weights, B, Hk, C), expected, 1e-4 * expected + 1e-6)
            assert layer.commit(path, counts).tolist() == (lengths + counts).tolist()
            for b in range(B):
                a = counts[b]
                moved = expected[b][:, lengths[b] + path[b, :a]].copy()
                expected[b][:, lengths[b]:lengths[b] + T] = 0
                expected[b][:, lengths[b]:lengths[b] + a] = moved
            lengths, position = lengths + counts, position + counts
            if n == 21:
                old_k = fetch(layer.k, B, Hk, C, D)
                held = fetch(layer.weights, B, Hk, C)
                kept = layer.evict()
                assert (np.minimum(lengths, keep) == rt.download(layer.lengths)).all()
                for b in range(B):
                    for h in range(Hk):
                        slots = kept[b, h][kept[b, h] >= 0]
                        assert len(slots) == min(lengths[b], keep) and (np.diff(slots) > 0).all()
                        assert set(range(lengths[b] - recent, lengths[b])) <= set(slots.tolist())
                        older = np.delete(np.arange(lengths[b]), slots)
                        others = slots[slots < lengths[b] - recent]
                        assert not len(older) or held[b, h, older].max() <= held[b, h, others].min()
                        np.testing.assert_array_equal(fetch(layer.k, B, Hk, C, D)[b, h, :len(slots)], old_k[b, h, slots])
                        expected[b, h] = 0
                        expected[b, h, :len(slots)] = held[b, h, slots]
                lengths = np.minimum(lengths, keep)
    finally:
        layer.release()
        rt.close()


@pytest.mark.gpu
def test_layer_refusals():
    rt = jc.Runtime(0)
    try:
        with pytest.raises(ValueError, match="dtype"):
            CachedAttention(rt, 1, 1, 64, 2, 1, 32, 16, dtype="fp32")
        with pytest.raises(ValueError, match="width"):
            CachedAttention(rt, 1, 1, 60, 2, 1, 32, 16)
        with pytest.raises(jc.JadeError, match="multiple of kv_heads"):
            CachedAttention(rt, 1, 1, 64, 3, 2, 32, 16)
        layer = CachedAttention(rt, 1, 1, 64, 2, 1, 32, 1)
        with pytest.raises(ValueError, match="keep=0"):
            layer.evict()
        layer.step(np.zeros((1, 1, 64)), [[0]])
        layer.commit()
        with pytest.raises(jc.JadeError, match="cache length"):  # the cache is full
            layer.step(np.zeros((1, 1, 64)), [[1]])
        layer.release()
    finally:
        rt.close()
