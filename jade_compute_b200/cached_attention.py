"""An attention layer that serves from a key/value cache, from the operators of a
cached attention step (csrc/rope.cu, attention_tree*.cu, cache.cu):

  step      gemm               qkv = x Wqkv^T
            qk_norm_rope       head norms, rotary positions; keys and values to the cache
            attention_tree     the new tokens, a drafted tree or plain ones, over the cache
            gemm               y = out Wo^T + x
  commit    cache_commit       keeps the accepted tokens of the step
  evict     cache_evict        keeps the cache entries of largest attention weight

A step takes ``seq`` tokens of every sequence. Plain decoding is a tree of one token
(``seq=1``); a prompt goes in pieces of ``seq`` tokens, each seeing the ones before it
(``causal_tree``); speculative decoding passes a tree of drafts and commits the
accepted branch. The step's tokens stay behind the committed entries until ``commit``
names the ones to keep, so an uncommitted step is simply overwritten by the next. The
same holds for the accumulated weights: a step adds its own to those of the last commit.
A committed step counts whole, drafts that its commit leaves out included (they have
attended to the committed entries; their own entries go with them); places without a
draft count nothing.

Weights are FP32 host arrays in the reference's K x N layout; activations and the
cache are BF16 or FP16, sums FP32.
"""
from __future__ import annotations

import numpy as np

from .runtime import JR_EINVAL, JadeError, Runtime, f32_to_bf16


def tree_words(parents) -> np.ndarray:
    """Parents [batch, seq] of drafted tokens (index of the parent draft, -1 for none, -2
    for a place without a draft) -> attention_tree's bits [batch, seq, ceil(seq / 32)]."""
    parents = np.asarray(parents)
    batch, seq = parents.shape
    if (parents >= np.arange(seq)).any() or (parents < -2).any():
        raise ValueError("a draft's parent comes before it (or is -1: none, -2: no draft)")
    sees = np.zeros((batch, seq, 32 * (-(-seq // 32))), np.uint32)
    rows = np.arange(batch)
    for i in range(seq):
        p = parents[:, i]
        sees[:, i] = np.where((p >= 0)[:, None], sees[rows, np.maximum(p, 0)], 0)
        sees[:, i, i] = p != -2
    bits = sees.reshape(batch, seq, -1, 32) << np.arange(32, dtype=np.uint32)
    return bits.sum(-1, dtype=np.uint32).view(np.int32)


def causal_tree(batch: int, seq: int) -> np.ndarray:
    """Every token sees the ones before it: consecutive tokens of a text."""
    return tree_words(np.tile(np.arange(-1, seq - 1), (batch, 1)))


class CachedAttention:
    """One layer on one device. ``keep`` > 0 accumulates attention weights and
    allocates the second cache that ``evict`` moves entries into. ``rotation``: fields of
    the qk_norm_rope spec; ``norm=False`` for a layer without head norms."""

    def __init__(self, rt: Runtime, batch: int, seq: int, width: int, heads: int, kv_heads: int, dim: int, capacity: int,
                 dtype: str = "bf16", eps: float = 1e-6, keep: int = 0, recent: int = 0, **rotation):
        if dtype not in ("bf16", "fp16"):
            raise ValueError("dtype must be bf16 or fp16")
        if width % 8:
            raise ValueError("width must be a multiple of 8 (16-byte rows)")
        self.rt, self.batch, self.seq, self.width, self.heads, self.kv_heads, self.dim = rt, batch, seq, width, heads, kv_heads, dim
        self.capacity, self.dtype, self.keep = capacity, dtype, keep
        tokens, packed = batch * seq, (heads + 2 * kv_heads) * dim
        heads_of = {"batch": batch, "kv_heads": kv_heads, "dim": dim, "capacity": capacity, "dtype": dtype}
        gemm = {"op": "gemm", "tiled": True, "dtype": dtype, "out_dtype": dtype, "b_layout": "nk", "m": tokens}
        self.k_qkv = rt.compile({**gemm, "n": packed, "k": width})
        norm = rotation.get("norm", True)
        self.k_rope = rt.compile({"op": "qk_norm_rope", "seq": seq, "heads": heads, "epsilon": eps, **heads_of, **rotation})
        self.k_attend = rt.compile({"op": "attention_tree", "seq": seq, "heads": heads, "weights": keep > 0, **({"drafts_only": True} if keep else {}), **heads_of})
        self.k_out = rt.compile({**gemm, "n": width, "k": heads * dim, "epilogue": "residual"})
        self.k_commit = rt.compile({"op": "cache_commit", "seq": seq, "weights": keep > 0, **heads_of})
        self.kernels = [self.k_qkv, self.k_rope, self.k_attend, self.k_out, self.k_commit]

        def alloc(n, kind=dtype):
            return rt.alloc(n, kind)

        cache = batch * kv_heads * capacity
        self.x, self.y = alloc(tokens * width), alloc(tokens * width)
        self.wqkv, self.wo = alloc(packed * width), alloc(width * heads * dim)
        self.q_weight, self.k_weight = (alloc(dim), alloc(dim)) if norm else (None, None)
        self.norm_weights = [self.q_weight, self.k_weight] if norm else []
        self.qkv, self.q, self.out = alloc(tokens * packed), alloc(tokens * heads * dim), alloc(tokens * heads * dim)
        self.k, self.v = alloc(cache * dim), alloc(cache * dim)
        self.positions, self.tree = alloc(tokens, "i32"), alloc(tokens * (-(-seq // 32)), "i32")
        self.lengths, self.next_lengths = alloc(batch, "i32"), alloc(batch, "i32")
        self.path, self.counts = alloc(tokens, "i32"), alloc(batch, "i32")
        self.buffers = [self.x, self.y, self.wqkv, self.wo, *self.norm_weights, self.qkv, self.q, self.out, self.k, self.v, self.positions,
                        self.tree, self.lengths, self.next_lengths, self.path, self.counts]
        if keep:
            self.k_evict = rt.compile({"op": "cache_evict", "keep": keep, "recent": recent, **heads_of})
            self.kernels.append(self.k_evict)
            # the weights with those of the step that is not committed yet, as of the last commit, and the eviction's
            self.weights, self.committed_weights, self.next_weights = (alloc(cache, "fp32") for _ in range(3))
            self.k_copy = rt.compile({"op": "copy", "bytes": 4 * cache, "direction": "d2d"})
            self.kernels.append(self.k_copy)
            self.next_k, self.next_v, self.kept = alloc(cache * dim), alloc(cache * dim), alloc(batch * kv_heads * keep, "i32")
            self.buffers += [self.weights, self.committed_weights, self.next_weights, self.next_k, self.next_v, self.kept]
        rt.upload(self.tree, causal_tree(batch, seq))

    def release(self) -> None:
        """Frees the layer's buffers and kernels."""
        for b in self.buffers:
            b.free()
        for k in self.kernels:
            k.release()

    # -- jobs, for use in a larger batch
    def step_jobs(self):
        accumulated = [self.weights] if self.keep else []
        back = [(self.k_copy, [self.committed_weights, self.weights])] if self.keep else []
        return [*back, (self.k_qkv, [self.x, self.wqkv, self.qkv]),
                (self.k_rope, [self.qkv, *self.norm_weights, self.positions, self.lengths, self.q, self.k, self.v]),
                (self.k_attend, [self.q, self.k, self.v, self.lengths, self.tree, self.out, *accumulated]),
                (self.k_out, [self.out, self.wo, self.x, self.y])]

    def commit_jobs(self):
        accumulated = [self.weights] if self.keep else []
        hold = [(self.k_copy, [self.weights, self.committed_weights])] if self.keep else []
        return [(self.k_commit, [self.path, self.counts, self.lengths, self.k, self.v, *accumulated, self.next_lengths]), *hold]

    # -- host side
    def _to_dtype(self, x) -> np.ndarray:
        x = np.asarray(x, np.float32).ravel()
        return f32_to_bf16(x) if self.dtype == "bf16" else x.astype(np.float16)

    def load(self, wqkv, wo, q_weight=None, k_weight=None) -> None:
        """wqkv [width, (heads + 2 kv_heads) dim], wo [heads dim, width], norm weights [dim]
        (none for a layer without head norms)."""
        weights = [w for w in (q_weight, k_weight) if w is not None]
        if len(weights) != len(self.norm_weights):
            raise ValueError(f"this layer has {len(self.norm_weights)} norm weights, not {len(weights)}")
        self.rt.upload(self.wqkv, self._to_dtype(np.asarray(wqkv, np.float32).reshape(self.width, -1).T))
        self.rt.upload(self.wo, self._to_dtype(np.asarray(wo, np.float32).reshape(-1, self.width).T))
        for buf, weight in zip(self.norm_weights, weights):
            self.rt.upload(buf, self._to_dtype(weight))

    def step(self, x, positions, tree=None) -> np.ndarray:
        """x [batch, seq, width], positions [batch, seq]; tree: bits as tree_words gives them
        (kept from the last step when omitted). Returns y as FP32."""
        self.rt.upload(self.x, self._to_dtype(x))
        self.rt.upload(self.positions, np.asarray(positions, np.int32).ravel())
        if tree is not None:
            self.rt.upload(self.tree, np.asarray(tree, np.int32).ravel())
        self.rt.execute(self.step_jobs())
        return self.rt.download_f32(self.y).reshape(self.batch, self.seq, self.width)

    def commit(self, path=None, counts=None) -> np.ndarray:
        """Keeps drafts path[b, :counts[b]] (ascending) of the last step, all of them by
        default. Returns the sequences' new lengths."""
        everything = np.tile(np.arange(self.seq), (self.batch, 1))
        path = np.asarray(everything if path is None else path, np.int32).reshape(self.batch, self.seq)
        counts = np.full(self.batch, self.seq, np.int32) if counts is None else np.asarray(counts, np.int32).reshape(self.batch)
        # refused here for all sequences: the operator leaves out a bad one and moves the others
        taken = np.arange(self.seq) < counts[:, None]
        ascends = np.diff(path, axis=1, prepend=-1) > 0
        if (counts < 0).any() or (counts > self.seq).any() or not ascends[taken].all() or (path[taken] >= self.seq).any():
            raise JadeError(JR_EINVAL, "commit: a path must ascend within the step's tokens, its count be at most their number")
        self.rt.upload(self.path, path.ravel())
        self.rt.upload(self.counts, counts)
        self.rt.execute(self.commit_jobs())
        self.lengths, self.next_lengths = self.next_lengths, self.lengths
        return self.rt.download(self.lengths)

    def evict(self) -> np.ndarray:
        """Keeps ``keep`` committed entries a head, by their weights as of the last commit.
        Returns the slots that they had [batch, kv_heads, keep], -1 where a sequence has fewer."""
        if not self.keep:
            raise ValueError("this layer accumulates no weights (keep=0)")
        self.rt.execute([(self.k_evict, [self.k, self.v, self.committed_weights, self.lengths, self.next_k, self.next_v, self.next_weights, self.kept,
                                         self.next_lengths]), (self.k_copy, [self.next_weights, self.committed_weights])])
        for name in ("k", "v", "weights", "lengths"):
            new = "next_" + name
            old = getattr(self, name)
            setattr(self, name, getattr(self, new))
            setattr(self, new, old)
        return self.rt.download(self.kept).reshape(self.batch, self.kv_heads, self.keep)
