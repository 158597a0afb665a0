"""Plain 64-bit (numpy) statements of the cached attention operators, written from
their formulas, and a runner that takes a spec and named arrays through the
public API. Used by the tests only."""
import numpy as np

import jade_compute_b200 as jc

ROUNDOFF = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -23}


def rounded(x, dtype):
    """x as the type holds it, widened to 64 bits."""
    x = np.asarray(x, np.float32)
    if dtype == "bf16":
        return jc.bf16_to_f32(jc.f32_to_bf16(x.ravel())).reshape(x.shape).astype(np.float64)
    return x.astype(np.float16 if dtype == "fp16" else np.float32).astype(np.float64)


def run(rt, spec, arrays, repeats=1):
    """Outputs by binding name, in 64 bits (whole numbers as int64), from one batch of `repeats`."""
    kernel = rt.compile(spec)
    buffers = []
    try:
        for b in kernel.info["bindings"]:
            buf = rt.alloc(b["elements"], b["dtype"])
            buffers.append(buf)
            if b["name"] in arrays:
                x = np.asarray(arrays[b["name"]]).ravel()
                rt.upload(buf, x if b["dtype"] == "i32" else jc.f32_to_bf16(x.astype(np.float32)) if b["dtype"] == "bf16" else x)
        rt.execute([(kernel, buffers)], repeats=repeats)
        out = {}
        for b, buf in zip(kernel.info["bindings"], buffers):
            if b["write"]:
                out[b["name"]] = rt.download(buf).astype(np.int64) if b["dtype"] == "i32" else rt.download_f32(buf).astype(np.float64)
        return out
    finally:
        for buf in buffers:
            buf.free()
        kernel.release()


def frequencies(rotary, base=10000.0, scaling="none", factor=1.0, original=0):
    i = np.arange(rotary // 2)
    if scaling == "ntk":
        base = base * factor ** (rotary / (rotary - 2))
    theta = base ** (-2.0 * i / rotary)
    gain = 1.0
    if scaling == "linear":
        theta = theta / factor
    if scaling == "yarn":
        keep = np.clip((original * theta / (2 * np.pi) - 1) / 31, 0, 1)
        theta = keep * theta + (1 - keep) * theta / factor
        gain = 0.1 * np.log(factor) + 1
    return theta, gain


def turn(x, positions, spec, sign=1.0):
    """x [..., dim] with positions broadcast over its leading axes, turned; and the bound's magnitude |a cos| + |b sin|."""
    R = spec.get("rotary", spec["dim"])
    theta, gain = frequencies(R, spec.get("base", 10000.0), spec.get("scaling", "none"), spec.get("factor", 1.0), spec.get("original", 0))
    angle = np.asarray(positions, np.float64)[..., None] * theta
    c, s = gain * np.cos(angle), sign * gain * np.sin(angle)
    a, b = (slice(0, R, 2), slice(1, R, 2)) if spec.get("interleaved") else (slice(0, R // 2), slice(R // 2, R))
    y, m = x.copy(), np.abs(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    m[..., a] = m[..., b] = gain * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, m


def norm_rope(spec, x):
    """(values, magnitudes) of q [B, H, T, D], k, v [B, T, Hk, D] for qkv [B, T, H + 2 Hk, D]."""
    H, Hk = spec["heads"], spec["kv_heads"]
    q, k, v = np.split(x["qkv"], [H, H + Hk], axis=2)
    if spec.get("norm", True):
        q = q / np.sqrt((q * q).mean(-1, keepdims=True) + spec["epsilon"]) * x["q_weight"]
        k = k / np.sqrt((k * k).mean(-1, keepdims=True) + spec["epsilon"]) * x["k_weight"]
    at = x["positions"][:, :, None]
    return turn(q, at, spec), turn(k, at, spec), (v, np.abs(v))


def attention(q, k, v, sees):
    """q [M, D], k, v [N, D], sees [M, N] -> out [M, D], sum p |v|, p [M, N]; rows that see nothing are 0."""
    s = np.where(sees, q @ np.where(sees.any(0)[:, None], k, 0).T / np.sqrt(q.shape[1]), -np.inf)
    top = s.max(-1, keepdims=True)
    p = np.exp(s - np.where(np.isfinite(top), top, 0))
    p = np.where(sees, p, 0)
    total = p.sum(-1, keepdims=True)
    p = p / np.where(total > 0, total, 1)
    vv = np.where(sees.any(0)[:, None], v, 0)
    return p @ vv, p @ np.abs(vv), p


def tree_words(sees):
    """[B, T, T] bools -> [B, T, ceil(T / 32)] int32 words."""
    B, T, _ = sees.shape
    W = -(-T // 32)
    bits = np.zeros((B, T, W * 32), np.uint32)
    bits[:, :, :T] = sees
    return (bits.reshape(B, T, W, 32) << np.arange(32, dtype=np.uint32)).sum(-1, dtype=np.uint32).view(np.int32)


def random_tree(rng, B, T):
    sees = np.zeros((B, T, T), bool)
    for b in range(B):
        for i in range(T):
            if i and rng.random() < 0.9:
                sees[b, i] = sees[b, rng.integers(i)]
            sees[b, i, i] = True
    return sees
