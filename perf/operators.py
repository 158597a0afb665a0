"""The operators of a cached attention step, each in its plain form (elementary
torch operations in 32 bits) and as a call of this framework.

    qk_norm_rope       a projection's packed [q | k | v] rows: RMS norm of every query
                       and key head, position rotation, queries to [batch, heads, seq,
                       dim], keys and values to their slots of the cache
    qk_norm_rope_grad  its gradient: of the packed rows and of the two norm weights
    attention_tree     attention of a sequence's newest tokens (one, or a tree of
                       drafted ones) over its cache, with the weight that each cached
                       key received
    cache_evict        the cache entries with the largest accumulated weight, moved
                       together into another cache
    cache_commit       the accepted branch of a drafted tree, moved behind the
                       committed cache entries

Layouts: qkv [batch, seq, heads + 2 kv_heads, dim]; q [batch, heads, seq, dim];
k, v [batch, kv_heads, capacity, dim]; out [batch, seq, heads, dim]; weights
[batch, kv_heads, capacity]; one cache length per sequence.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token for each of 8 sequences behind its projection: all latency
        rope("rope_token", batch=8, seq=1, heads=32, kv_heads=8, dim=128, capacity=512, start=400),
        # a prompt batch of 4 x 2048 tokens, the shape that the framework's own prompt attention runs
        rope("rope_prompt", batch=4, seq=2048, heads=16, kv_heads=16, dim=128),
        # the same batch in training
        rope("rope_train_grad", op="qk_norm_rope_grad", batch=4, seq=2048, heads=16, kv_heads=16, dim=128),
        # a ragged training batch in half precision: part of the head rotated in neighbouring
        # pairs, frequencies scaled for a context eight times longer
        rope("rope_ragged_grad", op="qk_norm_rope_grad", batch=3, seq=511, heads=12, kv_heads=4, dim=96, dtype="fp16",
             rotary=40, interleaved=True, scaling="yarn", factor=8.0, start=30000),
        # serving: 16 sequences of 1,000 to 8,000 tokens, one new token each
        tree("tree_token", batch=16, seq=1, heads=32, kv_heads=8, dim=128, capacity=8192, shortest=1000, longest=8000),
        # 4 sequences that verify 32 drafted tokens each and keep the keys' weights for the eviction
        tree("tree_draft", batch=4, seq=32, heads=32, kv_heads=8, dim=128, capacity=16384, shortest=9000, longest=16000,
             weights=True),
        # one long document in half precision with a tree of 64 drafted tokens
        tree("tree_long", batch=1, seq=64, heads=32, kv_heads=8, dim=128, capacity=131072, shortest=130987, longest=130987,
             dtype="fp16"),
        # short ragged sequences in single precision, one of them empty, odd sizes throughout
        tree("tree_ragged", batch=3, seq=7, heads=6, kv_heads=2, dim=80, capacity=611, shortest=0, longest=600, dtype="fp32",
             weights=True),
        # one step of a small model's cache, from about 500 entries down to 257
        evict("evict_small", batch=2, kv_heads=2, dim=80, capacity=611, shortest=500, longest=600, keep=257, recent=16,
              dtype="fp32"),
        # 8 sequences of up to 8192 entries down to 2048
        evict("evict_batch", batch=8, kv_heads=8, dim=128, capacity=8192, shortest=1500, longest=8192, keep=2048, recent=128),
        # a few accepted tokens of one sequence's tree
        commit("commit_one", batch=1, kv_heads=8, dim=128, seq=16, capacity=1024, shortest=700, longest=700),
        # 32 sequences with trees of 64 tokens in half precision
        commit("commit_batch", batch=32, kv_heads=8, dim=64, seq=64, capacity=1024, shortest=0, longest=960, dtype="fp16",
               weights=True),
    ]


def rope(name, op="qk_norm_rope", *, batch, seq, heads, kv_heads, dim, rotary=None, interleaved=False, scaling="none", factor=1.0,
         original=4096, base=10000.0, norm=True, capacity=0, start=0, dtype="bf16"):
    """capacity 0: keys and values of these tokens alone. start: the first position (and, with a cache, about the slot)."""
    return dict(name=name, op=op, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, rotary=dim if rotary is None else rotary,
                interleaved=interleaved, scaling=scaling, factor=factor, original=original, base=base, norm=norm, capacity=capacity,
                start=start, dtype=dtype)


def tree(name, *, batch, seq, heads, kv_heads, dim, capacity, shortest, longest, weights=False, dtype="bf16"):
    return dict(name=name, op="attention_tree", batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, capacity=capacity,
                shortest=shortest, longest=longest, weights=weights, dtype=dtype)


def evict(name, *, batch, kv_heads, dim, capacity, shortest, longest, keep, recent, dtype="bf16"):
    return dict(name=name, op="cache_evict", batch=batch, kv_heads=kv_heads, dim=dim, capacity=capacity, shortest=shortest,
                longest=longest, keep=keep, recent=recent, dtype=dtype)


def commit(name, *, batch, kv_heads, dim, seq, capacity, shortest, longest, weights=False, dtype="bf16"):
    return dict(name=name, op="cache_commit", batch=batch, kv_heads=kv_heads, dim=dim, seq=seq, capacity=capacity, shortest=shortest,
                longest=longest, weights=weights, dtype=dtype)


def draw(rng):
    def spread(low, high):
        return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))

    def sizes():
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        return dict(heads=kv_heads * rng.choice([1, 2, 3, 4, 7, 8]), kv_heads=kv_heads, dim=rng.choice([64, 128, 128, 8 * rng.randint(4, 16)]),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))

    op = rng.choice(["qk_norm_rope", "qk_norm_rope_grad", "attention_tree", "attention_tree", "cache_evict", "cache_commit"])
    s = sizes()
    if op.startswith("qk_norm_rope"):
        batch = spread(1, 32)
        most = 4 * 2048 * 48 * 128 // (2 if s["dtype"] == "fp32" else 1)
        seq = spread(1, max(1, min(4096, most // (batch * (s["heads"] + 2 * s["kv_heads"]) * s["dim"]))))
        cached = op == "qk_norm_rope" and seq <= 512 and rng.random() < 0.6
        scaling = rng.choice(["none", "none", "linear", "ntk", "yarn"])
        c = rope("", op=op, batch=batch, seq=seq, rotary=s["dim"] if rng.random() < 0.5 else 2 * rng.randint(2, s["dim"] // 2),
                 interleaved=rng.random() < 0.4, scaling=scaling, factor=1.0 if scaling == "none" else float(rng.choice([2, 4, 8.5])),
                 base=rng.choice([10000.0, 500000.0]), norm=rng.random() < 0.8, capacity=seq + spread(1, 300) if cached else 0,
                 start=spread(1, 100000), **s)
    elif op == "attention_tree":
        batch, seq = spread(1, 24), rng.choice([1, spread(2, 128)])
        capacity = max(seq + 1, min(131072, spread(64, 131072 * 8 * 128 // (2 * batch * s["kv_heads"] * s["dim"]))))
        rows = seq * s["heads"] // s["kv_heads"]
        capacity = max(seq + 1, min(capacity, 131072 * 8 * 256 * 128 // (2 * batch * s["kv_heads"] * rows * s["dim"])))
        if s["dtype"] == "fp32":  # without the tensor cores the products count eight-fold
            capacity = max(seq + 1, capacity // 8)
        longest = capacity - seq
        c = tree("", batch=batch, seq=seq, capacity=capacity, longest=longest, shortest=rng.randint(0, longest), weights=rng.random() < 0.5, **s)
    else:
        batch = spread(1, 32)
        del s["heads"]
        capacity = min(65536, spread(160, 2 ** 26 // (batch * s["kv_heads"] * s["dim"])))
        if op == "cache_evict":
            keep = spread(1, capacity)
            longest = rng.randint(capacity // 2, capacity)
            c = evict("", batch=batch, capacity=capacity, longest=longest, shortest=rng.randint(0, longest), keep=keep, recent=rng.randint(0, min(keep, 256)), **s)
        else:
            seq = spread(1, 128)
            longest = capacity - seq
            c = commit("", batch=batch, seq=seq, capacity=capacity, longest=longest, shortest=rng.randint(0, longest), weights=rng.random() < 0.5, **s)
    del c["name"]
    return c


def lengths_of(case):
    """The sequences' cache lengths, from the shortest to the longest in equal steps."""
    n = max(1, case["batch"] - 1)
    return [case["longest"] - (case["longest"] - case["shortest"]) * i // n for i in range(case["batch"])]


# ------------------------------------------------------------------ inputs
def spec(case):
    """The framework's kernel spec of a case."""
    s = {k: case[k] for k in ("op", "batch", "kv_heads", "dim", "dtype")}
    for k in ("seq", "heads", "keep", "recent", "weights"):
        if k in case:
            s[k] = case[k]
    if case.get("capacity"):
        s["capacity"] = case["capacity"]
    if case["op"].startswith("qk_norm_rope"):
        for k in ("rotary", "interleaved", "base", "norm"):
            s[k] = case[k]
        if case["norm"]:
            s["epsilon"] = 1e-6
        if case["scaling"] != "none":
            s |= {"scaling": case["scaling"], "factor": case["factor"]}
            if case["scaling"] == "yarn":
                s["original"] = case["original"]
    return s


OUTPUTS = {
    "qk_norm_rope": ("q", "k", "v"),
    "qk_norm_rope_grad": ("dqkv", "dq_weight", "dk_weight"),
    "attention_tree": ("out", "weights"),
    "cache_evict": ("k_out", "v_out", "weights_out", "kept", "lengths_out"),
    "cache_commit": ("k", "v", "weights", "lengths_out"),
}


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    t = TYPES[case["dtype"]]
    B, H, D, T, C = case["batch"], case["kv_heads"], case["dim"], case.get("seq", 0), case.get("capacity", 0)

    def normal(*shape, scale=1.0, mean=0.0):
        x = torch.empty(shape, dtype=t, device="cuda")
        return x.normal_(mean, scale, generator=g)

    def gamma_like(*shape):  # accumulated attention weights: positive, a few large
        return torch.empty(shape, device="cuda").log_normal_(-2.0, 1.5, generator=g)

    def whole(values):
        return torch.as_tensor(values, dtype=torch.int32).cuda()

    x = {}
    if case["op"].startswith("qk_norm_rope"):
        Q, rows = case["heads"], C or T
        x["qkv"] = normal(B, T, Q + 2 * H, D, scale=1.5)
        if case["norm"]:
            x["q_weight"], x["k_weight"] = normal(D, scale=0.2, mean=1.0), normal(D, scale=0.2, mean=1.0)
        first = case["start"] + torch.randint(0, 50, (B, 1), generator=host)
        x["positions"] = whole(first + torch.arange(T))
        if case["op"] == "qk_norm_rope":
            if C:
                x["starts"] = whole(torch.randint(0, C - T + 1, (B,), generator=host))
            x["q"] = torch.zeros(B, Q, T, D, dtype=t, device="cuda")
            x["k"], x["v"] = (normal(B, H, rows, D) if C else torch.zeros(B, H, rows, D, dtype=t, device="cuda") for _ in range(2))
        else:
            x["dq"], x["dk"], x["dv"] = normal(B, Q, T, D), normal(B, H, T, D), normal(B, H, T, D)
            x["dqkv"] = torch.zeros_like(x["qkv"])
            if case["norm"]:
                x["dq_weight"], x["dk_weight"] = torch.zeros(D, device="cuda"), torch.zeros(D, device="cuda")
    else:
        order = torch.randperm(B, generator=host)
        lengths = torch.tensor(lengths_of(case))[order]
        x["lengths"] = whole(lengths)
        x["k"], x["v"] = normal(B, H, C, D), normal(B, H, C, D)
        if case["op"] == "cache_evict" or case["weights"]:
            x["weights"] = gamma_like(B, H, C)
        if case["op"] == "attention_tree":
            x["q"] = normal(B, case["heads"], T, D)
            x["tree"] = whole(draft_trees(B, T, host))
            x["out"] = torch.zeros(B, T, case["heads"], D, dtype=t, device="cuda")
        elif case["op"] == "cache_evict":
            x["k_out"], x["v_out"] = torch.zeros_like(x["k"]), torch.zeros_like(x["v"])
            x["weights_out"] = torch.zeros_like(x["weights"])
            x["kept"] = torch.zeros(B, H, case["keep"], dtype=torch.int32, device="cuda")
            x["lengths_out"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        else:  # the accepted tokens of each sequence, parents before children
            counts = torch.randint(0, T + 1, (B,), generator=host)
            taken = torch.rand(B, T, generator=host).argsort(dim=1)
            path = torch.where(torch.arange(T) < counts[:, None], taken, T).sort(dim=1).values
            x["path"], x["counts"] = whole(path.clamp(max=T - 1)), whole(counts)
            x["lengths_out"] = torch.zeros(B, dtype=torch.int32, device="cuda")
    return {"case": case, "x": x} if not own else framework_state(case, x)


def draft_trees(B, T, host):
    """[B, T, ceil(T / 32)] words: bit j of token i says that i sees drafted token j, itself
    and its ancestors. A sequence may have fewer drafts than T: the rest see none of them."""
    parent = (torch.rand(B, T, generator=host) * torch.arange(T).clamp(min=1)).long()
    sees = torch.zeros(B, T, T, dtype=torch.bool)
    for i in range(T):
        if i:
            sees[:, i] = sees[torch.arange(B), parent[:, i]]
        sees[:, i, i] = True
    drafts = torch.randint(max(1, T // 2), T + 1, (B,), generator=host)
    sees &= (torch.arange(T) < drafts[:, None])[:, :, None]
    W = -(-T // 32)
    bits = torch.nn.functional.pad(sees, (0, 32 * W - T)).view(B, T, W, 32).long()
    words = (bits << torch.arange(32)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words)


class Span:
    """A framework buffer as torch sees device memory; it keeps the buffer alive."""

    def __init__(self, buffer):
        kind, size = {"bf16": ("<i2", 2), "fp16": ("<f2", 2), "fp32": ("<f4", 4), "i32": ("<i4", 4)}[buffer.dtype]
        self.buffer = buffer
        self.__cuda_array_interface__ = {"shape": (buffer.nbytes // size,), "typestr": kind, "data": (buffer.ptr, False), "version": 3}


def framework_state(case, x):
    """What a program of this framework keeps: a runtime, the compiled kernel and its buffers."""
    import jade_compute_b200 as jc

    rt = jc.Runtime(0)
    kernel = rt.compile(spec(case))
    buffers, views = [], {}
    for b in kernel.info["bindings"]:
        buffers.append(rt.alloc(b["elements"], b["dtype"]))
        source = x[b["name"]]
        views[b["name"]] = torch.as_tensor(Span(buffers[-1]), device="cuda").view(source.dtype).view(source.shape)
        views[b["name"]].copy_(source)
    torch.cuda.synchronize()  # the runtime works on a stream of its own
    return {"rt": rt, "jobs": [(kernel, buffers)], "out": {n: views[n] for n in OUTPUTS[case["op"]] if n in views}}


def run(state):
    if own:
        state["rt"].execute(state["jobs"])
        return state["out"]
    return PLAIN[state["case"]["op"]](state["case"], state["x"])


# ------------------------------------------------------------------ plain forms
def rotation(case, positions):
    """cos and sin [..., 1, rotary / 2] of the positions' angles. The angle is reduced to one turn in 64 bits: in 32 bits
    the product of a position of 100,000 and a frequency is already off by 0.004."""
    R = case["rotary"]
    pair = torch.arange(R // 2, device="cuda", dtype=torch.float64)
    size, magnitude = case["base"], 1.0
    if case["scaling"] == "ntk":
        size = size * case["factor"] ** (R / (R - 2))
    frequency = size ** (-2 * pair / R)
    if case["scaling"] == "linear":
        frequency = frequency / case["factor"]
    if case["scaling"] == "yarn":
        kept = ((case["original"] * frequency / (2 * math.pi) - 1) / 31).clamp(0, 1)
        frequency = frequency * kept + frequency / case["factor"] * (1 - kept)
        magnitude = 0.1 * math.log(case["factor"]) + 1
    turns = positions.double()[..., None] * (frequency / (2 * math.pi))
    angle = ((turns - turns.floor()) * (2 * math.pi)).float()[..., None, :]
    return angle.cos() * magnitude, angle.sin() * magnitude


def rotate(case, x, cos, sin):
    """The first `rotary` elements of each head turned by the angles, in pairs of neighbours or of halves."""
    R = case["rotary"]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if case["interleaved"] else (x[..., : R // 2], x[..., R // 2 : R])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., R:]), -1)


def plain_rope(case, x):
    Q, H, D, t = case["heads"], case["kv_heads"], case["dim"], x["qkv"].dtype
    q, k, v = x["qkv"].float().split((Q, H, H), 2)
    if case["norm"]:
        q = q * (q.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * x["q_weight"].float()
        k = k * (k.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * x["k_weight"].float()
    cos, sin = rotation(case, x["positions"])
    q, k = rotate(case, q, cos, sin), rotate(case, k, cos, sin)
    x["q"].copy_(q.transpose(1, 2))
    slots = torch.arange(case["seq"], device="cuda") + (x["starts"].long()[:, None] if case["capacity"] else 0)
    batch = torch.arange(case["batch"], device="cuda")[:, None]
    slots = slots.expand(case["batch"], -1)
    x["k"][batch, :, slots] = k.to(t)
    x["v"][batch, :, slots] = v.to(t)
    return {n: x[n] for n in OUTPUTS["qk_norm_rope"]}


def plain_rope_grad(case, x):
    Q, H, t = case["heads"], case["kv_heads"], x["qkv"].dtype
    q, k, _ = x["qkv"].float().split((Q, H, H), 2)
    cos, sin = rotation(case, x["positions"])
    dq = rotate(case, x["dq"].float().transpose(1, 2), cos, -sin)
    dk = rotate(case, x["dk"].float().transpose(1, 2), cos, -sin)
    out = {}
    if case["norm"]:
        dq, out["dq_weight"] = norm_grad(q, x["q_weight"].float(), dq)
        dk, out["dk_weight"] = norm_grad(k, x["k_weight"].float(), dk)
    out["dqkv"] = torch.cat((dq, dk, x["dv"].float().transpose(1, 2)), 2).to(t)
    return out


def norm_grad(x, weight, dy):
    scale = (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    unit = x * scale
    d = dy * weight
    return (d - unit * (d * unit).mean(-1, keepdim=True)) * scale, (dy * unit).sum((0, 1, 2))


def plain_tree(case, x):
    B, H, T, C, D = (case[n] for n in ("batch", "kv_heads", "seq", "capacity", "dim"))
    Q = case["heads"]
    G = Q // H
    slot = torch.arange(C, device="cuda")
    draft = slot - x["lengths"].long()[:, None]  # [B, C]: which drafted token a slot holds
    bits = ((x["tree"][..., None] >> torch.arange(32, device="cuda")) & 1).view(B, T, -1)
    drafted = bits.gather(2, draft.clamp(0, T - 1)[:, None, :].expand(B, T, C)) > 0
    live = draft < T
    sees = ((draft < 0)[:, None] | (drafted & (draft >= 0)[:, None])) & live[:, None]  # [B, T, C]
    sees = sees[:, None].expand(B, G, T, C).reshape(B, 1, G * T, C)
    s = x["q"].float().view(B, H, G * T, D) @ x["k"].float().transpose(2, 3) * (1 / math.sqrt(D))
    s = torch.where(sees, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - torch.where(top > -math.inf, top, 0)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1)
    o = p @ torch.where(live[:, None, :, None], x["v"].float(), 0)
    out = {"out": o.view(B, Q, T, D).transpose(1, 2).to(x["q"].dtype)}
    if case["weights"]:
        out["weights"] = x["weights"].add_(p.sum(2))
    return out


def plain_evict(case, x):
    B, H, C, keep = (case[n] for n in ("batch", "kv_heads", "capacity", "keep"))
    slot = torch.arange(C, device="cuda")
    length = x["lengths"].long()[:, None, None]
    rank = torch.where(slot < length, x["weights"], -1.0)
    rank = torch.where((slot >= length - case["recent"]) & (slot < length), math.inf, rank)
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(dim=-1).values
    count = length.clamp(max=keep)
    new = torch.arange(keep, device="cuda")
    live = new < count  # [B, 1, keep]
    rows = kept[..., None].expand(B, H, keep, case["dim"])
    x["k_out"][:, :, :keep] = torch.where(live[..., None], x["k"].gather(2, rows), x["k_out"][:, :, :keep])
    x["v_out"][:, :, :keep] = torch.where(live[..., None], x["v"].gather(2, rows), x["v_out"][:, :, :keep])
    x["weights_out"].zero_()
    x["weights_out"][..., :keep] = torch.where(live, x["weights"].gather(2, kept), 0.0)
    return {"k_out": x["k_out"], "v_out": x["v_out"], "weights_out": x["weights_out"],
            "kept": torch.where(live, kept, -1).int(), "lengths_out": count.view(B).int()}


def plain_commit(case, x):
    B, T = case["batch"], case["seq"]
    batch = torch.arange(B, device="cuda")[:, None]
    first, step = x["lengths"].long()[:, None], torch.arange(T, device="cuda")
    taken = step < x["counts"].long()[:, None]  # [B, T]
    source, target = first + x["path"].long(), first + step
    x["k"][batch, :, target] = torch.where(taken[..., None, None], x["k"][batch, :, source], x["k"][batch, :, target])
    x["v"][batch, :, target] = torch.where(taken[..., None, None], x["v"][batch, :, source], x["v"][batch, :, target])
    out = {"k": x["k"], "v": x["v"], "lengths_out": x["lengths"] + x["counts"]}
    if case["weights"]:
        x["weights"][batch, :, target] = torch.where(taken[..., None], x["weights"][batch, :, source], 0.0)
        out["weights"] = x["weights"]
    return out


PLAIN = {"qk_norm_rope": plain_rope, "qk_norm_rope_grad": plain_rope_grad, "attention_tree": plain_tree, "cache_evict": plain_evict,
         "cache_commit": plain_commit}


# ------------------------------------------------------------------ work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    B, H, D, T = case["batch"], case["kv_heads"], case["dim"], case.get("seq", 0)
    row = D * size
    if case["op"].startswith("qk_norm_rope"):
        rows = B * T * (case["heads"] + 2 * H)
        if case["op"] == "qk_norm_rope":  # each row read and written
            return {"bytes": 2 * rows * row + B * T * 4, "flops": 10 * rows * D}
        # queries and keys, every gradient in, every gradient out (values' gradients pass through)
        return {"bytes": (3 * rows - B * T * H) * row + B * T * 4 + 8 * D, "flops": 20 * rows * D}
    lengths = lengths_of(case)
    if case["op"] == "attention_tree":
        keys = sum(n + T for n in lengths)
        extra = 8 * keys * H if case["weights"] else 0
        return {"bytes": 2 * keys * H * row + 2 * B * T * case["heads"] * row + extra, "flops": 4 * keys * case["heads"] * T * D}
    if case["op"] == "cache_evict":
        kept = sum(min(n, case["keep"]) for n in lengths)
        return {"bytes": H * (4 * kept * row + 4 * sum(lengths) + 4 * B * case["capacity"] + 4 * B * case["keep"]), "flops": 0}
    # half of a tree is accepted on average: its keys and values read and written
    return {"bytes": 4 * B * H * (T / 2) * row + 4 * B * (T + 3) + (12 * B * H * T / 2 if case["weights"] else 0), "flops": 0}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    x = prepare(case, seed)["x"]
    return EXACT[case["op"]](case, {n: v.double() if v.is_floating_point() else v.long() for n, v in x.items()})


def turned(case, x, position, back=False):
    """One token's heads [n, dim] as complex numbers times e^(i angle)."""
    R = case["rotary"]
    i = torch.arange(R // 2, dtype=torch.float64, device=x.device)
    theta = torch.exp(-(2 * i / R) * math.log(case["base"]))
    gain = 1.0
    if case["scaling"] == "linear":
        theta = theta / case["factor"]
    elif case["scaling"] == "ntk":
        theta = torch.exp(-(2 * i / R) * (math.log(case["base"]) + R / (R - 2) * math.log(case["factor"])))
    elif case["scaling"] == "yarn":
        share = torch.clamp((case["original"] * theta / (2 * math.pi) - 1) / (32 - 1), 0, 1)
        theta = (1 - share) * theta / case["factor"] + share * theta
        gain = 1 + 0.1 * math.log(case["factor"])
    angle = position.double() * theta
    turn = torch.polar(torch.full_like(angle, gain), -angle if back else angle)
    out = x.clone()
    if case["interleaved"]:
        z = torch.complex(x[..., 0:R:2], x[..., 1:R:2]) * turn
        out[..., 0:R:2], out[..., 1:R:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., : R // 2], x[..., R // 2 : R]) * turn
        out[..., : R // 2], out[..., R // 2 : R] = z.real, z.imag
    return out


def exact_rope(case, x):
    Q, H, T = case["heads"], case["kv_heads"], case["seq"]
    for b in range(case["batch"]):
        row, at = x["qkv"][b], x["positions"][b][:, None, None]
        q, k, v = row[:, :Q], row[:, Q : Q + H], row[:, Q + H :]
        if case["norm"]:
            q = q / torch.sqrt(torch.mean(q * q, -1, True) + 1e-6) * x["q_weight"]
            k = k / torch.sqrt(torch.mean(k * k, -1, True) + 1e-6) * x["k_weight"]
        first = int(x["starts"][b]) if case["capacity"] else 0
        x["q"][b] = turned(case, q, at).permute(1, 0, 2)
        x["k"][b, :, first : first + T] = turned(case, k, at).permute(1, 0, 2)
        x["v"][b, :, first : first + T] = v.permute(1, 0, 2)
    return {n: x[n] for n in OUTPUTS["qk_norm_rope"]}


def exact_rope_grad(case, x):
    Q, H = case["heads"], case["kv_heads"]
    sums = {"dq_weight": 0, "dk_weight": 0}
    for b in range(case["batch"]):
        at = x["positions"][b][:, None, None]
        for name, weight, lo, hi in (("dq", "q_weight", 0, Q), ("dk", "k_weight", Q, Q + H)):
            g = turned(case, x[name][b].permute(1, 0, 2), at, back=True)
            if case["norm"]:
                row = x["qkv"][b][:, lo:hi]
                size = torch.sqrt(torch.mean(row * row, -1, True) + 1e-6)
                sums[name + "_weight"] = sums[name + "_weight"] + torch.sum(g * row / size, (0, 1))
                u = g * x[weight]
                g = u / size - row * torch.mean(u * row, -1, True) / size**3
            x["dqkv"][b][:, lo:hi] = g
        x["dqkv"][b][:, Q + H :] = x["dv"][b].permute(1, 0, 2)
    return {"dqkv": x["dqkv"], **(sums if case["norm"] else {})}


def exact_tree(case, x):
    T, G = case["seq"], case["heads"] // case["kv_heads"]
    for b in range(case["batch"]):
        n = int(x["lengths"][b])
        may = torch.ones(T, n + T, dtype=torch.bool, device="cuda")
        j = torch.arange(T, device="cuda")
        may[:, n:] = ((x["tree"][b][:, j // 32] >> (j % 32)) & 1).bool()
        for h in range(case["kv_heads"]):
            k, v = x["k"][b, h, : n + T], x["v"][b, h, : n + T]
            heads = slice(h * G, (h + 1) * G)
            e = torch.exp(x["q"][b, heads] @ k.T / math.sqrt(case["dim"])) * may  # these scores stay far below e^700
            p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
            x["out"][b][:, heads] = (p @ v).permute(1, 0, 2)
            if case["weights"]:
                x["weights"][b, h, : n + T] += p.sum((0, 1))
    return {n: x[n] for n in OUTPUTS["attention_tree"] if n in x}


def exact_evict(case, x):
    keep, recent = case["keep"], case["recent"]
    x["kept"].fill_(-1)
    x["weights_out"].zero_()
    for b in range(case["batch"]):
        n = int(x["lengths"][b])
        count, last = min(n, keep), max(0, n - recent)
        x["lengths_out"][b] = count
        for h in range(case["kv_heads"]):
            w = x["weights"][b, h, :last].cpu().numpy()
            best = sorted((-w).argsort(kind="stable")[: count - (n - last)].tolist()) + list(range(last, n))
            rows = torch.tensor(best, dtype=torch.long, device="cuda")
            x["kept"][b, h, :count] = rows
            for name in ("k", "v", "weights"):
                x[name + "_out"][b, h, :count] = x[name][b, h].index_select(0, rows)
    return {n: x[n] for n in OUTPUTS["cache_evict"]}


def exact_commit(case, x):
    for b in range(case["batch"]):
        n, a = int(x["lengths"][b]), int(x["counts"][b])
        rows = n + x["path"][b, :a]
        for name in ("k", "v", "weights"):
            if name in x:
                moved = x[name][b].index_select(1, rows)
                if name == "weights":
                    x[name][b, :, n : n + case["seq"]] = 0
                x[name][b, :, n : n + a] = moved
    x["lengths_out"] = x["lengths"] + x["counts"]
    return {n: x[n] for n in OUTPUTS["cache_commit"] if n in x}


EXACT = {"qk_norm_rope": exact_rope, "qk_norm_rope_grad": exact_rope_grad, "attention_tree": exact_tree, "cache_evict": exact_evict,
         "cache_commit": exact_commit}
