"""The cached attention operators at sizes where a persistent warp works on several items
and a block on several tiles, against the same references as at small ones."""
import numpy as np
import pytest

import jade_compute_b200 as jc
from tests import test_gpu_cached_attention as base

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    r = jc.Runtime(0)
    yield r
    r.close()


# about 3,000 warps are resident: one, one and a half, two and more items a warp; halves,
# neighbours, halves through rows; a warp's next item in the next sequence of the batch
ROPES = [
    dict(batch=3, seq=2003, heads=3, kv_heads=1, dim=64),
    dict(batch=2, seq=3001, heads=6, kv_heads=2, dim=128, interleaved=True, capacity=3100),
    dict(batch=5, seq=1301, heads=4, kv_heads=4, dim=80, rotary=20),
    dict(batch=37, seq=83, heads=9, kv_heads=3, dim=128, rotary=64, capacity=90),
    dict(batch=9, seq=501, heads=6, kv_heads=1, dim=136, rotary=40, norm=False, scaling="linear", factor=2.0),
    dict(batch=1, seq=6500, heads=2, kv_heads=1, dim=256, interleaved=True, rotary=130),
    dict(batch=2, seq=1700, heads=32, kv_heads=8, dim=64, rotary=12, capacity=1800),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", range(len(ROPES)))
def test_qk_norm_rope(rt, monkeypatch, case, dtype):
    monkeypatch.setattr(base, "ROPES", ROPES)
    base.test_qk_norm_rope(rt, case, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", range(len(ROPES)))
def test_qk_norm_rope_grad(rt, monkeypatch, case, dtype):
    monkeypatch.setattr(base, "ROPES", ROPES)
    base.test_qk_norm_rope_grad(rt, case, dtype)


# clusters of two, four and eight blocks, also with several tiles a block; several tiles a
# block without a cluster (more heads than half the SMs)
EVICTS = [
    dict(batch=2, kv_heads=2, dim=16, capacity=12000, keep=3000, recent=40, lengths=[12000, 8193]),
    dict(batch=3, kv_heads=1, dim=16, capacity=30000, keep=29000, recent=1, lengths=[30000, 29999, 16385]),
    dict(batch=2, kv_heads=25, dim=8, capacity=40000, keep=20000, recent=0, lengths=[40000, 16500]),
    dict(batch=40, kv_heads=2, dim=8, capacity=9000, keep=700, recent=100, lengths=[9000 - 227 * b for b in range(40)]),
    dict(batch=77, kv_heads=1, dim=8, capacity=25000, keep=8200, recent=8200, lengths=[25000 - 300 * b for b in range(77)]),
]


@pytest.mark.parametrize("kind", ["spread", "ties", "strange"])
@pytest.mark.parametrize("case", range(len(EVICTS)))
def test_cache_evict(rt, monkeypatch, case, kind):
    monkeypatch.setattr(base, "EVICTS", EVICTS)
    base.test_cache_evict(rt, case, kind, "bf16")
