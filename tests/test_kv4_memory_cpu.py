"""The engine's memory plan over a 4-bit KV cache: what a prefill call expands is set aside from the pool's share."""

import types

import pytest

from minisgl import ops
from minisgl.attention import native
from minisgl.attention.native import kv4_scratch_bytes
from minisgl.engine.engine import Engine
from minisgl.parallel import DistributedInfo
from minisgl.parallel import info as parallel_info

GB = 1 << 30


@pytest.fixture(autouse=True)
def _one_rank(monkeypatch):
    monkeypatch.setattr(parallel_info, "_TP", DistributedInfo(0, 1))


def _pages(kv_quant, ratio, longest, heads=8, requests=256, free=180 * GB, model=16 * GB):
    engine = Engine.__new__(Engine)
    engine.is_cuda, engine.page_size = True, 64
    engine.dtype = types.SimpleNamespace(itemsize=2)
    engine.model_config = types.SimpleNamespace(kv_quant=kv_quant, is_mla=False, num_kv_heads=heads, head_dim=128,
                                                num_layers=36, architectures=["Qwen3ForCausalLM"])
    engine._sync_get_memory = lambda: (free - model, free - model)
    config = types.SimpleNamespace(model_config=engine.model_config, num_page_override=None, memory_ratio=ratio,
                                   max_seq_len=longest, max_running_req=requests)
    return engine._determine_num_pages(free, config) * engine._bytes_per_page()


@pytest.mark.parametrize("ratio", [0.9, 1.0])
@pytest.mark.parametrize("longest,heads,requests", [(40960, 8, 256), (1 << 20, 8, 256), (4096, 40, 1279), (512, 8, 4)])
def test_the_pool_leaves_room_for_a_prefill_call(ratio, longest, heads, requests):
    pool = _pages("int4", ratio, longest, heads, requests)
    # the requests of a call, as long as they may be together, expanded in whole tiles: K and V in bf16
    counts = [longest] * max(1, min(requests, native.KV4_PLAN_KEYS // longest))
    counts += [1] * (requests - len(counts))
    plan = ops.KV4PrefillPlan(counts, native.torch.device("cpu"))
    assert 16 * GB + pool + plan.rows * heads * 128 * 2 * 2 <= ratio * 180 * GB
    assert pool >= 0.9 * (ratio * 180 * GB - 16 * GB - kv4_scratch_bytes(heads, 128, longest, requests))


def test_pools_of_16_bits_are_as_large_as_they_were():
    page = 2 * 36 * 8 * 64 * 128 * 2
    assert _pages("none", 0.9, 40960) == int(0.9 * 180 * GB - 16 * GB) // page * page
