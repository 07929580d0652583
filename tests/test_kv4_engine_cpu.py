"""The engine over a 4-bit KV cache on the CPU: paged, chunked and
prefix-shared runs against the dense fp32 oracle whose keys and values go
through the same format, the pool's memory, and what is refused."""

import random

import pytest
import torch

from minisgl import ops
from minisgl.core import SamplingParams
from minisgl.engine.config import EngineConfig
from minisgl.kvcache import MHAKV4Cache, create_kvcache_pool
from minisgl.kvcache.mha_pool import MHAKVCache
from minisgl.llm import LLM
from minisgl.models.oracle import dense_logits
from minisgl.parallel import DistributedInfo
from minisgl.server.args import parse_args
from minisgl.utils.synthetic import make_model_dir


def _make(shape="tiny-qwen3", **kw):
    args = dict(dtype=torch.float32, device="cpu", use_dummy_weight=True, page_size=16, max_extend_tokens=32,
                num_page_override=256, max_running_req=16, max_seq_len_override=512, cache_type="radix",
                kv_quant="int4")
    args.update(kw)
    return LLM(make_model_dir(shape, overrides={"tie_word_embeddings": False}), **args)


def _near_best(llm, prompt, tokens):
    """Each token is the oracle's choice or within 1 % of the largest logit of
    it: sums in another order may move a value over a rounding boundary of its
    code, which shifts one element of one key by a step."""
    model = llm.engine.model
    rows = dense_logits(model.state_dict(), llm.engine.model_config, prompt + tokens[:-1],
                        fused_layout=getattr(model, "fused_layout", False))[len(prompt) - 1:]
    for t, row in zip(tokens, rows):
        assert row[t] >= row.max() - 0.01 * row.abs().max(), (t, int(row.argmax()))


@pytest.mark.parametrize("shape", ["tiny-qwen3", "tiny-llama"])
def test_engine_follows_the_quantised_oracle(shape):
    llm = _make(shape)
    try:
        assert isinstance(llm.engine.kv_cache, MHAKV4Cache)
        rng = random.Random(0)
        prefix = [rng.randrange(1024) for _ in range(40)]
        prompts = [[rng.randrange(1024) for _ in range(rng.randint(1, 70))] for _ in range(5)]
        prompts += [prefix + [rng.randrange(1024) for _ in range(n)] for n in (1, 17, 30)]
        for _ in range(2):  # the second time from cached prefixes
            outs = llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True))
            for p, o in zip(prompts, outs):
                assert len(o["token_ids"]) == 8
                _near_best(llm, p, o["token_ids"])
        assert llm.cache_manager.prefix_cache.size_info.total_size >= 40
        llm.cache_manager.check_integrity()
    finally:
        llm.shutdown()


def test_parts_of_a_prefill_batch(monkeypatch):
    """Requests of a batch fall into calls of a bounded number of keys, in order, none left out."""
    from minisgl.attention import native

    backend = native.NativeAttnBackend.__new__(native.NativeAttnBackend)
    backend.hq, backend.hk, backend.device = 8, 2, torch.device("cpu")
    lens, qlens = [100, 250, 40, 10, 900, 5, 5], [30, 1, 40, 2, 7, 5, 1]
    cu = [0]
    for n in qlens:
        cu.append(cu[-1] + n)
    cu_q = torch.tensor(cu, dtype=torch.int32)
    for limit, want in ((1 << 18, [(0, 7)]), (300, [(0, 1), (1, 4), (4, 5), (5, 7)]), (1, [(i, i + 1) for i in range(7)])):
        monkeypatch.setattr(native, "KV4_PLAN_KEYS", limit)
        parts = backend._kv4_parts(lens, qlens, cu, cu_q)
        assert [(p.first, p.last) for p in parts] == want
        for p in parts:
            assert (p.q0, p.q1, p.max_q) == (cu[p.first], cu[p.last], max(qlens[p.first:p.last]))
            assert p.cu_q.dtype == torch.int32 and p.cu_q.tolist() == [c - p.q0 for c in cu[p.first:p.last + 1]]


def test_a_batch_in_parts_gives_the_same_tokens(monkeypatch):
    from minisgl.attention import native

    rng = random.Random(3)
    prompts = [[rng.randrange(1024) for _ in range(rng.randint(1, 30))] for _ in range(6)]
    outs = []
    for limit in (native.KV4_PLAN_KEYS, 25):
        monkeypatch.setattr(native, "KV4_PLAN_KEYS", limit)
        llm = _make(max_extend_tokens=256)
        try:
            outs.append(llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=4, ignore_eos=True)))
            for p, o in zip(prompts, outs[-1]):
                _near_best(llm, p, o["token_ids"])
        finally:
            llm.shutdown()


def test_pool_bytes_and_pages():
    """A page costs what its codes and scales take, and pages copy whole."""
    llm = _make()
    try:
        kv = llm.engine.kv_cache
        cfg = llm.engine.model_config
        per_page = 2 * cfg.num_layers * cfg.num_kv_heads * (16 * 32 + 16 * 2)
        assert llm.engine._bytes_per_page() == per_page == kv.pool.numel() // kv.num_pages
        assert per_page == MHAKV4Cache.bytes_per_page(cfg.num_kv_heads, cfg.num_layers, cfg.head_dim, 16, torch.float32)
        kv.pool.random_(0, 256)
        before = kv.pool.clone()
        kv.copy_pages([3, 3], [5, 7])
        before[:, :, [5, 7]] = before[:, :, [3]]
        assert torch.equal(kv.pool, before)
        pool = MHAKVCache(2, 3, 64, 6, 16, torch.float32, torch.device("cpu"))
        pool.pool.random_()
        before = pool.pool.clone()
        pool.copy_pages([1], [4])
        before[:, :, 4] = before[:, :, 1]
        assert torch.equal(pool.pool, before)
    finally:
        llm.shutdown()


def test_latent_pool_copies_pages():
    from minisgl.kvcache.mla_pool import MLAKVCache

    pool = MLAKVCache(2, 32, 16, 5, 16, torch.float32, torch.device("cpu"))
    pool.pool.random_()
    before = pool.pool.clone()
    pool.copy_pages([4, 0], [1, 2])
    before[:, [1, 2]] = before[:, [4, 0]]
    assert torch.equal(pool.pool, before)


def _config(shape, **kw):
    return EngineConfig(make_model_dir(shape), DistributedInfo(0, 1), torch.float32, device="cpu", **kw).model_config


def test_what_a_4bit_cache_refuses():
    dev = torch.device("cpu")
    with pytest.raises(ValueError, match="MLA latent"):
        create_kvcache_pool(_config("tiny-kimi", kv_quant="int4"), 4, 16, torch.float32, dev)
    with pytest.raises(ValueError, match="none or int4"):
        create_kvcache_pool(_config("tiny-qwen3", kv_quant="int8"), 4, 16, torch.float32, dev)
    for kw, said in ((dict(page_size=1), "page_size"), (dict(page_size=24), "page_size"),
                     (dict(max_running_req=ops.KV4_MAX_BATCH), "at most"), (dict(kv_quant="int8"), "none or int4"),
                     (dict(shape="tiny-kimi"), "MLA latent"),
                     (dict(device="cuda:0", dtype=torch.float16), "bfloat16")):
        with pytest.raises(ValueError, match=said):
            _make(**kw)


def test_flag():
    args, _ = parse_args(["--model", "synthetic:tiny-qwen3", "--kv-quant", "int4"])
    assert args.kv_quant == "int4" and args.model_config.kv_quant == "int4"
    args, _ = parse_args(["--model", "synthetic:tiny-qwen3"])
    assert args.kv_quant == "none"
    with pytest.raises(SystemExit):
        parse_args(["--model", "synthetic:tiny-qwen3", "--kv-quant", "int3"])
