"""A 4-bit KV cache under tensor parallelism on CPU ranks (gloo): each rank holds its KV heads, replicated where
there are more ranks than heads, and every token is near the best of the dense oracle whose keys and values go
through the same format. And prefill batches in several calls: as many as the limit on keys asks for."""

import random
import shutil
import tempfile

import pytest
import torch
import torch.multiprocessing as mp

from minisgl.attention import native
from minisgl.core import SamplingParams
from minisgl.llm import LLM
from minisgl.models.oracle import dense_logits

from test_tp_cpu import PROMPTS, _free_port

ARGS = dict(dtype=torch.float32, device="cpu", page_size=16, num_page_override=64, max_running_req=8,
            max_seq_len_override=256, max_extend_tokens=64, kv_quant="int4")


def _run(rank, world, folder, port, sp, out_q):
    from minisgl.parallel import DistributedCommunicator, DistributedInfo

    llm = LLM(folder, tp_info=DistributedInfo(rank, world), distributed_port=port, **ARGS)
    if sp:  # token-sharded residual stream, token counts padded to the ranks
        DistributedCommunicator.plugins[-1].sequence_parallel = True
    assert llm.engine.model.model.fusable
    heads = llm.engine.kv_cache.pool.shape[3]
    outs = llm.generate(PROMPTS, [SamplingParams(temperature=0.0, max_tokens=m, ignore_eos=True) for m in (8, 5)])
    out_q.put((rank, ([o["token_ids"] for o in outs], heads)))
    llm.shutdown()


@pytest.fixture(scope="module")
def checkpoint():
    from minisgl.utils.synthetic import make_model_dir, write_random_checkpoint

    folder = tempfile.mkdtemp(prefix="minisgl_kv4_ranks_")
    shutil.rmtree(folder)
    # 128-dim heads and halves of 128 columns a rank: layers have a fused form
    make_model_dir("tiny-qwen3", folder=folder, overrides={"tie_word_embeddings": False, "head_dim": 128,
                                                           "intermediate_size": 1024})
    write_random_checkpoint(folder, seed=3, std=0.05)
    yield folder
    shutil.rmtree(folder, ignore_errors=True)


@pytest.mark.parametrize("world,sp", [(2, False), (4, False), (2, True)])
def test_ranks_hold_their_heads_in_4_bits(checkpoint, world, sp):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_run, args=(r, world, checkpoint, port, sp, q)) for r in range(world)]
    for p in procs:
        p.start()
    results = dict(q.get(timeout=300) for _ in range(world))
    for p in procs:
        p.join(timeout=120)
        assert p.exitcode == 0
    llm = LLM(checkpoint, **ARGS)
    try:
        model, cfg = llm.engine.model, llm.engine.model_config
        tokens, _ = results[0]
        assert all(t == tokens and heads == max(1, cfg.num_kv_heads // world) for t, heads in results.values())
        for prompt, out, n in zip(PROMPTS, tokens, (8, 5)):
            assert len(out) == n
            rows = dense_logits(model.state_dict(), cfg, prompt + out[:-1],
                                fused_layout=getattr(model, "fused_layout", False))[len(prompt) - 1:]
            for t, row in zip(out, rows):  # 1 %: a value that another order of sums moves over a code's border
                assert row[t] >= row.max() - 0.01 * row.abs().max()
    finally:
        llm.shutdown()


def test_a_limit_on_keys_makes_several_calls(checkpoint, monkeypatch):
    """Without a limit in reach a layer attends a prefill batch in one call; with one of 40 keys in as many as
    its requests need, and to the same tokens."""
    rng = random.Random(1)
    prompts = [[rng.randrange(1024) for _ in range(n)] for n in (30, 9, 25, 16, 20)]
    tokens, calls = [], []
    attend = native.ops.prefill_attention_kv4

    def counted(q, pool, layer, pt, rows, lens, *rest, **kw):
        calls[-1].append((layer, lens.tolist()))
        return attend(q, pool, layer, pt, rows, lens, *rest, **kw)

    monkeypatch.setattr(native.ops, "prefill_attention_kv4", counted)
    for limit in (1 << 18, 40):
        monkeypatch.setattr(native, "KV4_PLAN_KEYS", limit)
        calls.append([])
        llm = LLM(checkpoint, **dict(ARGS, max_extend_tokens=256))
        try:
            tokens.append([o["token_ids"] for o in llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=3,
                                                                                        ignore_eos=True))])
        finally:
            llm.shutdown()
    assert tokens[0] == tokens[1] and all(len(t) == 3 for t in tokens[0])
    first, second = ([lens for layer, lens in made if layer == 0] for made in calls)
    assert first == [[30, 9, 25, 16, 20]]
    assert second == [[30, 9], [25], [16, 20]]
