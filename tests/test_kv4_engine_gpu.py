"""The engine over a 4-bit KV cache on a B200: its kernels end to end against
the dense fp32 oracle whose keys and values go through the same format, graph
decode against eager decode, and prefixes shared between requests.

The margin of a token against the oracle's best: keys and values come out of
bf16 products, whose noise (2^-8 of a value against steps of 2/15 of a group's
largest) moves about 6 % of the codes by a step. That is an error of 0.25 of a
step per element beside the format's own 0.29, some 0.08 of a value's rms, and
attention keeps that share of its output. Attention makes about half of what
the two layers add, so a logit moves by 0.06 of the logits' rms and the
difference of two by 0.08: 4 deviations are 0.09 of the largest of 4096 logits
(3.5 rms). With the 0.03 that bf16 alone is allowed elsewhere: 0.12. A wrong
token's logit is near zero."""

import random

import pytest
import torch

from minisgl import ops
from minisgl.attention import native
from minisgl.core import SamplingParams
from minisgl.llm import LLM
from minisgl.models.oracle import dense_logits
from minisgl.utils.synthetic import make_model_dir

pytestmark = pytest.mark.gpu


def _make(graph_bs, **kw):
    args = dict(dtype=torch.bfloat16, device="cuda:0", use_dummy_weight=True, dummy_weight_device="cpu",
                page_size=64, max_running_req=16, max_seq_len_override=2048, num_page_override=256,
                cuda_graph_max_bs=graph_bs, max_extend_tokens=256, kv_quant="int4")
    args.update(kw)
    return LLM(make_model_dir("small-qwen3"), **args)


def _prompts(n, seed=0):
    rng = random.Random(seed)
    return [[rng.randrange(4096) for _ in range(rng.randint(1, 300))] for _ in range(n)]


@pytest.mark.parametrize("page", [16, 64, 256])
def test_engine_follows_the_quantised_oracle(page):
    """Prompts of one token to several chunks (both attention paths), decode
    by graphs, then the same prompts from cached prefixes."""
    llm = _make(16, page_size=page)
    try:
        prompts = _prompts(6)
        greedy = SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)
        state, cfg = llm.engine.model.state_dict(), llm.engine.model_config
        for _ in range(2):
            outs = llm.generate(prompts, greedy)
            ops.check_device_errors(torch.device("cuda:0"))
            for p, o in zip(prompts, outs):
                toks = o["token_ids"]
                assert len(toks) == 12
                logits = dense_logits(state, cfg, p + toks[:-1],
                                      fused_layout=llm.engine.model.fused_layout)[len(p) - 1:]
                for t, row in zip(toks, logits):
                    assert row[t] >= row.max() - 0.12 * row.abs().max(), (t, int(row.argmax()))
    finally:
        llm.shutdown()


def test_batches_of_many_cached_keys_take_several_calls(monkeypatch):
    """With a limit of 300 keys a call, prompts go through in parts, each token near the oracle's best."""
    outs = []
    for limit in (native.KV4_PLAN_KEYS, 300):
        monkeypatch.setattr(native, "KV4_PLAN_KEYS", limit)
        llm = _make(16, gemm_autotune=False, max_extend_tokens=2048)
        try:
            prompts = _prompts(12, 5)
            outs.append([o["token_ids"] for o in llm.generate(prompts, SamplingParams(temperature=0.0, max_tokens=1,
                                                                                      ignore_eos=True))])
            ops.check_device_errors(torch.device("cuda:0"))
            state, cfg = llm.engine.model.state_dict(), llm.engine.model_config
            for p, (t,) in zip(prompts, outs[-1]):
                row = dense_logits(state, cfg, p, fused_layout=llm.engine.model.fused_layout)[-1]
                assert row[t] >= row.max() - 0.12 * row.abs().max()
        finally:
            llm.shutdown()
    assert len(outs[0]) == len(outs[1]) == 12


def test_graph_decode_equals_eager_decode():
    """Every batch size is captured, so no graph pads its batch (the even split
    of the keys counts padding requests, and another split rounds otherwise)."""
    outs = []
    for sizes in ([], list(range(1, 10))):
        llm = _make(16, cuda_graph_bs=sizes, gemm_autotune=False)
        try:
            outs.append(llm.generate(_prompts(9, 3), SamplingParams(temperature=0.0, max_tokens=10, ignore_eos=True)))
            ops.check_device_errors(torch.device("cuda:0"))
        finally:
            llm.shutdown()
    assert [o["token_ids"] for o in outs[0]] == [o["token_ids"] for o in outs[1]]
