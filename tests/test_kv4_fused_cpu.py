"""The fused layer form (norms, activation and residual adds in the GEMMs' epilogues) with a 4-bit KV cache: only
the store of keys and values leaves the qkv GEMM's epilogue."""

import os
import random

import pytest
import torch

from minisgl import ops
from minisgl.core import SamplingParams
from minisgl.llm import LLM
from minisgl.models.oracle import dense_logits
from minisgl.models.weight import load_weight
from minisgl.ops import gemm_tune
from minisgl.utils.synthetic import make_model_dir, write_random_checkpoint

KEYS = ("norm_eps", "residual", "silu", "rope")
SHAPE = dict(head_dim=128, num_attention_heads=2, num_key_value_heads=1, hidden_size=256, intermediate_size=512,
             tie_word_embeddings=False)


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    """Norm weights that are not one, so that folding them counts."""
    path = os.path.join(tmp_path_factory.mktemp("kv4_fused"), "m")
    make_model_dir("tiny-qwen3", folder=path, overrides=SHAPE)
    write_random_checkpoint(path, seed=7, std=0.05, norm_std=0.3)
    return path


def _make(folder, kv_quant, **kw):
    args = dict(dtype=torch.float32, device="cpu", page_size=16, max_extend_tokens=64, num_page_override=64,
                max_running_req=16, max_seq_len_override=256, kv_quant=kv_quant)
    args.update(kw)
    return LLM(folder, **args)


@pytest.mark.parametrize("kv_quant", ["none", "int4"])
def test_layers_take_the_fused_form(folder, kv_quant, monkeypatch):
    made = []
    gemm = ops.gemm_fused

    def counted(x, w, **kw):
        made.append(tuple(k for k in KEYS if kw.get(k) is not None and kw[k] is not False))
        return gemm(x, w, **kw)

    monkeypatch.setattr(ops, "gemm_fused", counted)
    llm = _make(folder, kv_quant)
    try:
        model, cfg = llm.engine.model, llm.engine.model_config
        assert model.model.fusable and model.fused_layout and model.forward_variants() == (True, False)
        rng = random.Random(0)
        prompts = [[rng.randrange(1024) for _ in range(n)] for n in (1, 20, 9)]
        greedy = SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True)
        outs = [o["token_ids"] for o in llm.generate(prompts, greedy)]
        qkv = ("norm_eps", "rope") if kv_quant == "none" else ("norm_eps",)
        assert made and made == [qkv, ("residual",), ("norm_eps", "silu"), ("residual",)] * (len(made) // 4)
        state = dict(load_weight(folder, torch.device("cpu")))  # as they are in the checkpoint, not folded
        for p, out in zip(prompts, outs):
            rows = dense_logits(state, cfg, p + out[:-1])[len(p) - 1:]
            for t, row in zip(out, rows):  # 1 %: a value that another order of sums moves over a code's border
                assert row[t] >= row.max() - 0.01 * row.abs().max()
    finally:
        llm.shutdown()


def test_kinds_of_the_tuned_projections(folder):
    """The qkv projection is tuned with the norm alone; its plans are among those of the whole epilogue."""
    for kv_quant, kind in (("none", ops.EPI_NORM | ops.EPI_ROPE), ("int4", ops.EPI_NORM)):
        llm = _make(folder, kv_quant)
        try:
            model = llm.engine.model
            qkv = model.model.layers.op_list[0].self_attn.qkv_proj.weight
            assert model.fused_gemm_kinds()[tuple(qkv.shape)][0] == kind
        finally:
            llm.shutdown()
    for M in (1, 64, 256):
        assert gemm_tune._fused_candidates(M, 4096, ops.EPI_NORM) == gemm_tune._fused_candidates(
            M, 4096, ops.EPI_NORM | ops.EPI_ROPE)


def test_heads_of_64_dims_have_no_fused_form():
    llm = _make(make_model_dir("tiny-qwen3", overrides={"tie_word_embeddings": False, "head_dim": 64}), "int4",
                use_dummy_weight=True)
    try:
        assert not llm.engine.model.model.fusable and not llm.engine.model.fused_layout
        assert llm.engine.model.forward_variants() == (None,)
        assert len(llm.generate([[3, 4, 5]], SamplingParams(temperature=0.0, max_tokens=3, ignore_eos=True))[0]["token_ids"]) == 3
    finally:
        llm.shutdown()
