"""The 4-bit pool's own methods take rows of either shape that those of the 16-bit pool take."""

import pytest
import torch

from minisgl import ops
from minisgl.kvcache import MHAKV4Cache
from minisgl.kvcache.mha_pool import MHAKVCache
from minisgl.parallel import DistributedInfo
from minisgl.parallel import info as parallel_info

import kv4_oracle as oracle


@pytest.fixture(autouse=True)
def _one_rank(monkeypatch):
    monkeypatch.setattr(parallel_info, "_TP", DistributedInfo(0, 1))


def _rows_in_and_out(device, dtype):
    heads, d, page, T = 2, 64, 16, 9
    g = torch.Generator().manual_seed(0)
    kv = torch.randn(2, T, heads * d + 16, generator=g).to(dtype)[:, :, :heads * d].to(device)
    slots = torch.randperm(3 * page, generator=g)[:T].to(torch.int32).to(device)
    wide = MHAKVCache(heads, 2, d, 3, page, dtype, device)
    pool = MHAKV4Cache(heads, 2, d, 3, page, dtype, device)
    for layer, shape in ((0, (T, heads * d)), (1, (T, heads, d))):
        k, v = (x.reshape(shape) if layer else x for x in kv)
        for p in (wide, pool):
            p.store_kv(k, v, slots, layer)
        for got, want in zip(pool.load_kv(slots, layer), kv):
            c, byte = oracle.quantize(want.cpu().reshape(T, heads, d))
            assert torch.equal(got.double().cpu(), oracle.values(c[..., 0::2] | (c[..., 1::2] << 4), byte))


def test_rows_in_and_out_on_the_cpu():
    _rows_in_and_out(torch.device("cpu"), torch.float32)


@pytest.mark.gpu
def test_rows_in_and_out():
    _rows_in_and_out(torch.device("cuda"), torch.bfloat16)
    torch.cuda.synchronize()
    ops.check_device_errors(torch.device("cuda"))
