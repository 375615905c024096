"""Serving operators without a GPU: what the C ABI refuses before it touches a device, and the
shape and dtype checks of the Python layer (made on a context that never reaches the library)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from headshot_b200 import _lib
from headshot_b200.build import OUT as LIB_PATH
from headshot_b200.build import build
from headshot_b200.engine import GpuContext, PagedKv, Rope


@pytest.fixture(scope="module")
def L():
    if not LIB_PATH.exists():
        build()
    return _lib.lib()


def test_null_context_is_a_status(L):
    bf16 = _lib.HS_BF16
    n = ctypes.c_size_t()
    calls = [
        L.hs_kv_append(None, *[None] * 10, 0, 0, 0, 1, 1, 8, 8, 64, 4, 16, 4, bf16, None, None, 0, 0, 0),
        L.hs_attention_varlen(None, *[None] * 4, 0, 0, 0, None, None, 1, 1, 1, 8, 8, 64, 1, bf16, 0.0),
        L.hs_attention_paged(None, *[None] * 6, 0, 1, 8, 8, 64, 4, 16, 4, bf16, 0.0, None, 0),
        L.hs_attention_paged_workspace(None, ctypes.byref(n)),
    ]
    assert calls == [_lib.HS_ERR_INVALID] * 4
    assert "hs_attention_paged_workspace" in _lib.last_error()


class Unreached(GpuContext):
    """The Python checks alone: tensors stay on the CPU and no call may get to the library."""

    def __init__(self):
        self.device = torch.device("cpu")
        self._index = -1
        self._L = None
        self._h = None

    def _bind_stream(self):
        raise RuntimeError("reached the library")


@pytest.fixture
def ctx():
    return Unreached()


def cache(pages=4, heads=2, page=16, d=64, seqs=3, per_seq=2, dtype=torch.bfloat16):
    return PagedKv(torch.zeros(pages, heads, page, d, dtype=dtype), torch.zeros(pages, heads, page, d, dtype=dtype),
                   torch.zeros(seqs, per_seq, dtype=torch.int32))


def rows(t, h, d=64, dtype=torch.bfloat16):
    return torch.zeros(t, h, d, dtype=dtype)


LENS = torch.ones(3, dtype=torch.int32)


def test_accepted_calls_reach_the_library(ctx):
    fused = torch.zeros(3, 8 + 4, 64, dtype=torch.bfloat16)  # one projection's q, k, v
    with pytest.raises(RuntimeError, match="reached"):
        ctx.kv_append(cache(), fused[:, 8:10], fused[:, 10:], LENS, q=fused[:, :8])
    with pytest.raises(RuntimeError, match="reached"):
        ctx.attention_varlen(fused[:, :8], fused[:, 8:10], fused[:, 10:], torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="reached"):
        ctx.attention_paged(rows(3, 8), cache(), LENS, workspace=torch.zeros(16, dtype=torch.uint8))


@pytest.mark.parametrize("change", [
    dict(k=rows(3, 4)),                                     # heads other than the cache's
    dict(v=rows(2, 2)),                                     # k and v differ
    dict(v=rows(3, 2, dtype=torch.float16)),
    dict(k=rows(3, 2, dtype=torch.float16), v=rows(3, 2, dtype=torch.float16)),  # not the cache's type
    dict(k=rows(4, 2), v=rows(4, 2)),                       # one token per sequence
    dict(k=rows(3, 2, 128), v=rows(3, 2, 128)),
    dict(k=torch.zeros(3, 64, 2, dtype=torch.bfloat16).transpose(1, 2), v=rows(3, 2)),  # heads not contiguous
    dict(lens=torch.ones(3)),                               # not int32
    dict(lens=torch.ones(4, dtype=torch.int32)),
    dict(cu_new=torch.zeros(3, dtype=torch.int32)),         # needs n_seqs + 1
    dict(q=rows(3, 3)),                                     # not a multiple of 2 heads
    dict(q=rows(2, 4)),
    dict(q_out=rows(3, 4)),                                 # without q
    dict(q=rows(3, 4), q_out=rows(3, 8)),
    dict(k_out=rows(3, 4)),
    dict(rope=Rope(torch.zeros(9, 64), torch.zeros(8, 64), 0)),
    dict(rope=Rope(torch.zeros(9, 32), torch.zeros(9, 32), 0)),
    dict(rope=Rope(torch.zeros(9, 64).double(), torch.zeros(9, 64).double(), 0)),
])
def test_kv_append_refusals(ctx, change):
    a = dict(k=rows(3, 2), v=rows(3, 2), lens=LENS)
    a.update(change)
    k, v, lens = a.pop("k"), a.pop("v"), a.pop("lens")
    with pytest.raises(AssertionError):
        ctx.kv_append(cache(), k, v, lens, **a)


CU = torch.tensor([0, 1, 3], dtype=torch.int32)


@pytest.mark.parametrize("change", [
    dict(q=rows(3, 3)),
    dict(v=rows(3, 4)),
    dict(k=rows(3, 2, dtype=torch.float16), v=rows(3, 2, dtype=torch.float16)),
    dict(k=rows(4, 2), v=rows(4, 2)),                       # other lengths need cu_k
    dict(cu_q=CU.long()),
    dict(cu_k=CU[:2].contiguous()),
    dict(out=rows(3, 4)),
    dict(q=torch.zeros(3, 512, dtype=torch.bfloat16)),      # heads not split
    dict(q=rows(1, 8).expand(3, 8, 64)),                    # tokens on top of one another
])
def test_attention_varlen_refusals(ctx, change):
    a = dict(q=rows(3, 8), k=rows(3, 2), v=rows(3, 2), cu_q=CU)
    a.update(change)
    with pytest.raises(AssertionError):
        ctx.attention_varlen(**a)


@pytest.mark.parametrize("change", [
    dict(q=rows(2, 8)),
    dict(q=rows(3, 7)),
    dict(q=rows(3, 8, dtype=torch.float16)),
    dict(q=rows(3, 8, 128)),
    dict(kv_lens=LENS.long()),
    dict(out=rows(3, 4)),
    dict(cache=PagedKv(cache().k, cache(pages=5).v, cache().block_table)),
    dict(cache=PagedKv(cache().k, cache().v, cache().block_table.long())),
    dict(cache=PagedKv(cache().k, cache().v, cache().block_table[:, :1])),  # not contiguous
])
def test_attention_paged_refusals(ctx, change):
    a = dict(q=rows(3, 8), cache=cache(), kv_lens=LENS, workspace=torch.zeros(16, dtype=torch.uint8))
    a.update(change)
    with pytest.raises(AssertionError):
        ctx.attention_paged(**a)
