"""Calls on the 8-bit KV cache that are refused before anything is launched (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from __graft_entry__ import load_package
from oracle import q8 as Q

PKG = load_package()
from loop_sglang_b200 import ops  # noqa: E402

LIB = PKG._lib.lib()
P = ctypes.c_void_p(64)
F = ctypes.c_float


def attention(**over) -> int:
    a = dict(out=P, out_stride=1024, q=P, q_stride=1024, k=P, v=P, slot_stride=1024, num_slots=64,
             ks=P, vs=P, block=16, code=0, table=P, pt_stride=4, lens=P, cu=P, reqs=2, rows=2,
             hq=8, hkv=8, d=128, page=16, max_seqlen=64, scale=F(1.0), ws=P, ws_bytes=1 << 40)
    a.update(over)
    return LIB.lsb_paged_attention_q8(*a.values(), None)


@pytest.mark.parametrize("over", [
    dict(d=80), dict(hq=7), dict(hkv=0), dict(code=2), dict(block=3), dict(block=256),
    dict(block=0), dict(page=8), dict(page=0), dict(max_seqlen=65), dict(max_seqlen=0),
    dict(pt_stride=0), dict(num_slots=0), dict(num_slots=1 << 31), dict(reqs=0),
    dict(slot_stride=1016), dict(slot_stride=512), dict(q_stride=1020), dict(out_stride=512),
    dict(out=None), dict(ks=None), dict(cu=None), dict(q=ctypes.c_void_p(8)),
    dict(k=ctypes.c_void_p(72)), dict(vs=ctypes.c_void_p(66)), dict(ws=None), dict(ws_bytes=64)])
def test_attention_refusals(over) -> None:
    before = PKG._lib.launch_count()
    assert attention(**over) == PKG._lib.LSB_ERR_INVALID, over
    assert LIB.lsb_last_error().startswith(b"lsb_paged_attention_q8")
    assert PKG._lib.launch_count() == before


def append(**over) -> int:
    a = dict(qkv=P, qkv_stride=3 * 1024, q_out=P, q_out_stride=1024, pos=P, cos_sin=P, max_pos=8,
             k=P, v=P, slot_stride=1024, num_slots=64, ks=P, vs=P, block=16, code=1, loc=P,
             tokens=4, hq=8, hkv=8, d=128)
    a.update(over)
    return LIB.lsb_rope_store_kv_q8(*a.values(), None)


@pytest.mark.parametrize("over", [
    dict(d=48), dict(hq=12), dict(hkv=0), dict(code=-1), dict(block=5), dict(block=512),
    dict(qkv_stride=1024), dict(qkv_stride=3 * 1024 + 4), dict(q_out_stride=1000),
    dict(slot_stride=1000), dict(slot_stride=1032), dict(num_slots=0), dict(max_pos=0),
    dict(qkv=None), dict(loc=None), dict(ks=None), dict(qkv=ctypes.c_void_p(72)),
    dict(v=ctypes.c_void_p(72)), dict(cos_sin=ctypes.c_void_p(72))])
def test_append_refusals(over) -> None:
    assert append(**over) == PKG._lib.LSB_ERR_INVALID, over
    assert LIB.lsb_last_error().startswith(b"lsb_rope_store_kv_q8")


def test_store_refusals_and_empty_calls() -> None:
    def store(k_stride=1024, tokens=4, d=128):
        return LIB.lsb_store_kv_q8(P, P, 1024, 64, P, P, 16, 0, P, k_stride, P, 1024, P, tokens, 8,
                                   d, None)

    bad = PKG._lib.LSB_ERR_INVALID
    assert store(k_stride=512) == bad and store(k_stride=1028) == bad and store(d=72) == bad
    before = PKG._lib.launch_count()
    assert store(tokens=0) == 0 and append(tokens=0) == 0 and attention(rows=0) == 0
    assert PKG._lib.launch_count() == before


def test_wrappers_want_cuda_tensors_of_the_right_types() -> None:
    code = torch.zeros(32, 128, dtype=torch.int8)
    scale = torch.zeros(2, 1)
    with pytest.raises(ValueError):
        ops._q8_layer(code.float(), code, scale, scale, 16, 1, 128)
    with pytest.raises(ValueError):
        ops._q8_layer(code, code[:16], scale, scale, 16, 1, 128)
    with pytest.raises(ValueError):
        ops._q8_layer(code, code, scale, scale, 8, 1, 128)  # four blocks, two scales
    x, at = torch.zeros(1, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="bf16"):
        ops.store_kv_q8(code, code, scale, scale, at, x.float(), x, 1, 128, 16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.store_kv_q8(code, code, scale, scale, at, x, x, 1, 128, 16)
    q, cu = x.view(1, 1, 128), torch.tensor([0, 1], dtype=torch.int32)
    table = torch.zeros(1, 2, dtype=torch.int32)

    def attend(**over):
        a = dict(q=q, table=table, lens=at, cu=cu, page=16, longest=32, hkv=1)
        a.update(over)
        ops.paged_attention_q8(a["q"], code, code, scale, scale, a["table"], a["lens"], a["cu"],
                               a["page"], a["longest"], 1.0, a["hkv"], 16)

    with pytest.raises(ValueError, match="CUDA"):
        attend()
    for over, match in ((dict(longest=33), "max_seqlen"), (dict(cu=at), "cu_seqlens_q"),
                        (dict(q=x), "rows, heads"), (dict(hkv=2), "divide"),
                        (dict(lens=at.long()), "cache_seqlens"), (dict(table=at), "page_table")):
        with pytest.raises(ValueError, match=match):
            attend(**over)
    with pytest.raises(ValueError, match="columns"):
        ops.rope_store_kv_q8(x, at, torch.zeros(4, 128), 1, 1, 128, code, code, scale, scale, at,
                             16)


def test_workspace_size_is_host_only() -> None:
    size = LIB.lsb_paged_attention_q8_workspace_size
    assert size(1, 16, 16, 128) > 0 and size(1, 3, 2, 128) == 0 and size(0, 1, 1, 128) == 0


@pytest.mark.parametrize("amax,scale", [(448.0, 1.0), (448.5, 2.0), (1.0, 2.0 ** -8), (0.0, 0.0),
                                        (1.75, 2.0 ** -8), (1.76, 2.0 ** -7)])
def test_e4m3_scale_is_the_least_power_of_two(amax, scale) -> None:
    assert Q.needed_scale(amax, False) == scale
