"""What the wrappers of the 8-bit KV cache hand to the C entry points, with the launch replaced by
a recorder (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from __graft_entry__ import load_package

PKG = load_package()
from loop_sglang_b200 import ops  # noqa: E402

BF16 = torch.bfloat16


class Recorder:
    """Stands in for the launch. Page tables are read while the call's own copies live: as many
    columns as ``pages`` of every request's row, as the kernel walks them."""

    def __init__(self) -> None:
        self.pages, self.name, self.args, self.table = 0, "", (), []

    def __call__(self, device, name, *args) -> None:
        self.name, self.args = name, args
        if name == "lsb_paged_attention_q8":
            ids = ctypes.cast(args[12], ctypes.POINTER(ctypes.c_int32))
            stride, reqs = args[13], args[16]
            self.table = [[ids[r * stride + c] for c in range(self.pages)] for r in range(reqs)]


@pytest.fixture
def launch(monkeypatch) -> Recorder:
    recorder = Recorder()
    monkeypatch.setattr(ops, "_call_on", recorder)
    monkeypatch.setattr(ops, "_one_device", lambda *tensors: 0)
    monkeypatch.setattr(ops, "_q8_workspace_bytes", lambda *sizes: 64)
    return recorder


def attend(table, reqs=3, pages_of=16, hq=2, hkv=2, d=64, longest=None, q=None):
    layer = [torch.zeros(20 * pages_of, hkv * d, dtype=torch.int8) for _ in range(2)]
    scales = [torch.ones(20, hkv) for _ in range(2)]
    q = torch.zeros(reqs, hq, d, dtype=BF16) if q is None else q
    lens = torch.full((reqs,), 5, dtype=torch.int32)
    cu = torch.arange(reqs + 1, dtype=torch.int32)
    return ops.paged_attention_q8(q, *layer, *scales, table, lens, cu, pages_of,
                                  longest or table.shape[1] * pages_of, 1.0, hkv, pages_of)


def test_rows_of_a_page_table_that_overlap(launch) -> None:
    """Requests that share a row (stride 0) or a window of it (a stride below the width) are walked
    as they are, never past the tensor."""
    base = torch.arange(1, 41, dtype=torch.int32)
    for table in (base[:4].expand(3, -1), base.as_strided((3, 4), (1, 1)),
                  base.as_strided((3, 4), (3, 1)), base.as_strided((2, 5), (5, 1)),
                  base[:24].view(3, 8)[:, :4], base.as_strided((1, 4), (0, 1))):
        launch.pages = table.shape[1]
        attend(table, reqs=table.shape[0])
        assert launch.args[13] >= table.shape[1]
        assert launch.table == table.tolist(), table.stride()


def test_appends_of_no_tokens_want_no_pointers() -> None:
    """An empty tensor's pointer is null."""
    lib, at = PKG._lib.lib(), ctypes.c_void_p(64)
    before = PKG._lib.launch_count()
    assert lib.lsb_store_kv_q8(at, at, 1024, 64, at, at, 16, 0, None, 1024, None, 1024, None, 0, 8,
                               128, None) == 0
    assert lib.lsb_rope_store_kv_q8(None, 4096, None, 1024, None, at, 8, at, at, 1024, 64, at, at,
                                    16, 0, None, 0, 16, 8, 128, None) == 0
    assert PKG._lib.launch_count() == before


def test_strides_of_a_single_row_or_head_say_nothing(launch) -> None:
    """A tensor of one row, or of one head a row, may have any stride there."""
    d, hkv = 64, 2
    table = torch.tensor([[1, 2]], dtype=torch.int32)
    q = torch.zeros(2 * d, dtype=BF16).as_strided((1, 2, d), (d, d, 1))
    attend(table, reqs=1, q=q)
    assert launch.args[3] == 2 * d
    one_head = torch.zeros(3, 3 * d, dtype=BF16).as_strided((3, 1, d), (3 * d, 5, 1))
    attend(table.expand(3, -1), hq=1, hkv=1, q=one_head)
    assert launch.args[3] == 3 * d
    layer = [torch.zeros(32, hkv * d, dtype=torch.int8) for _ in range(2)]
    scales = [torch.ones(2, hkv) for _ in range(2)]
    at = torch.tensor([3], dtype=torch.int32)
    row = torch.zeros(4 * hkv * d, dtype=BF16)
    qkv = row.as_strided((1, 4 * hkv * d), (0, 1))
    ops.rope_store_kv_q8(qkv, at, torch.zeros(8, d), 2 * hkv, hkv, d, *layer, *scales, at, 16)
    assert launch.args[1] == 4 * hkv * d and launch.args[3] >= 2 * hkv * d
    kv = row.as_strided((1, hkv * d), (1, 1))
    ops.store_kv_q8(*layer, *scales, at, kv, kv, hkv, d, 16)
    assert launch.args[9] == hkv * d and launch.args[11] == hkv * d
