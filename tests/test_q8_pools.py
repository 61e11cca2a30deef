"""What the 8-bit KV pools say of themselves (no GPU)."""

from __future__ import annotations

import pytest
import torch

from __graft_entry__ import load_package

load_package()
from loop_sglang_b200.kvcache import LastExitedKVCache, LastExitedKVCacheQ8  # noqa: E402

SHAPES = [(24, 4, 20, 4, 16, 128), (9, 3, 9, 3, 5, 96), (6, 2, 4, 1, 2, 64)]


def storage(pool) -> int:
    names = ["_kv_buffer", "slot_map", "completed_depth", "_free_slots"]
    names += ["k_scale", "v_scale"] if hasattr(pool, "k_scale") else []
    return sum(getattr(pool, n).nbytes for n in names)


@pytest.mark.parametrize("layers,start,end,steps,hkv,d", SHAPES)
@pytest.mark.parametrize("kind", ["bf16", "q8"])
def test_memory_per_page_is_what_a_page_takes(kind, layers, start, end, steps, hkv, d) -> None:
    """The growth of a pool's storage with its pages, which callers size pools by."""
    make = LastExitedKVCache if kind == "bf16" else LastExitedKVCacheQ8
    size = [storage(make(hkv, layers, d, pages, start, end, steps, torch.device("cpu")))
            for pages in (5, 15)]
    args = (layers, end - start, steps, hkv * d * (2 if kind == "bf16" else 1))
    said = make.memory_per_page(*args) if kind == "bf16" else make.memory_per_page(*args, hkv)
    assert size[1] - size[0] == 10 * said
