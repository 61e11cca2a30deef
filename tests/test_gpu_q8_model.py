"""The 8-bit KV pools in the models and the attention backend, as serving uses them: prefill and
decode under every looped-KV policy against the oracle whose pool rounds the same way.

The models' bf16 tolerance (max |diff| <= 2e-2 * max |ref|) does not hold by itself here: a key
that two bf16 computations round 2^-8 apart may fall on either side of a border between two
codes, and then differs by a whole step (2^-3 of the value for e4m3). The oracle says how much
that is: its bf16 run is off its fp32 run by `floor`, the CUDA path by as much again, so by the
triangle inequality the two are within 2 * floor.
"""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

import replay
from __graft_entry__ import load_package
from oracle import model as om
from oracle import q8 as Q

load_package()
from loop_sglang_b200 import ops, plugins  # noqa: E402
from loop_sglang_b200.kvcache import LastExitedKVCacheQ8, MHAKVCacheQ8  # noqa: E402
from test_gpu_model import greedy_agrees, rel_err  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("name", sorted(replay.CB_CASES))
def test_cb_decode_over_an_8_bit_pool(name: str, code: str, monkeypatch) -> None:
    from loop_sglang_b200.model import LoopedDecoder

    make = LoopedDecoder.make_kv_cache
    made = []

    def make_q8(self, num_pages, page_size):
        made.append(make(self, num_pages, page_size, kv_dtype=CODES[code]))
        return made[-1]

    monkeypatch.setattr(LoopedDecoder, "make_kv_cache", make_q8)
    _, got = replay.gpu_replay_cb(name)
    block = made[0].block
    assert isinstance(made[0], (MHAKVCacheQ8, LastExitedKVCacheQ8))
    pool = replay.make_pool
    monkeypatch.setattr(replay, "make_pool", lambda model, pages, page, dtype: Q.quantised_pool(
        pool(model, pages, page, torch.float32), block, code == "int8"))
    _, ref, _ = replay.replay_cb(name, dtype=torch.bfloat16)
    _, fp32, _ = replay.replay_cb(name)
    for prefix, logits in got.items():
        tol = max(2e-2, 2 * rel_err(ref[prefix], fp32[prefix]))
        assert rel_err(logits, ref[prefix]) < tol, prefix
        assert greedy_agrees(logits, ref[prefix], tol), prefix
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_device_routed_cdb_engine_over_an_8_bit_pool(code: str, graph: bool, monkeypatch) -> None:
    """The CDB engine on 8-bit version slots, eager and as a CUDA graph, against the oracle
    whose slots round the same way: exit depths, version maps and tokens (up to near ties)."""
    import cdb_lockstep as cl
    from loop_sglang_b200.model import LoopedDecoder
    from test_gpu_cdb_engine import K, _setup, check_versions

    make, slot_pool = LoopedDecoder.make_kv_cache, om.SlotKVPool
    monkeypatch.setattr(LoopedDecoder, "make_kv_cache", lambda self, pages, page: make(
        self, pages, page, kv_dtype=CODES[code]))
    monkeypatch.setattr(cl, "SlotKVPool", lambda layout, pages, heads, d, dtype: Q.quantised_pool(
        slot_pool(layout, pages, heads, d, torch.float32), 1, code == "int8"))
    cfg, weights, sc = _setup(21)
    ref = cl.oracle_run(cfg, weights, sc)
    eng, kv = cl.gpu_run(replay.gpu_model(cfg, weights, "last_exited"), sc, graph=graph)
    assert isinstance(kv, LastExitedKVCacheQ8)
    toks, deps = eng.out_tokens.cpu(), eng.out_depths.cpu()
    for r in range(len(sc.prompts)):
        assert deps[r, :K].tolist() == ref["depths"][r]
        for k in range(K):
            assert cl.token_matches(int(toks[r, k]), ref["preds"][r][k],
                                    ref["topk"][r][k]) != "mismatch", (r, k)
    check_versions(kv, ref["pool"])
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_attention_backend_over_an_8_bit_pool(code: str) -> None:
    """``B200AttnBackend`` stores and attends through the pool: a prefill, then a decode step."""
    hq, hkv, d, page = 8, 2, 64, 16
    kv = MHAKVCacheQ8(hkv, 1, d, 9, page, DEV, dtype=CODES[code])
    table = torch.zeros(3, 64, dtype=torch.int32)
    table[1, :64] = torch.arange(page, page + 64)
    table[2, :64] = torch.arange(5 * page, 5 * page + 64)
    ctx = SimpleNamespace(page_size=page, page_table=table.to(DEV), kv_cache=kv)
    be = plugins.B200AttnBackend(SimpleNamespace(head_dim=d, num_kv_heads=hkv), ctx)
    pool = Q.quantised_pool(om.PagedKVPool(1, 9, page, hkv, d, torch.float32), kv.block,
                            code == "int8")
    from oracle import ops as O

    g = torch.Generator().manual_seed(0)
    for seq, ext in (([21, 40], [21, 40]), ([22, 41], [1, 1])):
        t = sum(ext)
        pos = torch.cat([torch.arange(s - e, s) for s, e in zip(seq, ext)])
        loc = table[torch.repeat_interleave(torch.tensor([1, 2]), torch.tensor(ext)), pos]
        q = torch.randn(t, hq, d, generator=g).bfloat16()
        k, v = (torch.randn(t, hkv * d, generator=g).bfloat16() for _ in range(2))
        b = SimpleNamespace(is_decode=ext == [1, 1], is_prefill=ext != [1, 1],
                            size=2, padded_size=2, seq_lens_cpu=seq, extend_lens_cpu=ext,
                            seq_lens=torch.tensor(seq, dtype=torch.int32, device=DEV),
                            extend_lens=torch.tensor(ext, dtype=torch.int32, device=DEV),
                            req_pool_indices=torch.tensor([1, 2], dtype=torch.int32, device=DEV),
                            out_loc=loc.to(DEV))
        be.prepare_metadata(b)
        got = be.forward(q.to(DEV), k.to(DEV), v.to(DEV), 0, b)
        pool.store(0, k, v, loc)
        cu = torch.tensor([0, ext[0], t], dtype=torch.int32)
        want = O.paged_attention(q, pool.k_cache(0), pool.v_cache(0), table[1:, ::page] // page,
                                 torch.tensor(seq, dtype=torch.int32), cu, d ** -0.5)
        # one bf16 rounding each side, and the kernel's f16 weights
        torch.testing.assert_close(got.float().cpu(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -9)
    with pytest.raises(NotImplementedError):
        kv.get_cpu_copy(torch.arange(3))
