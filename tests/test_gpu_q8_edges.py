"""The 8-bit KV cache where state outlives a call or an item: many items of unequal halves on one
SM, blocks that had another owner, NaN codes inside a block, scores far below zero, empty calls.

Tolerances are those of the operators' other tests: half a step of each rounding on the way.
"""

from __future__ import annotations

import pytest
import torch

from __graft_entry__ import load_package
from oracle import q8 as Q

load_package()
from loop_sglang_b200 import ops  # noqa: E402
from loop_sglang_b200._lib import LSB_DEVERR_SLOT  # noqa: E402
from test_gpu_q8 import CODES, DEV, gen, kernel, random_layer  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def prompt_reference(q, k, v, v_scale, sm_scale):
    """One request's causal attention in fp64 on the device: q [n, hq, D], k, v [len, hkv, D]
    values, v_scale [len, hkv]. The output, the weighted mean of |v|, the largest sum of |q||k| of
    each row, and what the smallest step of the f16 weights can move the output by."""
    n, hq, d = q.shape
    length, hkv, _ = k.shape
    out, mean_abs, small = (torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
                            for _ in range(3))
    reach = torch.zeros(n, hq, dtype=torch.float64, device=q.device)
    later = torch.ones(n, length, dtype=torch.bool, device=q.device).triu(length - n + 1)
    for h in range(hq):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        s = (q[:, h].double() @ kh.T * sm_scale).masked_fill(later, -torch.inf)
        p = torch.softmax(s, -1)
        out[:, h], mean_abs[:, h] = p @ vh, p @ vh.abs()
        size = q[:, h].double().abs() @ kh.abs().T * abs(sm_scale)
        reach[:, h] = size.masked_fill(later, 0.0).amax(-1)
        # A weight w = p * v_scale is held in f16, scaled by a power of two that takes the row's
        # largest to 2^6 or more: below f16's normal numbers it is off by up to half of 2^-24, so
        # by 2^-25 / 2^6 = 2^-31 of the row's largest w, which the key's |code| multiplies.
        vs = v_scale[:, h // (hq // hkv)].double()
        codes = (vh / vs[:, None]).abs().cumsum(0)[length - n:]  # of the keys that a row sees
        small[:, h] = 2.0 ** -31 * (p * vs).amax(-1, keepdim=True) * codes
    return out, mean_abs, reach, small


@pytest.mark.parametrize("kernel", [1], indirect=True)
@pytest.mark.parametrize("code,hq,hkv,block", [("int8", 16, 16, 16), ("int8", 16, 16, 1),
                                               ("e4m3", 32, 16, 16)])
def test_items_without_a_second_half_before_items_with_one(kernel, code, hq, hkv, block) -> None:
    """Several items a CTA, the longest (first) ones blocks whose second 128 rows are empty:
    lengths 256 n + 16 and 256 n + 76. Scales differ by orders of magnitude from key to key, so
    that a scale of another tile or item shows."""
    g = gen(21)
    d, page = 128, 16
    lens = [1552, 1100, 1552, 76, 1100, 1552, 16]
    assert all(0 < n % 256 <= 128 for n in lens)
    width = -(-max(lens) // page)
    table = (1 + torch.randperm(len(lens) * width, generator=g)).view(len(lens), width).int()
    k, v, ks, vs = (x.to(DEV) for x in random_layer(g, (len(lens) * width + 1) * page, hkv, d,
                                                    block, code, spread=2.0))
    cu = torch.tensor([0] + lens).cumsum(0)
    q = (torch.randn(int(cu[-1]), hq, d, generator=g) / 8).bfloat16().to(DEV)
    kv, vv = (Q.codes_to_values(c, s, block, hkv) for c, s in ((k, ks), (v, vs)))
    args = (q, k, v, ks, vs, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
            cu.int().to(DEV), page, width * page, d ** -0.5, hkv, block)
    got = ops.paged_attention_q8(*args)
    for _ in range(20):  # whichever item a CTA takes next
        assert torch.equal(ops.paged_attention_q8(*args), got)
    for r, n in enumerate(lens):
        slots = (table[r].long()[torch.arange(n) // page] * page + torch.arange(n) % page).to(DEV)
        lo, hi = int(cu[r]), int(cu[r + 1])
        ref, mean_abs, reach, small = prompt_reference(q[lo:hi], kv[slots], vv[slots],
                                                       vs[slots // block], d ** -0.5)
        # D fp32 roundings of a score (twice: truncated sums), f16 weights, the bf16 output
        score = (2 * (d + 8) * 2.0 ** -23 * reach)[..., None]
        tol = 2.0 ** -8 * ref.abs() + mean_abs * (2.0 ** -10 + 4 * score) + small + 1e-30
        worst = float(((got[lo:hi].double() - ref).abs() - tol).max())
        assert worst <= 0, (r, worst)
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
def test_requests_that_share_a_row_of_the_page_table(kernel) -> None:
    """An expanded row, and rows that are windows of one list: what a table of their own gives."""
    g = gen(22)
    hq, hkv, d, page, rows = 4, 2, 64, 16, 3
    layer = [x.to(DEV) for x in random_layer(g, 9 * page, hkv, d, page, "e4m3")]
    ids = (1 + torch.randperm(8, generator=g)).int().to(DEV)
    q = torch.randn(3 * rows, hq, d, generator=g).bfloat16().to(DEV)
    lens = torch.tensor([64, 20, 51], dtype=torch.int32, device=DEV)
    cu = torch.arange(0, 3 * rows + 1, rows, dtype=torch.int32, device=DEV)

    def attend(table):
        return ops.paged_attention_q8(q, *layer, table, lens, cu, page, 64, d ** -0.5, hkv, page)

    for table in (ids[:4].expand(3, -1), ids.as_strided((3, 4), (2, 1))):
        assert torch.equal(attend(table), attend(table.clone(
            memory_format=torch.contiguous_format)))
    assert ops.device_error_word(reset=True) == 0


# tokens of the first call into each block and of the second, blocks: single tokens (a warp per few
# of them, and 16 a warp from 2^21 elements on), whole runs, runs longer than a warp holds
REUSE = [(1, 1, 5, 2, 64, 4), (1, 1, 5, 3, 96, 16), (3, 9, 40, 2, 128, 16), (1, 2, 600, 16, 128, 4),
         (20, 12, 3, 2, 128, 32), (1, 60, 2, 1, 64, 64), (50, 30, 70, 8, 128, 128),
         (1, 0, 600, 16, 128, 1), (1, 0, 7, 4, 32, 1)]


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("first,then,blocks,hkv,d,block", REUSE)
def test_a_block_that_had_another_owner_starts_afresh(code, first, then, blocks, hkv, d,
                                                      block) -> None:
    """Pages are handed on with their old scales, NaN and large ones. Heads of zeros at a block's
    first slot leave a scale of 0, which small values behind them then set."""
    g = gen(23)
    int8, slots = code == "int8", (blocks + 1) * block
    loc0 = 1 + torch.randperm(blocks, generator=g)  # the blocks
    stale = torch.tensor([float("nan"), 1e4, 3e-5]).repeat((blocks + 1) * hkv)
    layer = [torch.randint(0, 256, (slots, hkv * d), generator=g, dtype=torch.uint8).to(DEV)
             .view(CODES[code]) for _ in range(2)]
    scales = [stale[i: i + (blocks + 1) * hkv].view(blocks + 1, hkv).clone().to(DEV)
              for i in range(2)]
    values = [torch.zeros(slots, hkv, d, dtype=torch.float64) for _ in range(2)]
    want = [s.cpu() for s in scales]
    written = []
    for step, (lo, n) in enumerate(((0, first), (first, then))):
        loc = (loc0[:, None] * block + torch.arange(lo, lo + n)).flatten()
        if n == 0:
            continue
        x = [torch.randn(loc.numel(), hkv, d, generator=g) * (1e-3 if step else 1.0)
             for _ in range(2)]
        if step == 0:
            x[0][:, ::2] = 0.0
            x[1][:, -1:] = 0.0
        x = [t.bfloat16() for t in x]
        ops.store_kv_q8(*layer, *scales, loc.int().to(DEV), *(t.to(DEV) for t in x), hkv, d, block)
        written.append(loc)
        seen = torch.cat(written)
        for i in range(2):
            values[i], want[i] = Q.append(values[i], want[i], x[i].double(), loc, block, int8)
            got = scales[i].cpu().double()
            torch.testing.assert_close(got[loc0], want[i][loc0], rtol=2.0 ** -22 if int8 else 0,
                                       atol=0)
            held = Q.codes_to_values(layer[i].cpu(), scales[i].cpu(), block, hkv)[seen]
            s = want[i].repeat_interleave(block, 0)[seen][:, :, None]
            # a rounding of each call: half a step of the final scale, where the first call's codes
            # are expressed in it again half a step more; and the fp32 scale's, its inverse's and
            # the product's, 2^-22 of the value in all
            step_of = Q.half_step(values[i][seen], s * (1 + 2.0 ** -20), int8)
            err = (held - values[i][seen]).abs() - 2.0 ** -22 * values[i][seen].abs()
            assert float((err - (1 + step) * step_of).max()) <= 0
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
@pytest.mark.parametrize("block", [16, 4, 1])
def test_nan_codes_inside_a_block_reach_every_row_that_sees_them(kernel, block) -> None:
    """e4m3 0x7f and 0xff among V's and K's codes: rows at and behind the key are NaN, in tiles that
    some rows see whole and others in part, and the rows before it are as without it."""
    g = gen(24)
    hq = hkv = 2
    d, page, n = 64, 16, 330
    k, v, ks, vs = random_layer(g, (n // page + 2) * page, hkv, d, block, "e4m3")
    table = torch.arange(1, n // page + 2, dtype=torch.int32).view(1, -1).to(DEV)
    q = torch.randn(n, hq, d, generator=g).bfloat16().to(DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)

    def attend(k, v):
        return ops.paged_attention_q8(q, k.to(DEV), v.to(DEV), ks.to(DEV), vs.to(DEV), table, lens,
                                      cu, page, n, d ** -0.5, hkv, block).cpu()

    for which, key, head, dim, nan in ((1, 5, 0, 3, 0x7F), (1, 100, 1, 63, 0xFF),
                                       (1, 47, 0, 17, 0x7F), (1, 256, 1, 0, 0xFF),
                                       (0, 9, 1, 7, 0x7F), (0, 130, 0, 40, 0xFF)):
        bad, clean = (k.clone(), v.clone()), (k.clone(), v.clone())
        bad[which].view(torch.uint8)[page + key, head * d + dim] = nan
        clean[which].view(torch.uint8)[page + key, head * d + dim] = 0
        got, without = attend(*bad), attend(*clean)
        rows = torch.isnan(got[:, head])
        rows = rows.any(-1) if which == 0 else rows[:, dim]
        assert not rows[:key].any() and rows[key:].all(), (which, key)
        assert torch.equal(got[:key], without[:key])
        assert torch.equal(got[:, 1 - head], without[:, 1 - head])
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_scores_far_below_zero(kernel, code) -> None:
    """All of a row's scores near -10^31 and equal: the mean of the values, not zeros."""
    g = gen(25)
    d, page, n = 64, 16, 40
    k = torch.ones(4 * page, d).to(CODES[code])
    _, v, ks, vs = random_layer(g, 4 * page, 1, d, page, code)
    ks.fill_(1.0)
    q = torch.full((n, 2, d), -2.0 ** 100, dtype=torch.bfloat16)
    table = torch.tensor([[1, 2, 3]], dtype=torch.int32)
    got = ops.paged_attention_q8(q.to(DEV), k.to(DEV), v.to(DEV), ks.to(DEV), vs.to(DEV),
                                 table.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV),
                                 torch.tensor([0, n], dtype=torch.int32, device=DEV), page, n,
                                 d ** -0.5, 1, page)
    x = Q.codes_to_values(v, vs, page, 1)[page: page + n]
    count = torch.arange(1, n + 1)[:, None, None]
    want, size = x.cumsum(0) / count, x.abs().cumsum(0) / count
    # f16 weights (2^-11), their fp32 sums and exponentials, the bf16 output. And a key's score and
    # the log2 of its value scale are one fp32 number, which at 10^31 (a unit of 2^80) holds nothing
    # of the log2: a key's w = p * v_scale is then off by its value scale, so two keys' weights by
    # up to the ratio of the largest to the smallest, and each share of the mean by as much.
    of = vs[1:].repeat_interleave(page, 0)[:n, 0].double()
    ratio = torch.stack([of[: i + 1].max() / of[: i + 1].min() for i in range(n)])[:, None, None]
    err = (got.cpu().double() - want).abs() - 2.0 ** -8 * want.abs() \
        - (2.0 ** -10 + ratio - 1) * size
    assert float(err.max()) <= 0


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("power", [18, 24, 27, 60, 100])
def test_scores_so_large_that_one_key_has_all_the_weight(kernel, code, power) -> None:
    """Scores of 2^power times whole numbers that differ from key to key: every row's output is the
    value of its largest key, whatever the value scales."""
    g = gen(27)
    d, page, n = 128, 16, 100
    slots = (n // page + 2) * page
    whole = torch.tensor([float(i) for i in range(-127, 128)])
    if code == "e4m3":
        whole = whole[whole.to(CODES[code]).float() == whole]
    number = whole[torch.randperm(whole.numel(), generator=g)]
    number = number.repeat(3)[:slots] if code == "e4m3" else number[:slots]
    n = min(n, whole.numel())
    k = torch.zeros(slots, d)
    k[:, 0] = number
    k = k.to(CODES[code])
    _, v, _, vs = random_layer(g, slots, 1, d, 4, code, spread=3.0)
    ks = torch.ones(slots // 4, 1)
    q = torch.zeros(n, 2, d, dtype=torch.bfloat16)
    q[:, 0, 0], q[:, 1, 0] = 2.0 ** power, -(2.0 ** power)
    table = torch.arange(-(-slots // page), dtype=torch.int32).view(1, -1)
    got = ops.paged_attention_q8(q.to(DEV), k.to(DEV), v.to(DEV), ks.to(DEV), vs.to(DEV),
                                 table.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV),
                                 torch.tensor([0, n], dtype=torch.int32, device=DEV), page, n,
                                 1.0, 1, 4)
    x = Q.codes_to_values(v, vs, 4, 1)[:n, 0]
    for row in range(n):
        for head, sign in ((0, 1), (1, -1)):
            want = x[int((sign * number[: row + 1]).argmax())]
            err = (got[row, head].cpu().double() - want).abs()
            # the bf16 output, and the f16 weight over the fp32 one of the sum
            assert bool((err <= (2.0 ** -8 + 2.0 ** -10) * want.abs()).all()), (row, head)
    assert ops.device_error_word(reset=True) == 0


def test_calls_of_no_tokens() -> None:
    """An empty batch, as the bf16 pool's store takes it."""
    hq, hkv, d, block = 4, 2, 64, 16
    layer = [x.to(DEV) for x in random_layer(gen(26), 64, hkv, d, block, "int8")]
    before = [x.clone() for x in layer]
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    x = torch.empty(0, hkv * d, dtype=torch.bfloat16, device=DEV)
    ops.store_kv_q8(*layer, none, x, x, hkv, d, block)
    q = ops.rope_store_kv_q8(torch.empty(0, (hq + 2 * hkv) * d, dtype=torch.bfloat16, device=DEV),
                             none, torch.ones(4, d, device=DEV), hq, hkv, d, *layer, none, block)
    assert q.shape == (0, hq, d)
    cu = torch.zeros(1, dtype=torch.int32, device=DEV)
    o = ops.paged_attention_q8(q, *layer, torch.empty(0, 4, dtype=torch.int32, device=DEV), none,
                               cu, 16, 64, 1.0, hkv, block)
    assert o.shape == (0, hq, d)
    assert all(torch.equal(a, b) for a, b in zip(layer, before))


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,d,block,per_request,heads", [
    (16, 16, 128, 16, 13, 1), (40, 10, 64, 2, 20, 1), (16, 16, 128, 16, 133, 4),
    (20, 20, 96, 4, 111, 4), (32, 8, 64, 64, 170, 4), (24, 24, 32, 1, 95, 4)])
def test_each_path_of_large_appends_equals_single_requests(code, hq, hkv, d, block, per_request,
                                                           heads) -> None:
    """From 2^21 elements on a warp takes 16 tokens, and four heads in turn where that still makes
    4736 warps: bit for bit what a call per request gives, into blocks that had another owner."""
    g = gen(hq * d + block)
    reqs = 48
    tokens = reqs * per_request
    warps = -(-tokens // 16) * (2 * -(-hkv // 4) + -(-hq // 4))
    assert tokens * (hq + 2 * hkv) * d >= 2 ** 21 and (warps >= 4736) == (heads == 4)
    pages = -(-per_request // block) + 1
    slots = (1 + reqs * pages) * block
    ids = 1 + torch.randperm(reqs * pages, generator=g).view(reqs, pages)
    start = torch.arange(reqs) % block  # blocks begun, and continued from an earlier owner's scale
    pos = start[:, None] + torch.arange(per_request)
    loc = (torch.gather(ids, 1, pos // block) * block + pos % block).int().to(DEV)
    pos = pos.int().to(DEV)
    inv = 1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    angle = torch.arange(512, dtype=torch.float64)[:, None] * inv
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float().to(DEV)
    qkv = torch.randn(reqs, per_request, (hq + 2 * hkv) * d, generator=g)
    qkv *= torch.exp(torch.randn(reqs, per_request, 1, generator=g))
    qkv[::3, :, hq * d: (hq + 1) * d] = 0.0  # heads of zeros
    qkv = qkv.bfloat16().to(DEV)
    one = [x.to(DEV) for x in random_layer(g, slots, hkv, d, block, code, spread=2.0)]
    many = [x.clone() for x in one]
    q = torch.empty(tokens, hq, d, dtype=torch.bfloat16, device=DEV)
    ops.rope_store_kv_q8(qkv.view(tokens, -1), pos.flatten(), cos_sin, hq, hkv, d, *one,
                         loc.flatten(), block, q_out=q)
    for r in range(reqs):
        got = torch.empty(per_request, hq, d, dtype=torch.bfloat16, device=DEV)
        ops.rope_store_kv_q8(qkv[r], pos[r], cos_sin, hq, hkv, d, *many, loc[r], block, q_out=got)
        assert torch.equal(got, q.view(reqs, per_request, hq, d)[r])
    for x, y in zip(one, many):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("block", [1, 4, 16])
@pytest.mark.parametrize("sm_scale", [-0.7, 0.0, 0.7])
def test_any_sign_of_the_softmax_scale(kernel, code, block, sm_scale) -> None:
    """A negative scale turns the order of the scores around, 0 makes all keys count alike."""
    g = gen(28)
    hq, hkv, d, page, n = 2, 2, 64, 16, 300
    k, v, ks, vs = (x.to(DEV) for x in random_layer(g, (n // page + 2) * page, hkv, d, block, code))
    table = torch.arange(1, n // page + 2, dtype=torch.int32, device=DEV).view(1, -1)
    q = torch.randn(n, hq, d, generator=g).bfloat16().to(DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    got = ops.paged_attention_q8(q, k, v, ks, vs, table, lens, cu, page, n, sm_scale, hkv, block)
    kv, vv = (Q.codes_to_values(c, s, block, hkv)[page: page + n] for c, s in ((k, ks), (v, vs)))
    of = vs[torch.arange(page, page + n, device=DEV) // block]
    ref, mean_abs, reach, small = prompt_reference(q, kv, vv, of, sm_scale)
    score = 2 * (d + 8) * 2.0 ** -23 * reach
    if code == "int8":  # the decode kernel's q in 16-bit fixed point, 1 / 65000 of its largest
        size = kv.abs().sum(-1).amax(0).repeat_interleave(hq // hkv)
        score = score + q.double().abs().amax(-1) * size * abs(sm_scale) / 65000
    tol = 2.0 ** -8 * ref.abs() + mean_abs * (2.0 ** -10 + 4 * score[..., None]) + small + 1e-30
    assert float(((got.double() - ref).abs() - tol).max()) <= 0
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_more_single_rows_than_one_launch_takes(code) -> None:
    """4500 requests of one row each, on the decode kernel in three launches, some of no keys."""
    g = gen(29)
    hq, hkv, d, page, reqs = 2, 1, 32, 4, 4500
    lens = torch.randint(0, 40, (reqs,), generator=g)
    table = torch.randint(1, 64, (reqs, 10), generator=g).int()
    k, v, ks, vs = (x.to(DEV) for x in random_layer(g, 64 * page, hkv, d, page, code))
    q = torch.randn(reqs, hq, d, generator=g).bfloat16().to(DEV)
    got = ops.paged_attention_q8(q, k, v, ks, vs, table.to(DEV), lens.int().to(DEV),
                                 torch.arange(reqs + 1, dtype=torch.int32, device=DEV), page, 40,
                                 d ** -0.5, hkv, page)
    kv, vv = (Q.codes_to_values(c, s, page, hkv)[:, 0] for c, s in ((k, ks), (v, vs)))
    at = torch.arange(40)
    slot = (table.long()[:, at // page] * page + at % page).to(DEV)
    there = (at < lens[:, None]).to(DEV)[:, None]
    s = torch.einsum("bhd,bkd->bhk", q.double(), kv[slot]) * d ** -0.5
    p = torch.softmax(s.masked_fill(~there, -torch.inf), -1).nan_to_num(0.0)
    ref = torch.einsum("bhk,bkd->bhd", p, vv[slot])
    mean_abs = torch.einsum("bhk,bkd->bhd", p, vv[slot].abs())
    reach = torch.einsum("bhd,bkd->bhk", q.double().abs(), kv[slot].abs()).amax(-1) * d ** -0.5
    score = 2 * (d + 8) * 2.0 ** -23 * reach
    if code == "int8":  # q in 16-bit fixed point, off by 1 / 65000 of its largest element
        score = score + q.double().abs().amax(-1) * kv.abs().sum(-1).max() * d ** -0.5 / 65000
    tol = 2.0 ** -8 * ref.abs() + mean_abs * (2.0 ** -10 + 4 * score[..., None]) + 1e-30
    assert float(((got.double() - ref).abs() - tol).max()) <= 0
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
@pytest.mark.parametrize("slots", [1, 5, 20, 40])
def test_pools_smaller_than_a_page(kernel, slots) -> None:
    """Keys whose slots the pool does not have are skipped and flagged, as many as there may be."""
    g = gen(30)
    d, page, block, n = 64, 64, 4, 30
    k, v, ks, vs = random_layer(g, 64, 1, d, block, "int8")
    held = -(-slots // block)
    q = torch.randn(n, 1, d, generator=g).bfloat16()
    got = ops.paged_attention_q8(
        q.to(DEV), k[:slots].to(DEV), v[:slots].to(DEV), ks[:held].to(DEV), vs[:held].to(DEV),
        torch.zeros(1, 1, dtype=torch.int32, device=DEV),
        torch.tensor([n], dtype=torch.int32, device=DEV),
        torch.tensor([0, n], dtype=torch.int32, device=DEV), page, n, d ** -0.5, 1, block)
    assert ops.device_error_word(reset=True) == (LSB_DEVERR_SLOT if slots < n else 0)
    kv, vv = (Q.codes_to_values(c[:slots], s[:held], block, 1) for c, s in ((k, ks), (v, vs)))
    for row in range(n):
        m = min(row + 1, slots)
        s = (kv[:m, 0] @ q[row, 0].double()) * d ** -0.5
        p = torch.softmax(s, 0)
        want, size = p @ vv[:m, 0], p @ vv[:m, 0].abs()
        reach = float((kv[:m, 0].abs() @ q[row, 0].double().abs()).max()) * d ** -0.5
        fixed = float(q[row].double().abs().max() * kv.abs().sum(-1).max()) * d ** -0.5 / 65000
        tol = 2.0 ** -8 * want.abs() + size * (2.0 ** -10 + 8 * (d + 8) * 2.0 ** -23 * reach
                                               + 4 * fixed)
        assert bool(((got[row, 0].cpu().double() - want).abs() <= tol).all()), row
