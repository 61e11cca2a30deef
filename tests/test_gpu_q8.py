"""The 8-bit KV cache's append and attention against their definition in 64 bits (oracle.q8).

Tolerances count the roundings on the way: half a step of the output type (bf16 2^-8, e4m3 2^-4,
int8 half a scale), f16 weights 2^-11, fp32 sums of D products 2^-23 each.
"""

from __future__ import annotations

import pytest
import torch

from __graft_entry__ import load_package
from oracle import q8 as Q

load_package()
from loop_sglang_b200 import ops  # noqa: E402
from loop_sglang_b200._lib import LSB_DEVERR_POSITION, LSB_DEVERR_SEQLEN, LSB_DEVERR_SLOT  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def gen(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def table_of(max_pos: int, d: int) -> torch.Tensor:
    inv = 1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def empty_layer(slots: int, hkv: int, d: int, block: int, code: str):
    return [torch.zeros(slots, hkv * d, dtype=torch.uint8, device=DEV).view(CODES[code])
            for _ in range(2)] + [torch.zeros(-(-slots // block), hkv, device=DEV)
                                  for _ in range(2)]


def check_layer(cache, scale, before, after, scales, written, block, hkv, int8, slack):
    """Scales and codes of one of K / V after an append: ``after`` the unrounded values,
    ``before`` what the layer held, ``written`` the slots of the call."""
    got = Q.codes_to_values(cache.cpu(), scale.cpu(), block, hkv)
    s = scales.repeat_interleave(block, 0)[: after.shape[0], :, None]
    # int8: amax / 127 in fp32; e4m3: a power of two, exact
    torch.testing.assert_close(scale.cpu().double(), scales, rtol=2.0 ** -22 if int8 else 0, atol=0)
    # half a step, plus the fp32 roundings of the scale, its inverse and value * inverse: each
    # at most 2^-24 of the value (of up to 127 steps), so 3 * 2^-24 |value| < 2^-22 |value|
    step = Q.half_step(after, s * (1 + 2.0 ** -20), int8) + 2.0 ** -22 * after.abs()
    new = torch.zeros(after.shape[0], dtype=torch.bool)
    new[written] = True
    over = (got - after).abs() - step
    worst = float((over - slack)[new].max())
    assert worst <= 0, worst
    # earlier tokens of a block: rounded again only where the scale grew
    worst = float(over[~new].max())
    assert worst <= 0, worst


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,d,page,block", [(16, 16, 128, 16, 16), (8, 2, 64, 4, 4),
                                                 (5, 5, 96, 1, 1), (4, 4, 32, 64, 64),
                                                 (6, 3, 96, 16, 2), (8, 1, 128, 128, 128)])
def test_append_in_steps(code, hq, hkv, d, page, block) -> None:
    """A prompt, then single tokens, then a chunk, into scattered pages: scales and values
    after every call, the q heads, and everything not written left as it was."""
    g = gen(hq * d + block)
    int8 = code == "int8"
    reqs, max_pos = 3, 400
    pages = -(-max_pos // page)
    slots = (1 + reqs * pages) * page
    ids = 1 + torch.randperm(reqs * pages, generator=g).view(reqs, pages)
    k, v, ks, vs = empty_layer(slots, hkv, d, block, code)
    cos_sin = table_of(max_pos, d)
    lens = [0] * reqs
    for step, counts in enumerate([[21, 1, 150], [1, 1, 1], [1, 1, 1], [0, 40, 7], [1, 0, 1]]):
        pos = torch.cat([torch.arange(n, n + c) for n, c in zip(lens, counts)]).int()
        req = torch.cat([torch.full((c,), r) for r, c in enumerate(counts)])
        lens = [n + c for n, c in zip(lens, counts)]
        loc = (ids[req, pos // page] * page + pos % page).int()
        t = pos.numel()
        # magnitudes vary, so scales grow inside blocks; a head of zeros; a wider row stride
        wide = torch.randn(t, (hq + 2 * hkv) * d + 16, generator=g)
        wide *= torch.exp(torch.randn(t, 1, generator=g))
        wide[:, hq * d: hq * d + d] *= step % 2
        wide = wide.bfloat16().to(DEV)
        qkv = wide[:, : (hq + 2 * hkv) * d]
        raw = qkv.cpu().view(t, -1, d)
        turned = Q.rotate(raw[:, : hq + hkv], pos, cos_sin)
        # fp32 products and sums of the rotation
        size = raw[:, : hq + hkv].double().abs()
        slack = 2.0 ** -22 * (size + size.roll(d // 2, -1))
        before = [Q.codes_to_values(c.cpu(), s.cpu(), block, hkv) for c, s in ((k, ks), (v, vs))]
        scales0 = [ks.cpu(), vs.cpu()]
        q = ops.rope_store_kv_q8(qkv, pos.to(DEV), cos_sin.to(DEV), hq, hkv, d, k, v, ks, vs,
                                 loc.to(DEV), block,
                                 q_out=None if step % 2 else torch.empty(t, hq, d, device=DEV,
                                                                         dtype=torch.bfloat16))
        err = (q.cpu().double() - turned[:, :hq]).abs()
        assert bool((err <= 2.0 ** -8 * turned[:, :hq].abs() + slack[:, :hq] + 1e-38).all())
        assert torch.equal(wide.cpu()[:, hq * d: (hq + 2 * hkv) * d].view(t, -1, d), raw[:, hq:])
        for i, (cache, scale, x) in enumerate(((k, ks, turned[:, hq:]),
                                               (v, vs, raw[:, hq + hkv:].double()))):
            after, want = Q.append(before[i], scales0[i], x, loc, block, int8)
            full = torch.zeros_like(after)
            if i == 0:
                full[loc.long()] = slack[:, hq:]
            check_layer(cache, scale, before[i], after, want, loc.long(), block, hkv, int8, full)
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,d,block", [(16, 16, 128, 16), (20, 20, 96, 4), (40, 10, 64, 2),
                                            (17, 17, 128, 1), (24, 24, 32, 64),
                                            (32, 8, 128, 32)])
def test_large_append_equals_its_requests(code, hq, hkv, d, block) -> None:
    """A call of many tokens gives what a call per request gives, bit for bit: runs that end
    inside a warp's tokens, blocks begun by an earlier call (with scales that grow), tokens of a
    block in another order than their slots, padding between requests."""
    g = gen(hq * d + block)
    reqs, t = 48, 0
    pages = 4 * (128 // block)  # blocks per request
    slots = (1 + reqs * pages) * block
    ids = 1 + torch.randperm(reqs * pages, generator=g).view(reqs, pages)
    cos_sin = table_of(1024, d).to(DEV)
    layers = [empty_layer(slots, hkv, d, block, code) for _ in range(2)]
    held = torch.randint(0, 40, (reqs,), generator=g)
    for step in range(2):
        counts = held if step == 0 else torch.randint(1, 230, (reqs,), generator=g)
        parts = []
        for r in range(reqs):
            pos = torch.arange(int(counts[r])) + (int(held[r]) if step else 0)
            if step and r % 5 == 0:  # the tokens of each block backwards
                order = sorted(range(len(pos)), key=lambda i: (int(pos[i]) // block, -int(pos[i])))
                pos = pos[torch.tensor(order, dtype=torch.long)]
            loc = ids[r, pos // block] * block + pos % block
            if step and r % 3 == 0:  # padding behind the request
                pos, loc = torch.cat([pos, pos[:1]]), torch.cat([loc, torch.zeros(1).long()])
            parts.append((pos.int(), loc.int()))
        t = sum(len(pos) for pos, _ in parts)
        assert t > 0
        qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=g) * torch.exp(
            torch.randn(t, 1, generator=g))
        qkv = qkv.bfloat16().to(DEV)
        if step:  # the path of large calls: 16 tokens of a head for 4736 warps
            assert t * (hq + 2 * hkv) >= 16 * 4736
        q = [torch.empty(t, hq, d, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
        pos, loc = (torch.cat(x).to(DEV) for x in zip(*parts))
        k, v, ks, vs = layers[0]
        ops.rope_store_kv_q8(qkv, pos, cos_sin, hq, hkv, d, k, v, ks, vs, loc, block, q_out=q[0])
        k, v, ks, vs = layers[1]
        at = 0
        for pos, loc in parts:
            n = len(pos)
            if n:
                ops.rope_store_kv_q8(qkv[at: at + n], pos.to(DEV), cos_sin, hq, hkv, d, k, v, ks,
                                     vs, loc.to(DEV), block, q_out=q[1][at: at + n])
            at += n
        assert torch.equal(q[0], q[1])
        for x, y in zip(*layers):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_store_matches_append_without_rotation(code) -> None:
    """store_kv_q8 of rotated rows equals rope_store_kv_q8 at position 0 (angle 0)."""
    g = gen(3)
    hq, hkv, d, block, t = 4, 2, 64, 8, 29
    qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=g).bfloat16().to(DEV)
    loc = torch.arange(19, 19 + t, dtype=torch.int32, device=DEV)
    cos_sin = table_of(4, d).to(DEV)
    zero = torch.zeros(t, dtype=torch.int32, device=DEV)
    a, b = empty_layer(64, hkv, d, block, code), empty_layer(64, hkv, d, block, code)
    ops.rope_store_kv_q8(qkv, zero, cos_sin, hq, hkv, d, a[0], a[1], a[2], a[3], loc, block)
    kv = qkv[:, hq * d:]
    ops.store_kv_q8(b[0], b[1], b[2], b[3], loc, kv[:, : hkv * d], kv[:, hkv * d:], hkv, d, block)
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("block", [1, 16])
def test_append_bad_slots_positions_and_values(code, block) -> None:
    """Slot 0 is skipped, slots and positions out of range are flagged and skipped; a value
    that is not finite makes its block NaN and no other."""
    hkv, d, slots = 2, 64, 64
    k, v, ks, vs = empty_layer(slots, hkv, d, block, code)
    x = torch.ones(5, hkv * d, dtype=torch.bfloat16, device=DEV)
    loc = torch.tensor([0, 64, -3, 17, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    ops.store_kv_q8(k, v, ks, vs, loc, x, x, hkv, d, block)
    assert ops.device_error_word(reset=True) == LSB_DEVERR_SLOT
    held = k.float().view(slots, -1).abs().sum(1) > 0
    assert held.nonzero().flatten().tolist() == [17]
    assert (ks > 0).sum() == hkv
    bad = x[:2].clone()
    bad[0, 5], bad[1, d + 1] = float("inf"), float("nan")
    at = torch.tensor([32, 48], dtype=torch.int32, device=DEV)
    ops.store_kv_q8(k, v, ks, vs, at, bad, x[:2], hkv, d, block)
    nan = torch.isnan(ks).nonzero().tolist()
    assert nan == [[32 // block, 0], [48 // block, 1]] and not torch.isnan(vs).any()
    ops.store_kv_q8(k, v, ks, vs, at, x[:2], x[:2], hkv, d, block)  # starts afresh
    assert not torch.isnan(ks).any()
    qkv = torch.ones(1, 3 * hkv * d, dtype=torch.bfloat16, device=DEV)
    ops.rope_store_kv_q8(qkv, torch.tensor([9], dtype=torch.int32, device=DEV),
                         table_of(9, d).to(DEV), hkv, hkv, d, k, v, ks, vs, at[:1], block)
    assert ops.device_error_word(reset=True) == LSB_DEVERR_POSITION


def random_layer(g, slots, hkv, d, block, code, spread=0.3, row=None):
    """A layer of random codes (rows of ``row`` codes, the first hkv * d used) and scales."""
    row = row or hkv * d
    out = []
    for _ in range(2):
        if code == "int8":
            c = torch.randint(-127, 128, (slots, row), generator=g, dtype=torch.int8)
        else:
            c = (torch.randn(slots, row, generator=g) * 100).clamp(-448, 448).to(CODES["e4m3"])
        s = torch.exp(spread * torch.randn(-(-slots // block), hkv, generator=g)) / 100
        out.append((c, s))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def check_attention(got, q, k, v, ks, vs, table, lens, cu, page, max_seqlen, hkv, block, before):
    d = q.shape[2]
    kv, vv = (Q.codes_to_values(c[:, : hkv * d], s, block, hkv) for c, s in ((k, ks), (v, vs)))
    ref, mean_abs, reach, owned = Q.attention(q.float(), kv, vv, table, lens, cu, page,
                                              max_seqlen, d ** -0.5)
    # scores off by D fp32 roundings (twice: truncated sums), weights by twice that and 2^-11
    score = 2 * (d + 8) * 2.0 ** -23 * reach
    if k.dtype == torch.int8:
        # q in 16-bit fixed point with its largest element at 32500: each element is off by at
        # most half a unit, 1 / 65000 of the largest, which a key multiplies by sum |k|
        size = kv.nan_to_num(0.0).abs().sum(-1).amax(0).repeat_interleave(q.shape[1] // hkv)
        score = score + q.double().abs().amax(-1) * size * d ** -0.5 / 65000
    score = score[..., None]
    tol = 2.0 ** -8 * ref.abs() + mean_abs * (2.0 ** -10 + 4 * score) + 1e-30
    err = (got.cpu().double() - ref).abs()
    worst = float((err - tol)[owned].max()) if owned.any() else 0.0
    assert worst <= 0, f"off by {worst:.3e} beyond the bound (largest error {float(err.max()):.3e})"
    assert torch.equal(got.cpu()[~owned], before[~owned]), "rows behind the last request changed"


def attention_case(code, hq, hkv, d, page, block, lens, new, *, seed=0, max_seqlen=None,
                   spread=0.3, pad_rows=0, row=None, qpad=0, poison=False):
    g = gen(seed + hq + d + page)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    counts = [new(n) if callable(new) else new for n in lens]
    cu = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).int()
    rows = int(cu[-1]) + pad_rows
    longest = max(max(lens), 1)
    max_seqlen = max_seqlen or longest
    width = -(-max(longest, max_seqlen) // page)
    total = len(lens) * width
    slots = (total + 1) * page
    table = (1 + torch.randperm(total, generator=g)).view(len(lens), width).int()
    k, v, ks, vs = random_layer(g, slots, hkv, d, block, code, spread, row)
    if poison:  # everything no row may see: NaN codes and scales
        seen = torch.zeros(slots, dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(n):
                seen[int(table[b, j // page]) * page + j % page] = True
        dead = ~seen.view(-1, block).any(1)
        ks[dead], vs[dead] = float("nan"), float("nan")
        if code == "e4m3":
            for c in (k, v):
                c.view(torch.uint8)[~seen] = 0x7F
    q = torch.randn(rows, hq * d + qpad, generator=g).bfloat16()[:, : hq * d].view(rows, hq, d)
    before = torch.randn(rows, hq, d, generator=g).bfloat16()
    out = before.to(DEV)
    qd = torch.zeros(rows, hq * d + qpad, dtype=torch.bfloat16, device=DEV)
    qd[:, : hq * d] = q.reshape(rows, hq * d).to(DEV)
    qd = qd[:, : hq * d].view(rows, hq, d) if qpad == 0 else \
        qd.as_strided((rows, hq, d), (hq * d + qpad, d, 1))
    cut = (lambda c: c.to(DEV)[:, : hkv * d])
    got = ops.paged_attention_q8(qd, cut(k), cut(v), ks.to(DEV), vs.to(DEV), table.to(DEV),
                                 lens_t.to(DEV), cu.to(DEV), page, max_seqlen, d ** -0.5, hkv,
                                 block, out=out)
    assert got.data_ptr() == out.data_ptr()
    check_attention(got, q, k, v, ks, vs, table, lens_t, cu, page, max_seqlen, hkv, block, before)
    return got


SHAPES = [(16, 16, 128, 16, 16), (8, 8, 64, 4, 4), (55, 55, 96, 16, 16), (4, 4, 32, 64, 32),
          (32, 8, 128, 16, 1), (8, 1, 128, 1, 1), (24, 2, 96, 12, 4), (3, 3, 64, 1, 1),
          (40, 2, 64, 16, 8)]


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,d,page,block", SHAPES)
def test_decode_rows(code, hq, hkv, d, page, block) -> None:
    """One query row per request: contexts of nothing, one key, around tile, page and share
    boundaries, in one call; nothing beyond a context is read."""
    attention_case(code, hq, hkv, d, page, block,
                   [1, 0, 16, 17, 2, 15, 33, 64, 65, 300, 0, 129, 1], 1, poison=True)
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,d,page,block", SHAPES)
def test_prompt_rows(code, hq, hkv, d, page, block) -> None:
    """Several query rows per request, with and without cached keys, rows that see nothing
    (more rows than keys) and rows behind the last request."""
    attention_case(code, hq, hkv, d, page, block, [37, 5, 130, 1], lambda n: max(1, n // 2 + 3),
                   pad_rows=3, poison=True)
    attention_case(code, hq, hkv, d, page, block, [70, 3, 0], lambda n: n + 2, seed=1)
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_long_rows_are_split_and_merged(code) -> None:
    attention_case(code, 4, 2, 128, 64, 64, [9000, 3, 4097], 1)
    attention_case(code, 1, 1, 128, 1, 1, [5000], 1)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_scales_of_very_different_sizes(code) -> None:
    """Scales spread over e^(+-30): the weight and the value scale stay together."""
    attention_case(code, 4, 4, 128, 16, 4, [200, 64], 1, spread=8.0)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_strides_and_padded_rows(code) -> None:
    attention_case(code, 8, 4, 64, 16, 16, [40, 18, 77], 1, pad_rows=2, row=4 * 64 + 32, qpad=24)
    attention_case(code, 8, 4, 64, 16, 16, [40, 18, 77], 5, pad_rows=2, row=4 * 64 + 32, qpad=24)


def test_unequal_rows_that_count_as_many_as_requests() -> None:
    """As many rows as requests, but not one each: [2, 0, 1] rows."""
    counts = iter([2, 0, 1])
    attention_case("e4m3", 4, 4, 64, 4, 4, [20, 9, 33], lambda n: next(counts))


@pytest.mark.parametrize("new", [1, 4])
def test_long_context_is_cut_and_bad_pages_are_skipped(new) -> None:
    attention_case("int8", 4, 4, 64, 16, 16, [50, 20], new, max_seqlen=32)
    assert ops.device_error_word(reset=True) == LSB_DEVERR_SEQLEN
    g = gen(5)
    hq = hkv = 4
    d, page, block = 64, 16, 16
    k, v, ks, vs = random_layer(g, 6 * page, hkv, d, block, "int8")
    table = torch.tensor([[1, 900, 3, -7], [2, 2, 2, 2]], dtype=torch.int32)
    lens = torch.tensor([64, 20], dtype=torch.int32)
    cu = torch.tensor([0, new, 2 * new], dtype=torch.int32)
    q = torch.randn(2 * new, hq, d, generator=g).bfloat16()
    got = ops.paged_attention_q8(q.to(DEV), k.to(DEV), v.to(DEV), ks.to(DEV), vs.to(DEV),
                                 table.to(DEV), lens.to(DEV), cu.to(DEV), page, 64, d ** -0.5,
                                 hkv, block)
    check_attention(got, q, k, v, ks, vs, table, lens, cu, page, 64, hkv, block, q)
    assert ops.device_error_word(reset=True) == LSB_DEVERR_SLOT


def test_append_then_attend_captured_and_on_another_stream() -> None:
    """The two as a model runs them, eagerly, on a side stream and in a replayed graph: the
    same bits each time, and two graphs replayed at once keep apart."""
    g = gen(11)
    hq, hkv, d, page, block, reqs = 8, 4, 128, 16, 16, 5
    lens0 = torch.tensor([30, 5, 200, 63, 1])
    width = 16
    table = (1 + torch.randperm(reqs * width, generator=g)).view(reqs, width).int()
    cos_sin = table_of(512, d).to(DEV)
    k, v, ks, vs = random_layer(g, (reqs * width + 1) * page, hkv, d, block, "e4m3")
    qkv = torch.randn(reqs, (hq + 2 * hkv) * d, generator=g).bfloat16().to(DEV)
    pos = lens0.int().to(DEV)
    loc = (table[torch.arange(reqs), lens0 // page] * page + lens0 % page).int().to(DEV)
    lens = (lens0 + 1).int().to(DEV)
    cu = torch.arange(reqs + 1, dtype=torch.int32, device=DEV)
    tab = table.to(DEV)

    def layer():
        return [x.to(DEV) for x in (k, v, ks, vs)]

    def step(lay):
        q = torch.empty(reqs, hq, d, dtype=torch.bfloat16, device=DEV)
        ops.rope_store_kv_q8(qkv, pos, cos_sin, hq, hkv, d, *lay, loc, block, q_out=q)
        return ops.paged_attention_q8(q, *lay, tab, lens, cu, page, width * page, d ** -0.5, hkv,
                                      block)

    first = layer()
    want = step(first)
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    on_side = layer()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = step(on_side)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):
        lay = layer()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(lay)
        graphs.append((graph, res, lay))
    for _ in range(20):
        for s, (graph, _, _) in zip((side, other), graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, res, lay in graphs:
        assert torch.equal(res, want)
        for a, b in zip(lay, first):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert ops.device_error_word(reset=True) == 0


@pytest.fixture
def kernel(request):
    """Every call on the prompt kernel (1), or every call on the decode kernel (2)."""
    from loop_sglang_b200._lib import call

    call("lsb_attention_force_kernel", request.param)
    yield request.param
    call("lsb_attention_force_kernel", 0)


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,d,page,block", SHAPES)
def test_either_kernel_takes_any_rows(kernel, code, hq, hkv, d, page, block) -> None:
    """Both kernels on the same calls: single rows, prompts, rows that see nothing, rows behind
    the last request, NaN wherever no row may look."""
    attention_case(code, hq, hkv, d, page, block, [1, 0, 16, 65, 130], 1, poison=True)
    attention_case(code, hq, hkv, d, page, block, [1, 70, 130, 0, 64, 5], lambda n: n // 2 + 3,
                   pad_rows=2, poison=True, seed=3)
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("kernel", [1], indirect=True)
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 128), (6, 1, 96), (8, 2, 64), (2, 1, 32)])
def test_prompt_kernel_over_several_blocks_of_rows(kernel, code, hq, hkv, d) -> None:
    """Requests of more than one block of 256 packed rows, whole and continued, and scales that
    differ by e^(+-24)."""
    attention_case(code, hq, hkv, d, 16, 16, [600, 700], lambda n: n if n == 600 else 150)
    attention_case(code, hq, hkv, d, 16, 2, [200, 40], lambda n: n, spread=8.0)
    attention_case(code, hq, hkv, d, 4, 1, [333], lambda n: 300, qpad=8, pad_rows=1)
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
def test_nan_keys_reach_the_rows_that_see_them_and_no_other(kernel) -> None:
    """A key whose codes (e4m3 0x7f) or scales are NaN in the middle of a prompt."""
    g = gen(8)
    hq = hkv = 2
    d, page, n = 64, 1, 150
    k, v, ks, vs = random_layer(g, n + 1, hkv, d, 1, "e4m3")
    v.view(torch.uint8)[71, 5] = 0x7F          # head 0 of the key at position 70
    vs[101, 1] = float("nan")                  # head 1 of the key at position 100
    table = torch.arange(1, n + 1, dtype=torch.int32).view(1, -1)
    q = torch.randn(n, hq, d, generator=g).bfloat16()
    out = ops.paged_attention_q8(q.to(DEV), k.to(DEV), v.to(DEV), ks.to(DEV), vs.to(DEV),
                                 table.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV),
                                 torch.tensor([0, n], dtype=torch.int32, device=DEV), page, n,
                                 d ** -0.5, hkv, 1).cpu()
    bad = torch.isnan(out)
    assert not bad[:70, 0].any() and bad[70:, 0, 5].all()
    assert not bad[:100, 1].any() and bad[100:, 1].all()
    k2, v2, ks2, vs2 = k.clone(), v.clone(), ks.clone(), vs.clone()
    v2.view(torch.uint8)[71, 5] = 0
    vs2[101, 1] = 1.0
    clean = ops.paged_attention_q8(q.to(DEV), k2.to(DEV), v2.to(DEV), ks2.to(DEV), vs2.to(DEV),
                                   table.to(DEV),
                                   torch.tensor([n], dtype=torch.int32, device=DEV),
                                   torch.tensor([0, n], dtype=torch.int32, device=DEV), page, n,
                                   d ** -0.5, hkv, 1).cpu()
    assert torch.equal(out[:70, 0], clean[:70, 0]) and torch.equal(out[:100, 1], clean[:100, 1])


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_every_code_counts_as_its_value(kernel, code, d) -> None:
    """All codes of both types (but NaN, and int8's unused -128) in K and in V, in every place."""
    n, page = 256, 16
    codes = torch.arange(256, dtype=torch.int32)
    codes = codes[(codes & 127) != 127] if code == "e4m3" else codes[codes != 128]
    at = (torch.arange(n + page)[:, None] * 5 + torch.arange(d) * 3) % codes.numel()
    k = codes[at].to(torch.uint8).view(CODES[code])
    v = codes[(at + 7) % codes.numel()].to(torch.uint8).view(CODES[code])
    scale = torch.full((n // page + 1, 1), 2.0 ** -7)
    table = torch.arange(1, n // page + 1, dtype=torch.int32).view(1, -1)
    lens, cu = torch.tensor([n], dtype=torch.int32), torch.tensor([0, 40], dtype=torch.int32)
    q = torch.randn(40, 2, d, generator=gen(d)).bfloat16() / 8
    before = torch.zeros(40, 2, d, dtype=torch.bfloat16)
    got = ops.paged_attention_q8(q.to(DEV), k.to(DEV), v.to(DEV), scale.to(DEV), scale.to(DEV),
                                 table.to(DEV), lens.to(DEV), cu.to(DEV), page, n, d ** -0.5, 1,
                                 page)
    check_attention(got, q, k, v, scale, scale, table, lens, cu, page, n, 1, page, before)


@pytest.mark.parametrize("kernel", [1], indirect=True)
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,d,page,block", [(4, 4, 32, 16, 16), (6, 2, 64, 12, 4),
                                                 (3, 1, 96, 32, 2), (4, 2, 128, 128, 64),
                                                 (2, 2, 128, 8, 8)])
def test_prompt_kernel_over_many_requests(kernel, code, hq, hkv, d, page, block) -> None:
    """More requests than lanes and more blocks of rows than CTAs at a time: whole and continued
    prompts, empty ones between them, more keys than one round of 32 pages."""
    g = gen(11)
    lens = torch.randint(0, 90, (75,), generator=g).tolist()
    lens[3], lens[40], lens[74] = 900, 2100, 260
    counts = iter([0 if i % 9 == 4 else int(torch.randint(1, 60, (1,), generator=g)) if i % 3
                   else max(n, 1) for i, n in enumerate(lens)])
    attention_case(code, hq, hkv, d, page, block, lens, lambda n: next(counts), pad_rows=4)
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
def test_a_pool_that_ends_inside_a_block(kernel) -> None:
    """Slots past the pool's last are skipped and flagged, block and page or not."""
    g = gen(12)
    hq = hkv = 2
    d, page, n = 64, 16, 64
    k, v, ks, vs = random_layer(g, 64 + page, hkv, d, page, "int8")
    slots = 64 + page - 6  # the last page has 10 slots
    table = torch.tensor([[1, 2, 3, 4]], dtype=torch.int32)
    q = torch.randn(3, hq, d, generator=g).bfloat16()
    args = (ks.to(DEV), vs.to(DEV), table.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV),
            torch.tensor([0, 3], dtype=torch.int32, device=DEV), page, n, d ** -0.5, hkv, page)
    got = ops.paged_attention_q8(q.to(DEV), k[:slots].to(DEV), v[:slots].to(DEV), *args)
    assert ops.device_error_word(reset=True) == LSB_DEVERR_SLOT
    # as if the request had the keys that are there (all three rows see those)
    short = ops.paged_attention_q8(q.to(DEV), k.to(DEV), v.to(DEV), *args[:3],
                                   torch.tensor([n - 6 + 2], dtype=torch.int32, device=DEV),
                                   *args[4:])
    torch.testing.assert_close(got[0].float(), short[0].float(), rtol=2 * 2.0 ** -8, atol=2e-3)
    assert bool(torch.isfinite(got.float()).all())


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_slots_beyond_four_gigabytes(kernel, code) -> None:
    """Append and attention at the end of a pool whose offsets pass 32 bits: the bits of the same
    in a small pool."""
    g = gen(13)
    hq, hkv, d, page, n = 4, 2, 128, 16, 150
    row, slots = 65536, 66048  # 4.3 GB each of K and V
    first = slots // page - 12
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g).bfloat16().to(DEV)
    cos_sin = table_of(256, d).to(DEV)
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    order = torch.randperm(12, generator=g).int()
    outs = []
    for wide in (False, True):
        base = first if wide else 1
        table = (base + order).view(1, -1).to(DEV)
        loc = (table[0].cpu().long()[torch.arange(n) // page] * page + torch.arange(n) % page)
        count = slots if wide else 13 * page
        k, v = (torch.empty(count, row if wide else hkv * d, dtype=torch.uint8, device=DEV)
                .view(CODES[code])[:, : hkv * d] for _ in range(2))
        ks, vs = (torch.zeros(count // page, hkv, device=DEV) for _ in range(2))
        q = torch.empty(n, hq, d, dtype=torch.bfloat16, device=DEV)
        ops.rope_store_kv_q8(qkv, pos, cos_sin, hq, hkv, d, k, v, ks, vs, loc.int().to(DEV), page,
                             q_out=q)
        out = ops.paged_attention_q8(q, k, v, ks, vs, table,
                                     torch.tensor([n], dtype=torch.int32, device=DEV),
                                     torch.tensor([0, n], dtype=torch.int32, device=DEV), page,
                                     12 * page, d ** -0.5, hkv, page)
        held = torch.cat([x.view(torch.uint8)[loc.to(DEV)] for x in (k, v)])
        outs.append((out.cpu(), held.cpu()))
        del k, v
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("kernel", [1], indirect=True)
def test_more_heads_to_a_kv_head_than_rows_of_a_tile(kernel) -> None:
    """Groups of 136 heads (no whole positions to a tile of 128 rows) and of 128 and 256."""
    for hq in (136, 128, 256):
        attention_case("e4m3", hq, 1, 32, 16, 16, [40, 3], lambda n: min(n, 7), pad_rows=1,
                       poison=True)
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("kernel", [1], indirect=True)
def test_prompts_in_graphs_on_two_streams(kernel) -> None:
    """Two captured calls replayed at once, eager ones between them: the same bits throughout."""
    g = gen(14)
    hq, hkv, d, page = 8, 4, 128, 16
    lens = torch.tensor([700, 90, 300], dtype=torch.int32)
    cu = torch.tensor([0, 700, 720, 1020], dtype=torch.int32).to(DEV)
    width = 44
    table = (1 + torch.randperm(3 * width, generator=g)).view(3, width).int().to(DEV)
    layer = [x.to(DEV) for x in random_layer(g, (3 * width + 1) * page, hkv, d, page, "int8")]
    qs = [torch.randn(1020, hq, d, generator=g).bfloat16().to(DEV) for _ in range(2)]
    lens = lens.to(DEV)

    def attend(q):
        return ops.paged_attention_q8(q, *layer, table, lens, cu, page, width * page, d ** -0.5,
                                      hkv, page)

    want = [attend(q) for q in qs]
    graphs = []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = attend(q)
        graphs.append((graph, res))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(10):
        for s, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        assert torch.equal(attend(qs[i % 2]), want[i % 2])
    torch.cuda.synchronize()
    for (_, res), w in zip(graphs, want):
        assert torch.equal(res, w)
    assert ops.device_error_word(reset=True) == 0


@pytest.mark.parametrize("kernel", [1, 2], indirect=True)
def test_rows_of_no_request_are_left_alone(kernel) -> None:
    """Rows before the first request's and behind the last one's; the others as without them."""
    g = gen(15)
    hq = hkv = 2
    d, page = 64, 16
    layer = [x.to(DEV) for x in random_layer(g, 5 * page, hkv, d, page, "e4m3")]
    table = torch.tensor([[1, 2], [3, 4]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([30, 9], dtype=torch.int32, device=DEV)
    q = torch.randn(10, hq, d, generator=g).bfloat16().to(DEV)
    before = torch.randn(10, hq, d, generator=g).bfloat16().to(DEV)

    def attend(q, cu, out):
        return ops.paged_attention_q8(q, *layer, table, lens,
                                      torch.tensor(cu, dtype=torch.int32, device=DEV), page, 32,
                                      d ** -0.5, hkv, page, out=out)

    got = attend(q, [2, 5, 9], before.clone())
    want = attend(q[2:9], [0, 3, 7], torch.empty_like(q[2:9]))
    assert torch.equal(got[2:9], want)
    assert torch.equal(got[:2], before[:2]) and torch.equal(got[9:], before[9:])
    assert ops.device_error_word(reset=True) == 0
