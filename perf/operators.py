"""Cases, plain forms and 64-bit definitions of the 8-bit KV cache operators.

Two operators over one paged KV layer whose keys and values are held in 8 bits (e4m3 or int8)
with one fp32 scale per block of tokens and KV head:

* append: the neox rotation of the q and k heads of a fused QKV projection, and the k and v
  heads quantised into their slots (``ops.rope_store_kv_q8``);
* attention: causal attention of query rows over the paged 8-bit layer, for single tokens and
  for prompts (``ops.paged_attention_q8``).

The value a code stands for is ``code * scale[slot // block, head]``. A block's scale is the
smallest that holds the largest magnitude seen in the block since its first slot was written:
``amax / 127`` for int8, the power of two with ``amax / scale <= 448`` for e4m3. When a later
token raises it, the block's earlier codes are re-expressed in the new scale.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn
CODE = {"e4m3": F8, "int8": torch.int8}


# ----------------------------------------------------------------------------- cases --

def _append(name, code, reqs, lo, hi, cached, hq, hkv, dim, page, block):
    return {"name": name, "op": "append", "code": code, "reqs": reqs, "lo": lo, "hi": hi,
            "cached": cached, "hq": hq, "hkv": hkv, "dim": dim, "page": page, "block": block}


def _attend(name, code, reqs, lo, hi, new, hq, hkv, dim, page, block):
    return {"name": name, "op": "attention", "code": code, "reqs": reqs, "lo": lo, "hi": hi,
            "new": new, "hq": hq, "hkv": hkv, "dim": dim, "page": page, "block": block}


def listed():
    return [
        # one request decoding alone: every launch is latency
        _append("append_one", "e4m3", 1, 1, 1, 700, 16, 16, 128, 16, 16),
        # a continuous-depth batch: one-token pages (version slots), so one scale per token
        _append("append_versions", "int8", 265, 1, 1, 1500, 16, 16, 128, 1, 1),
        # a continuous batch with grouped KV heads, each token somewhere inside its block
        _append("append_grouped", "int8", 143, 1, 1, 2304, 32, 8, 128, 16, 16),
        # a prompt batch; half of the requests continue a cached prefix that ends inside a block
        _append("append_prompt", "e4m3", 8, 512, 1552, 37, 16, 16, 128, 16, 16),
        # one short request decoding alone: latency
        _attend("decode_one", "e4m3", 1, 700, 700, 0, 16, 16, 128, 16, 16),
        # a full-depth continuous batch over 16-token pages
        _attend("decode_paged", "e4m3", 143, 512, 2304, 0, 16, 16, 128, 16, 16),
        # a continuous-depth batch over scattered one-token version slots
        _attend("decode_versions", "int8", 265, 257, 1535, 0, 16, 16, 128, 1, 1),
        # 55 heads of 96, the shared-KV recurrent model's shape
        _attend("decode_55x96", "e4m3", 64, 513, 1033, 0, 55, 55, 96, 16, 16),
        # a few long contexts with grouped heads
        _attend("decode_long", "int8", 4, 32768, 131072, 0, 32, 8, 128, 64, 64),
        # whole prompts, 8256 tokens in all
        _attend("prompt", "e4m3", 8, 512, 1552, -1, 16, 16, 128, 16, 16),
        # 512-token chunks of longer prompts over what is cached already
        _attend("prompt_chunk", "int8", 4, 2048, 8704, 512, 32, 8, 128, 16, 16),
        # short prompts of a small model: 8 heads of 64, 4-token pages
        _attend("prompt_small", "e4m3", 4, 7, 128, -1, 8, 8, 64, 4, 4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    code = rng.choice(["e4m3", "int8"])
    hq, hkv, dim = rng.choice([(16, 16, 128), (8, 8, 64), (32, 8, 128), (2, 2, 128), (55, 55, 96),
                               (12, 4, 64), (8, 1, 128), (4, 4, 32), (32, 2, 128)])
    page = rng.choice([1, 4, 16, 64])
    block = rng.choice([b for b in (1, 2, 4, 16, 64) if page % b == 0])
    kind = rng.choice(["append1", "append", "decode", "decode", "prompt", "chunk"])
    if kind == "append1":
        c = _append("", code, _log(rng, 1, 400), 1, 1, _log(rng, 1, 8000), hq, hkv, dim, page, block)
    elif kind == "append":
        hi = _log(rng, 2, 1500)
        c = _append("", code, rng.randint(1, 7), max(1, hi // 3), hi, _log(rng, 1, 300), hq, hkv,
                    dim, page, block)
    elif kind == "decode":
        hi = _log(rng, 1, 60000)
        reqs = _log(rng, 1, max(1, min(300, 100_000_000 // (hi * hkv * dim))))
        c = _attend("", code, reqs, max(1, hi // rng.randint(1, 6)), hi, 0, hq, hkv, dim, page,
                    block)
    elif kind == "prompt":
        hi = _log(rng, 2, 1500)
        c = _attend("", code, rng.randint(1, 6), max(1, hi // 3), hi, -1, hq, hkv, dim, page, block)
    else:
        hi = _log(rng, 40, 6000)
        c = _attend("", code, rng.randint(1, 3), max(2, hi // 2), hi,
                    _log(rng, 2, max(2, min(hi // 2, 400))), hq, hkv, dim, page, block)
    del c["name"]
    return c


def _spread(lo, hi, n):
    """n lengths from lo to hi, evenly spaced (one request alone has the longest)."""
    return np.array([hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)], np.int64)


def _lengths(case):
    """(keys, query rows) of each request."""
    if case["op"] == "append":
        rows = _spread(case["lo"], case["hi"], case["reqs"])
        if case["hi"] == 1:  # single tokens: contexts of every length up to `cached`
            return _spread(max(1, case["cached"] // 4), case["cached"], case["reqs"]) + 1, rows
        return rows + np.arange(case["reqs"]) % 2 * case["cached"], rows
    keys = _spread(case["lo"], case["hi"], case["reqs"])
    new = case["new"]
    rows = keys if new < 0 else np.minimum(keys, new) if new else np.ones_like(keys)
    return keys, rows


def work(case):
    keys, rows = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    t = int(rows.sum())
    if case["op"] == "append":
        blocks = int((-(-keys // case["block"]) - (keys - rows) // case["block"]).sum())
        # qkv read, q written, codes written, each token's angles, position and slot, the scales
        b = t * ((hq + 2 * hkv) * d * 2 + hq * d * 2 + 2 * hkv * d + d * 4 + 8) + 2 * blocks * hkv * 4
        return {"bytes": b, "flops": t * (3 * (hq + hkv) * d + 4 * hkv * d)}
    k = int(keys.sum())
    blocks = int((-(-keys // case["block"])).sum())
    pages = int((-(-keys // case["page"])).sum())
    b = 2 * t * hq * d * 2 + 2 * k * hkv * d + 2 * blocks * hkv * 4 + pages * 4
    seen = int((rows * keys - rows * (rows - 1) // 2).sum())  # (row, key) pairs
    return {"bytes": b, "flops": 4 * seen * hq * d}


# ---------------------------------------------------------------------------- inputs --

def _bits(x):
    return x.view(torch.int32)


def _scale_of(amax, code):
    """The smallest scale that holds amax (fp32)."""
    if code == "int8":
        return amax * (1.0 / 127.0)
    e = ((_bits(amax.contiguous()) + 0x1FFFFF) >> 23) - 8  # biased exponent of the power of two
    s = (e.clamp(min=1) << 23).view(torch.float32)
    return torch.where(amax > 0, s, torch.zeros_like(s))


def _inverse(s):
    return torch.where(s > 0, torch.reciprocal(s), torch.zeros_like(s))


def _encode(x, code):
    if code == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(F8)


def _put(cache, rows, codes):
    cache.view(torch.uint8)[rows] = codes.view(torch.uint8)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 31))
    hq, hkv, d, page, block = (case[k] for k in ("hq", "hkv", "dim", "page", "block"))
    code, append = case["code"], case["op"] == "append"
    keys, rows = _lengths(case)
    order = rng.permutation(case["reqs"])
    keys, rows = keys[order], rows[order]
    first = keys - rows
    # pages of each request; an append keeps only those that its tokens reach
    lo_page = first // page if append else np.zeros_like(keys)
    pages = -(-keys // page) - lo_page
    total = int(pages.sum())
    spare = 3
    ids = 1 + rng.permutation(total + spare)[:total]  # page 0 is the padding page
    ends = np.cumsum(pages)
    width = int(pages.max())
    col = np.arange(width)[None]
    at = np.minimum((ends - pages)[:, None] + col, total - 1)
    table = np.where(col < pages[:, None], ids[at], 0).astype(np.int32)
    req = np.repeat(np.arange(case["reqs"]), rows)
    pos = np.arange(int(rows.sum())) - np.repeat(np.cumsum(rows) - rows, rows) + first[req]
    slots = (1 + total + spare) * page
    loc = table[req, pos // page - lo_page[req]].astype(np.int64) * page + pos % page

    def put(a, dtype=torch.int32):
        return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).to(dev)

    def pool(written=None):
        """Codes and scales of random values: keys with a few strong channels per head, values
        without; with `written`, only the first `written[b]` tokens of block b hold any."""
        out = []
        for gain in (torch.exp(0.7 * torch.randn(hkv, d, device=dev, generator=g)), None):
            x = torch.randn(slots // block, block, hkv, d, device=dev, generator=g)
            if gain is not None:
                x *= gain
            if written is not None:
                x *= torch.arange(block, device=dev)[None, :, None, None] < written[:, None, None, None]
            s = _scale_of(x.abs().amax(dim=(1, 3)), code)
            x *= _inverse(s)[:, None, :, None]
            out += [_encode(x, code).view(slots, hkv * d), s]
        return out[0], out[2], out[1], out[3]

    st = {"op": case["op"], "code": code, "hq": hq, "hkv": hkv, "dim": d, "page": page,
          "block": block, "max_q": int(rows.max()), "max_seqlen": int(keys.max()),
          "scale": d ** -0.5}
    if append:
        written = np.zeros(slots // block, np.int64)
        head = np.concatenate([[0], np.cumsum(rows)[:-1]])
        written[loc[head] // block] = loc[head] % block
        st["k"], st["v"], st["ks"], st["vs"] = pool(put(written, torch.int64))
        st["qkv"] = torch.randn(len(loc), (hq + 2 * hkv) * d, device=dev, generator=g).to(BF16)
        st["qkv"][:, hq * d:(hq + hkv) * d] *= torch.exp(
            0.7 * torch.randn(hkv * d, device=dev, generator=g)).to(BF16)
        inv = 1e6 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        angle = torch.arange(int(keys.max()) + 1, device=dev, dtype=torch.float64)[:, None] * inv
        st["cos_sin"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        st["positions"], st["loc"] = put(pos), put(loc)
        st["q_out"] = torch.empty(len(loc), hq, d, device=dev, dtype=BF16)
    else:
        st["k"], st["v"], st["ks"], st["vs"] = pool()
        st["q"] = (1.5 * torch.randn(len(loc), hq, d, device=dev, generator=g)).to(BF16)
        st["table"], st["lens"] = put(table), put(keys)
        st["cu"] = put(np.concatenate([[0], np.cumsum(rows)]))
    return st


# --------------------------------------------------------------------------- one pass --

def _ops():
    from __graft_entry__ import load_package

    load_package()
    from loop_sglang_b200 import ops

    return ops


def run(st):
    if st["op"] == "append":
        if own:
            _ops().rope_store_kv_q8(st["qkv"], st["positions"], st["cos_sin"], st["hq"], st["hkv"],
                                    st["dim"], st["k"], st["v"], st["ks"], st["vs"], st["loc"],
                                    st["block"], q_out=st["q_out"])
        else:
            _plain_append(st)
        return {"q": st["q_out"], "k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}
    if own:
        return _ops().paged_attention_q8(st["q"], st["k"], st["v"], st["ks"], st["vs"], st["table"],
                                         st["lens"], st["cu"], st["page"], st["max_seqlen"],
                                         st["scale"], st["hkv"], st["block"])
    return _plain_attention(st)


def _plain_append(st):
    hq, hkv, d, n = st["hq"], st["hkv"], st["dim"], st["qkv"].shape[0]
    x = st["qkv"].view(n, hq + 2 * hkv, d).float()
    cs = st["cos_sin"][st["positions"].long()][:, None]
    c, s = cs[..., :d // 2], cs[..., d // 2:]
    x1, x2 = x[:, :hq + hkv, :d // 2], x[:, :hq + hkv, d // 2:]
    turned = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)
    st["q_out"].copy_(turned[:, :hq])
    _plain_store(st["k"], st["ks"], turned[:, hq:], st["loc"].long(), st["block"], st["code"])
    _plain_store(st["v"], st["vs"], x[:, hq + hkv:], st["loc"].long(), st["block"], st["code"])


def _plain_store(cache, scale, x, loc, block, code):
    n, hkv, d = x.shape
    blocks, where = torch.unique(loc // block, return_inverse=True)
    nb = blocks.numel()
    amax = torch.zeros(nb, hkv, device=x.device).index_reduce_(0, where, x.abs().amax(-1), "amax")
    first = torch.full((nb,), block, device=x.device).index_reduce_(0, where, loc % block, "amin")
    old = torch.where(first[:, None] > 0, scale[blocks], 0.0)
    new = torch.maximum(old, _scale_of(amax, code))
    scale[blocks] = new
    # what the blocks held already, in the new scale
    offset = torch.arange(block, device=x.device)
    rows = (blocks[:, None] * block + offset).view(-1)
    held = cache[rows].view(nb, block, hkv, d)
    ratio = torch.where(new > 0, old / new, 1.0)
    again = _encode(held.float() * ratio[:, None, :, None], code)
    earlier = (offset < first[:, None])[..., None] & (ratio < 1)[:, None]
    held = torch.where(earlier[..., None], again.view(torch.uint8), held.view(torch.uint8))
    _put(cache, rows, held.view(nb * block, hkv * d))
    _put(cache, loc, _encode(x * _inverse(new)[where][..., None], code).view(n, hkv * d))


def _plain_attention(st):
    hq, hkv, d, page, block = (st[k] for k in ("hq", "hkv", "dim", "page", "block"))
    lens, cu = st["lens"].long(), st["cu"].long()
    dev, nreq, nk, nq = lens.device, lens.numel(), st["max_seqlen"], st["max_q"]
    key = torch.arange(nk, device=dev)
    slot = st["table"].long()[:, key // page] * page + key % page  # [reqs, keys]
    there = key < lens[:, None]
    row = torch.arange(nq, device=dev)
    count = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + row).clamp(max=st["q"].shape[0] - 1)
    q = st["q"][at].float().view(nreq, nq, hkv, hq // hkv, d) * st["scale"]
    seen = there[:, None] & (key <= (lens - count)[:, None, None] + row[:, None])  # [reqs, q, keys]

    def values(cache, scale):
        x = cache[slot].float().view(nreq, nk, hkv, d)
        return x.mul_(scale[slot // block][..., None])

    s = torch.einsum("bqhgd,bkhd->bhgqk", q, values(st["k"], st["ks"]))
    s.masked_fill_(~seen[:, None, None], -math.inf)
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    total = s.sum(-1)  # [reqs, hkv, group, q]
    o = torch.einsum("bhgqk,bkhd->bhgqd", s, values(st["v"], st["vs"])) / total[..., None]
    o = o.permute(0, 3, 1, 2, 4).reshape(nreq, nq, hq, d).to(BF16)
    return o[row < count[:, None]]


# --------------------------------------------------------------- definition in 64 bits --

def exact(case, seed):
    st = prepare(case, seed)
    return _exact_append(st) if st["op"] == "append" else _exact_attention(st)


def _exact_append(st):
    hq, hkv, d, block = st["hq"], st["hkv"], st["dim"], st["block"]
    n = st["qkv"].shape[0]
    z = st["qkv"].double().view(n, -1, d)
    table = st["cos_sin"].double()[st["positions"].long()]
    turn = torch.complex(table[:, :d // 2], table[:, d // 2:])[:, None]
    pairs = torch.complex(z[:, :hq + hkv, :d // 2], z[:, :hq + hkv, d // 2:]) * turn
    rotated = torch.cat([pairs.real, pairs.imag], -1)
    out = {"q": rotated[:, :hq]}
    top = 127.0 if st["code"] == "int8" else 448.0
    loc = st["loc"].tolist()
    groups = {}
    for t, slot in enumerate(loc):
        groups.setdefault(slot // block, []).append((slot % block, t))
    names = list(groups)
    owner = torch.zeros(n, dtype=torch.long)
    for i, b in enumerate(names):
        owner[[t for _, t in groups[b]]] = i
    owner = owner.to(z.device)
    begin = torch.tensor([min(groups[b])[0] for b in names], device=z.device)
    index = torch.tensor(names, device=z.device)
    for x, cache, scale, name in ((rotated[:, hq:], st["k"], st["ks"], "k"),
                                  (z[:, hq + hkv:], st["v"], st["vs"], "v")):
        peak = torch.zeros(len(names), hkv, dtype=torch.float64, device=z.device)
        peak.scatter_reduce_(0, owner[:, None].expand(n, hkv), x.abs().max(-1)[0], "amax")
        need = peak / top
        if st["code"] == "e4m3":
            need = torch.exp2(torch.ceil(torch.log2(need)))
        before = scale.double()[index] * (begin > 0)[:, None]
        after = torch.maximum(before, need)
        scales = scale.double().clone()
        scales[index] = after
        codes = None
        if st["code"] == "e4m3":
            codes = cache.double().view(-1, hkv, d)
            for o in range(block):  # earlier tokens of the touched blocks
                slots = (index * block + o)[begin > o]
                codes[slots] *= (before / after)[begin > o][..., None]
            codes[st["loc"].long()] = x / after[owner][..., None]
            codes = codes.view(-1, hkv * d)
        out[name], out[name + "s"] = codes, scales
    return out


def _exact_attention(st):
    hq, hkv, d, page, block = (st[k] for k in ("hq", "hkv", "dim", "page", "block"))
    cu, out = st["cu"].tolist(), []
    for r, n in enumerate(st["lens"].tolist()):
        slots = torch.cat([torch.arange(p * page, (p + 1) * page)
                           for p in st["table"][r, :-(-n // page)].tolist()])[:n].to("cuda")
        rows = cu[r + 1] - cu[r]
        k = st["k"][slots].double().view(n, hkv, d) * st["ks"][slots // block].double()[..., None]
        v = st["v"][slots].double().view(n, hkv, d) * st["vs"][slots // block].double()[..., None]
        q = st["q"][cu[r]:cu[r + 1]].double()
        o = torch.empty(rows, hq, d, dtype=torch.float64, device="cuda")
        later = torch.ones(rows, n, dtype=torch.bool, device="cuda").triu(n - rows + 1)
        for h in range(hq):
            kh = h // (hq // hkv)
            s = (q[:, h] @ k[:, kh].T) / math.sqrt(d)
            o[:, h] = torch.softmax(s.masked_fill(later, -math.inf), -1) @ v[:, kh]
        out.append(o)
    return torch.cat(out)
