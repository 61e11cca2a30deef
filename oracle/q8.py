"""The 8-bit KV cache in 64 bits: what an append leaves in a block, and attention over the
values its codes stand for. Written token by token and block by block, from the format's
definition alone.
"""

from __future__ import annotations

import math

import torch

E4M3_TOP, INT8_TOP = 448.0, 127.0
SMALLEST = 2.0 ** -126  # no scale of a block that holds something is below


def codes_to_values(codes: torch.Tensor, scale: torch.Tensor, block: int, hkv: int) -> torch.Tensor:
    """``[slots, hkv, D]`` fp64 values of a layer's codes ``[slots, hkv * D]``."""
    c = codes.float().double().view(codes.shape[0], hkv, -1)
    return c * scale.double().repeat_interleave(block, 0)[: c.shape[0], :, None]


def needed_scale(amax: float, int8: bool) -> float:
    """The scale a block needs for a largest magnitude ``amax``."""
    if not math.isfinite(amax):
        return math.nan
    if amax == 0:
        return 0.0
    if int8:
        return max(amax / INT8_TOP, SMALLEST)
    mantissa, exponent = math.frexp(amax / E4M3_TOP)  # 0.5 <= mantissa < 1
    return max(2.0 ** (exponent - 1 if mantissa == 0.5 else exponent), SMALLEST)


def half_step(value: torch.Tensor, scale: torch.Tensor, int8: bool) -> torch.Tensor:
    """How far a rounded code's value may be from ``value``: half a step of the code type."""
    if int8:
        return 0.5 * scale.expand_as(value)
    return torch.maximum(value.abs() * 2.0 ** -4, scale * 2.0 ** -10)


def rotate(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor) -> torch.Tensor:
    """Neox rotation of ``x [T, heads, D]`` in fp64 by the fp32 table's values."""
    half = x.shape[-1] // 2
    cs = cos_sin[positions.long()].double()[:, None]
    c, s = cs[..., :half], cs[..., half:]
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def append(held: torch.Tensor, scale: torch.Tensor, x: torch.Tensor, loc: torch.Tensor,
           block: int, int8: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """What a layer should hold after ``x [T, hkv, D]`` goes to slots ``loc``: the unrounded
    values ``[slots, hkv, D]`` and the scales. ``held`` are the values before."""
    held, scale = held.clone(), scale.double().clone()
    slots = held.shape[0]
    touched: dict[int, list[int]] = {}
    for t, s in enumerate(loc.tolist()):
        if 0 < s < slots:
            touched.setdefault(s // block, []).append(t)
    for b, tokens in touched.items():
        offsets = [int(loc[t]) % block for t in tokens]
        for h in range(x.shape[1]):
            need = needed_scale(float(x[tokens, h].abs().max()), int8)
            old = float(scale[b, h]) if min(offsets) > 0 else 0.0
            scale[b, h] = need if math.isnan(need) else max(old, need)
        for t in tokens:
            held[int(loc[t])] = x[t]
    return held, scale


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
              lens: torch.Tensor, cu: torch.Tensor, page: int, max_seqlen: int,
              sm_scale: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Causal attention in fp64 over the layer's values ``k``, ``v [slots, hkv, D]``. Returns
    the output ``[rows, hq, D]``, the weighted mean of ``|v|`` (what a relative error of the
    weights can move the output by), the largest ``sum |q||k| * sm_scale`` of each row and
    head (what a relative error of the products can move a score by) and which rows belong to
    a request."""
    rows, hq, d = q.shape
    group = hq // k.shape[1]
    out = torch.zeros(rows, hq, d, dtype=torch.float64)
    mean_abs = torch.zeros_like(out)
    reach = torch.zeros(rows, hq, dtype=torch.float64)
    owned = torch.zeros(rows, dtype=torch.bool)
    for b in range(lens.numel()):
        lo, hi = int(cu[b]), int(cu[b + 1])
        n = min(int(lens[b]), max_seqlen)
        for r in range(lo, min(hi, rows)):
            owned[r] = True
            sees = n - (hi - 1 - r)
            if sees <= 0:
                continue
            slots = torch.tensor([int(table[b, j // page]) * page + j % page for j in range(sees)])
            ok = (slots >= 0) & (slots < k.shape[0])
            slots = slots[ok]
            if slots.numel() == 0:
                continue
            kk = k[slots].repeat_interleave(group, 1)
            vv = v[slots].repeat_interleave(group, 1)
            qq = q[r].double()
            p = torch.softmax(torch.einsum("hd,khd->hk", qq, kk) * sm_scale, -1)
            out[r] = torch.einsum("hk,khd->hd", p, vv)
            mean_abs[r] = torch.einsum("hk,khd->hd", p, vv.abs())
            reach[r] = (torch.einsum("hd,khd->hk", qq.abs(), kk.abs()) * sm_scale).amax(-1)
    return out, mean_abs, reach, owned


def round_values(values: torch.Tensor, scale: torch.Tensor, block: int,
                 int8: bool) -> torch.Tensor:
    """``[slots, hkv, D]`` values as their codes hold them."""
    s = scale.double().repeat_interleave(block, 0)[: values.shape[0], :, None]
    x = torch.where(s > 0, values / s, 0.0)
    if int8:
        return x.round().clamp(-INT8_TOP, INT8_TOP) * s
    return x.clamp(-E4M3_TOP, E4M3_TOP).float().to(torch.float8_e4m3fn).float().double() * s


def quantised_pool(pool, block: int, int8: bool):
    """An oracle KV pool (fp32) whose stores round as an 8-bit pool's do."""
    scales: dict[tuple[int, int], torch.Tensor] = {}

    def store(layer, k, v, out_loc) -> None:
        for x, cache in ((k, pool.k_cache(layer)), (v, pool.v_cache(layer))):
            flat = cache.view(-1, *cache.shape[-2:])
            key = (flat.data_ptr(), flat.shape[0])
            scale = scales.get(key)
            if scale is None:
                scale = torch.zeros(-(-flat.shape[0] // block), flat.shape[1], dtype=torch.float64)
            held, scales[key] = append(flat.double(), scale,
                                       x.double().reshape(-1, *flat.shape[1:]), out_loc, block,
                                       int8)
            flat.copy_(round_values(held, scales[key], block, int8))

    pool.store = store
    return pool
