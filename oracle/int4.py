"""The paged 4-bit KV cache in plain torch, for tests: the formula of a held row and the layout of a
page, written from their definition (``include/solort_attn.h``) with an address for every code, and
attention over it in 64 bits. Runs on any device.

Slots and block tables are those of the bf16 arena (``src/solort/cache/kv_cache.py:136-149``).
"""

from __future__ import annotations

import torch

HD, GROUP, BLOCK = 128, 32, 1280


def quantise(x: torch.Tensor):
    """Codes ``[..., 128]`` int64, scales and mids ``[..., 4]`` fp32 of rows ``x [..., 128]``: each step
    in fp32, as the definition has it."""
    x = x.float().reshape(*x.shape[:-1], 4, GROUP)
    lo, hi = x.amin(-1), x.amax(-1)
    mid = (lo * 0.5 + hi * 0.5).to(torch.bfloat16).float()
    need = torch.maximum(hi - mid, mid - lo)
    need = need / torch.full_like(need, 7.5)
    down = (need.view(torch.int32) >> 16) << 16  # bf16 towards zero; a step up unless exact
    scale = torch.where(down == need.view(torch.int32), down, down + 0x10000).view(torch.float32)
    div = torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    codes = torch.round((x - mid[..., None]) / div + 7.5).clamp(0, 15).long()
    return codes.reshape(*codes.shape[:-2], HD), scale, mid


def held(x: torch.Tensor) -> torch.Tensor:
    """The values the cache holds for ``x``, in 64 bits."""
    codes, scale, mid = quantise(x)
    return values(codes, scale, mid)


def values(codes, scale, mid) -> torch.Tensor:
    scale, mid = (t.double().repeat_interleave(GROUP, -1) for t in (scale, mid))
    return mid + scale * (codes.double() - 7.5)


def code_place(row: torch.Tensor, is_value: bool):
    """Byte in its 8-token block and shift in that byte of the codes of dims 0..127 of rows ``row``
    (0..7): ``[..., 128]`` and ``[128]``."""
    d = torch.arange(HD, device=row.device)
    i, g = row[..., None], d // 32
    if is_value:
        p, u, j = i // 2, d % 32 // 4, d % 4
        return 640 + 128 * p + 16 * (u ^ (2 * p)) + 4 * g + 2 * (i % 2) + j // 2, 4 * (j % 2)
    t, j = d % 32 // 8, d % 8
    return 64 * i + 16 * t + 4 * g + j // 2, 4 * (j % 2)


def meta_place(row: torch.Tensor, is_value: bool) -> torch.Tensor:
    """Byte of the scale of groups 0..3 of rows ``row``; the mid is two bytes behind it."""
    return (1152 if is_value else 512) + 16 * row[..., None] + 4 * torch.arange(4, device=row.device)


def _block(pages: torch.Tensor, slots: torch.Tensor, head: int) -> torch.Tensor:
    P = pages.shape[2] // 160
    return ((slots // P * pages.shape[1] + head) * pages.shape[2] + slots % P // 8 * BLOCK)[:, None]


def store(pages: torch.Tensor, slots: torch.Tensor, key: torch.Tensor, value: torch.Tensor) -> None:
    """Write rows ``[n, nkv, 128]`` to a contiguous arena ``[num_pages, nkv, 160 * P]``."""
    flat, row = pages.view(-1), slots % 8
    for h in range(pages.shape[1]):
        at = _block(pages, slots, h)
        for x, is_value in ((key[:, h], False), (value[:, h], True)):
            codes, scale, mid = quantise(x)
            byte, shift = code_place(row, is_value)
            for s in (0, 4):  # two dims share a byte
                lane = shift[0] == s if shift.dim() > 1 else shift == s
                where = at + byte[:, lane]
                kept = flat[where].long() & (0xF0 if s == 0 else 0x0F)
                flat[where] = (kept | codes[:, lane] << s).to(torch.uint8)
            for t, off in ((scale, 0), (mid, 2)):
                bits = t.to(torch.bfloat16).contiguous().view(torch.int16).long() & 0xFFFF
                where = at + meta_place(row, is_value) + off
                flat[where] = (bits & 255).to(torch.uint8)
                flat[where + 1] = (bits >> 8).to(torch.uint8)


def load(pages: torch.Tensor, slots: torch.Tensor, mids: bool = False):
    """Held rows ``[n, nkv, 128]`` of K and V in 64 bits (with ``mids``, also V's mids per dim)."""
    flat, row = pages.view(-1), slots % 8
    found: list[list[torch.Tensor]] = [[], [], []]
    for h in range(pages.shape[1]):
        at = _block(pages, slots, h)
        for is_value in (False, True):
            byte, shift = code_place(row, is_value)
            codes = flat[at + byte].long() >> shift & 15
            where = at + meta_place(row, is_value)
            scale, mid = (
                ((flat[where + o].long() | flat[where + o + 1].long() << 8) << 16).to(torch.int32).view(torch.float32)
                for o in (0, 2))
            found[int(is_value)].append(values(codes, scale, mid))
            if is_value:
                found[2].append(mid.double().repeat_interleave(GROUP, -1))
    k, v, m = (torch.stack(f, 1) for f in found)
    return (k, v, m) if mids else (k, v)


def slots_of(table: torch.Tensor, n: int, P: int) -> torch.Tensor:
    """Slots of positions ``0 .. n - 1`` of a sequence with pages ``table``."""
    at = torch.arange(n, device=table.device)
    return table.long()[at // P] * P + at % P


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_pos: int, scale: float,
              v_mid: torch.Tensor | None = None):
    """``q [t, nh, 128]`` against ``k, v [n, nkv, 128]`` in 64 bits: row ``i`` sees keys
    ``0 .. q_pos + i``; a row that sees none is zero. With ``v_mid`` also
    ``(sum p |v - mid|, sum p |v|)``, what the roundings inside an attention scale with."""
    t, nh, _ = q.shape
    n, nkv, _ = k.shape
    if n == 0:
        zero = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        return zero if v_mid is None else (zero, zero, zero)
    qd = q.double().reshape(t, nkv, nh // nkv, HD)
    s = torch.einsum("tkgd,nkd->tkgn", qd, k) * scale
    seen = torch.arange(n, device=q.device) <= q_pos + torch.arange(t, device=q.device)[:, None]
    s = torch.where(seen[:, None, None], s, -torch.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.where(seen[:, None, None], (s - torch.where(m.isinf(), 0, m)).exp(), 0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1, total)

    def product(x):
        return torch.einsum("tkgn,nkd->tkgd", p, x).reshape(t, nh, HD)

    if v_mid is None:
        return product(v)
    return product(v), product((v - v_mid).abs()), product(v.abs())


def prologue(qkv, qn, kn, eps, cos, sin, positions, nh: int, nkv: int):
    """``(q, k, v)`` rows of the fused projection: norm and rotation in fp32 with the mean of squares in
    64 bits, the form in which the append op defines the keys it quantises."""
    x = qkv.float().view(qkv.shape[0], nh + 2 * nkv, HD)
    c, s = cos[positions].float()[:, None], sin[positions].float()[:, None]
    done = []
    for y, w in ((x[:, :nh], qn), (x[:, nh:nh + nkv], kn)):
        r = 1 / (y.double().pow(2).mean(-1, keepdim=True) + float(torch.tensor(eps, dtype=torch.float32))).sqrt()
        y = y * r.float() * w.float()
        done.append(y * c + torch.cat([-y[..., 64:], y[..., :64]], -1) * s)
    return done[0], done[1], x[:, nh + nkv:]
