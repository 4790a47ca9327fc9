"""The paged 4-bit KV cache in 64-bit numpy, from its definition (include/tilemix_hip.h): quantised
rows, page tables one request and one page at a time, attention one row at a time."""
from __future__ import annotations

import numpy as np

GROUP = 32
LIMIT = 65408.0


def width(dim: int) -> int:
    return -(-dim // GROUP) * GROUP


def quantise(x: np.ndarray):
    """Rows x [..., dim] (float64): codes uint8 [..., width / 2] and params fp16 [..., width / 32, 2]."""
    dim, w = x.shape[-1], width(x.shape[-1])
    codes = np.zeros((*x.shape[:-1], w), dtype=np.uint8)
    params = np.zeros((*x.shape[:-1], w // GROUP, 2), dtype=np.float16)
    for g in range(w // GROUP):
        part = np.clip(x[..., g * GROUP:(g + 1) * GROUP], -LIMIT, LIMIT)
        nan = np.isnan(part).any(-1)
        low, high = np.where(nan, 0.0, part.min(-1)), np.where(nan, 0.0, part.max(-1))
        s = np.where(nan, 0.0, (high - low) / 15).astype(np.float16)
        m = np.where(nan, np.nan, low).astype(np.float16)
        params[..., g, 0], params[..., g, 1] = s, m
        step = s.astype(np.float64)[..., None]
        with np.errstate(invalid="ignore", divide="ignore"):
            n = np.rint((part - m.astype(np.float64)[..., None]) / step)
        n = np.where((step > 0) & ~nan[..., None], np.clip(n, 0, 15), 0.0)
        codes[..., g * GROUP:g * GROUP + part.shape[-1]] = np.where(np.isnan(n), 0, n).astype(np.uint8)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), params


def dequantise(codes: np.ndarray, params: np.ndarray, dim: int) -> np.ndarray:
    """The values (float64, each an fp16 number) of codes and params."""
    n = np.empty((*codes.shape[:-1], codes.shape[-1] * 2))
    n[..., 0::2], n[..., 1::2] = codes & 15, codes >> 4
    s, m = (np.repeat(params[..., i].astype(np.float64), GROUP, axis=-1) for i in (0, 1))
    with np.errstate(over="ignore", invalid="ignore"):
        return (n * s + m).astype(np.float16).astype(np.float64)[..., :dim]


def read_rows(codes, params, dim, row, length, pages, page_size):
    """Values [heads, length, dim] of the first `length` tokens that a block-table row names and which
    of them there are."""
    out = np.zeros((codes.shape[1], length, dim))
    there = np.zeros(length, dtype=bool)
    for t in range(length):
        page = int(row[t // page_size]) if t // page_size < len(row) else -1
        if 0 <= page < pages:
            out[:, t] = dequantise(codes[page, :, t % page_size], params[page, :, t % page_size], dim)
            there[t] = True
    return out, there


def attention(q, k_codes, k_params, v_codes, v_params, dim, table, lens, cu, max_q, max_k, causal, scale):
    """(out, |.| sum, largest sum of |q k| scale): float64 [tokens, heads, dim] twice and [tokens, heads].
    The second is softmax @ |v|, the third what rounding errors of the scores grow with."""
    pages, hk, page_size = k_codes.shape[:3]
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    size = np.zeros(q.shape[:2])
    group = q.shape[1] // hk
    for b in range(len(lens)):
        n = min(max(int(lens[b]), 0), max_k, table.shape[1] * page_size)
        k, there = read_rows(k_codes, k_params, dim, table[b], n, pages, page_size)
        v, _ = read_rows(v_codes, v_params, dim, table[b], n, pages, page_size)
        nq = min(cu[b + 1] - cu[b], max_q)
        for i in range(nq):
            seen = there & ((np.arange(n) <= n - nq + i) if causal else True)
            if not seen.any():
                continue
            for h in range(q.shape[1]):
                row = q[cu[b] + i, h]
                kk, vv = k[h // group][seen], v[h // group][seen]
                s = kk @ row * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[cu[b] + i, h] = p @ vv
                mag[cu[b] + i, h] = p @ np.abs(vv)
                size[cu[b] + i, h] = (np.abs(kk) @ np.abs(row)).max() * abs(scale)
    return out, mag, size


def extend(table, lens, stack, count, new, page_size, tokens):
    """Changes table, lens and stack (lists) and returns (slots, positions, cu, granted, count)."""
    slots, positions, ends, granted, used, top = [-1] * tokens, [0] * tokens, [0], [], 0, count
    for b, n in enumerate(new):
        start = ends[-1]
        ends.append(start + max(n, 0))
        old, grown = -(-lens[b] // page_size), -(-(lens[b] + max(n, 0)) // page_size)
        if n < 0 or ends[-1] > tokens or lens[b] + n > len(table[b]) * page_size:
            granted.append(0)
            continue
        used += grown - old
        if grown > old and used > top:
            granted.append(0)
            continue
        granted.append(1)
        for c in range(old, grown):
            count -= 1
            table[b][c] = stack[count]
        for i in range(n):
            at = lens[b] + i
            slots[start + i] = table[b][at // page_size] * page_size + at % page_size
            positions[start + i] = at
        lens[b] += n
    return slots, positions, [min(e, tokens) for e in ends], granted, count


def truncate(table, lens, stack, count, keep, page_size):
    """Changes table, lens and stack (lists); returns the count."""
    for b in reversed(range(len(lens))):
        kept = min(lens[b], max(keep[b], 0))
        for c in reversed(range(-(-kept // page_size), -(-lens[b] // page_size))):
            stack[count] = table[b][c]
            table[b][c] = -1
            count += 1
        lens[b] = kept
    return count
