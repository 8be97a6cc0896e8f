"""The 4-bit cache and paged attention from their definitions, in 64 bits on the CPU (tests only).

Written from the formulas in include/kvx.h, one row at a time where that is the
plainest form; slow and small by design.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
# Every finite e4m3 number from 0 up: 8 steps below 2^-6, then 8 to a binade, the last (480) not a number.
E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
E4M3 = E4M3[:127]


def _nearest_even(table: list[float], x: float) -> int:
    """Index of the nearest entry, the even index of two equally near; the last one holds all beyond it."""
    if x >= table[-1]:
        return len(table) - 1
    hi = next(i for i, v in enumerate(table) if v > x)
    lo = hi - 1
    up, down = table[hi] - x, x - table[lo]
    return hi if up < down or (up == down and hi % 2 == 0) else lo


def q4_encode_row(row: torch.Tensor) -> tuple[list[int], list[int]]:
    """(codes, scale bytes) of one row of elements (already divided by k_scale or v_scale)."""
    codes, scales = [], []
    for group in row.double().view(-1, 16):
        xs = group.tolist()
        if not all(math.isfinite(x) for x in xs):
            codes += [0] * 16
            scales.append(0x7F)
            continue
        s = _nearest_even(E4M3, max(abs(x) for x in xs) / 6)
        scales.append(s)
        for x in xs:
            c = _nearest_even(LEVELS, abs(x) / E4M3[s]) if s else 0
            negative = math.copysign(1.0, x) < 0 and s > 0
            codes.append(c | (8 if negative else 0))
    return codes, scales


def q4_decode(codes: list[int], scales: list[int]) -> list[float]:
    out = []
    for i, c in enumerate(codes):
        s = scales[i // 16]
        s = math.nan if s & 0x7F == 0x7F else E4M3[s]
        out.append((-1.0 if c & 8 else 1.0) * LEVELS[c & 7] * s)
    return out


def q4_write(cache: torch.Tensor, slot: int, head: int, codes: list[int], scales: list[int]) -> None:
    """Codes and scales of one row into a CPU page tensor [N, bs, H, row] of bytes."""
    N, bs, H, row = cache.shape
    D = row // 9 * 16
    page = cache[slot // bs].view(H, bs * row)[head]
    at = slot % bs
    half = torch.tensor([codes[i] | (codes[i + 1] << 4) for i in range(0, D, 2)], dtype=torch.uint8)
    page[at * (D // 2):(at + 1) * (D // 2)] = half
    page[bs * (D // 2) + at * (D // 16):bs * (D // 2) + (at + 1) * (D // 16)] = torch.tensor(scales, dtype=torch.uint8)


def q4_read(cache: torch.Tensor, slot: int, head: int) -> list[float]:
    N, bs, H, row = cache.shape
    D = row // 9 * 16
    page = cache[slot // bs].reshape(H, bs * row)[head]
    at = slot % bs
    half = page[at * (D // 2):(at + 1) * (D // 2)].tolist()
    codes = [c for b in half for c in (b & 15, b >> 4)]
    return q4_decode(codes, page[bs * (D // 2) + at * (D // 16):bs * (D // 2) + (at + 1) * (D // 16)].tolist())


def q4_cache_rows(cache: torch.Tensor) -> torch.Tensor:
    """A whole 4-bit cache [N, bs, H, row] as values [N, bs, H, D] in 64 bits."""
    N, bs, H, row = cache.shape
    D = row // 9 * 16
    flat = cache.reshape(N, H, bs * row)
    half = flat[:, :, :bs * D // 2].reshape(N, H, bs, D // 2).long()
    sc = flat[:, :, bs * D // 2:].reshape(N, H, bs, D // 16).long()
    levels = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64)
    scales = torch.tensor(E4M3 + [math.nan], dtype=torch.float64)
    codes = torch.stack((half & 15, half >> 4), -1).reshape(N, H, bs, D // 16, 16)
    x = levels[codes] * scales[sc][..., None]
    return x.reshape(N, H, bs, D).permute(0, 2, 1, 3)


@dataclass
class Attended:
    out: torch.Tensor      # [T, Hq, D], rows of no sequence 0
    mass: torch.Tensor     # sum of weight * |value|, same shape
    reach: float           # largest scale * sum |q||k| of a visible key
    keys: int              # most visible keys of a row
    top: float             # largest |value| of a visible key


def attention(q, k_cache, v_cache, tables, ctx, cu=None, window=None, sinks=0, scale=None) -> Attended:
    """q [T, Hq, D]; caches [N, bs, H, D]; tables and lengths as lists or CPU tensors."""
    q, kc, vc = q.double(), k_cache.double(), v_cache.double()
    T, Hq, D = q.shape
    bs, H = kc.shape[1], kc.shape[2]
    scale = D ** -0.5 if scale is None else scale
    ctx = [int(c) for c in ctx]
    cu = list(range(len(ctx) + 1)) if cu is None else [int(c) for c in cu]
    res = Attended(torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64), 0.0, 0, 0.0)
    for s, c in enumerate(ctx):
        n = cu[s + 1] - cu[s]
        j_all = torch.arange(c)
        if c:
            ids = torch.tensor([int(tables[s][j]) for j in range((c - 1) // bs + 1)])
            k_all, v_all = kc[ids[j_all // bs], j_all % bs], vc[ids[j_all // bs], j_all % bs]
        for t in range(n):
            p = c - n + t
            see = [j for j in range(min(p + 1, c)) if window is None or p - j < window or j < sinks]
            if not see:
                continue
            res.keys = max(res.keys, len(see))
            for h in range(Hq):
                k, v = k_all[see, h // (Hq // H)], v_all[see, h // (Hq // H)]
                row = q[cu[s] + t, h]
                w = torch.softmax(scale * (k @ row), 0)
                res.out[cu[s] + t, h] = (w[:, None] * v).sum(0)
                res.mass[cu[s] + t, h] = (w[:, None] * v.abs()).sum(0)
                res.reach = max(res.reach, float((scale * (k.abs() @ row.abs())).max()))
                res.top = max(res.top, float(v.abs().max()))
    return res
