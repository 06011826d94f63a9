"""The 8-bit key/value cache and the attention over it in 64 bits, from the definitions.

A row x of one token and head is held as whole numbers c = 127 x / max|x| (to the nearest, ties to even) and the
scale max|x| / 127 in fp32.  Rows whose largest value is below 2^-119 are zeros; a row with an infinity or a NaN
has the scale NaN.  Caches here are plain: codes (B, Hkv, S, D) int64, scales (B, Hkv, S) float64.
"""
from __future__ import annotations

import torch


def encode(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of rows x."""
    x = x.double()
    top = x.abs().amax(dim=-1)  # NaN where the row holds one
    bad, tiny = ~torch.isfinite(top), top < 2.0**-119
    safe = torch.where(bad | tiny, torch.ones_like(top), top)
    codes = torch.round(127 * torch.where((bad | tiny)[..., None], torch.zeros_like(x), x) / safe[..., None])
    scales = torch.where(tiny, torch.zeros_like(top), (top.float() / torch.full_like(top, 127).float()).double())
    return codes.long(), torch.where(bad, torch.full_like(top, float("nan")), scales)


def positions(T: int, starts: list[int], counts: list[int], capacity: int) -> list[list[int]]:
    """Each token's position, -1 for padding."""
    return [[s + t if t < n and 0 <= s + t < capacity else -1 for t in range(T)] for s, n in zip(starts, counts)]


def write(codes, scales, x: torch.Tensor, starts: list[int], counts: list[int]) -> None:
    """Stores x (B, T, Hkv, D) in a plain cache, in place."""
    c, s = encode(x)
    for b, row in enumerate(positions(x.shape[1], starts, counts, codes.shape[2])):
        for t, p in enumerate(row):
            if p >= 0:
                codes[b, :, p] = c[b, t]
                scales[b, :, p] = s[b, t]


def read(codes, scales, T: int, starts: list[int], counts: list[int]) -> torch.Tensor:
    """(B, T, Hkv, D) values in 64 bits."""
    B, Hkv, S, D = codes.shape
    out = torch.zeros(B, T, Hkv, D, dtype=torch.float64)
    for b, row in enumerate(positions(T, starts, counts, S)):
        for t, p in enumerate(row):
            if p >= 0:
                out[b, t] = codes[b, :, p] * scales[b, :, p, None]
    return out


def attention(q, k, v, starts, counts, window=None, scale=None, prefix=None):
    """(o, a, s, v): the output (B, T, H, D); the sums of p |v|; of each row the largest scale sum_d |q_d k_d| and the largest
    value scale that it sees.

    k and v are plain caches; prefix a pair of them of batch 1, cut to the prefix's length."""
    B, T, H, D = q.shape
    Hkv, S = k[0].shape[1], k[0].shape[2]
    scale = D**-0.5 if scale is None else scale
    P = prefix[0][0].shape[2] if prefix else 0
    o, a = torch.zeros(B, T, H, D, dtype=torch.float64), torch.zeros(B, T, H, D, dtype=torch.float64)
    reach, top = torch.zeros(B, T, H, dtype=torch.float64), torch.zeros(B, T, H, dtype=torch.float64)
    for b, row in enumerate(positions(T, starts, counts, S)):
        for t, p in enumerate(row):
            if p < 0:
                continue
            first = 0 if window is None else max(0, P + p - window + 1)
            for h in range(H):
                g = h // (H // Hkv)
                rows = []
                for own, shared in zip((k, v), prefix or (None, None)):
                    x = own[0][b, g, max(0, first - P) : p + 1].double() * own[1][b, g, max(0, first - P) : p + 1, None]
                    if P:
                        y = shared[0][0, g, min(first, P) :].double() * shared[1][0, g, min(first, P) :, None]
                        x = torch.cat((y, x))
                    rows.append(x)
                kr, vr = rows
                top[b, t, h] = max([v[1][b, g, max(0, first - P) : p + 1].nan_to_num().max().item()]
                                   + ([prefix[1][1][0, g, min(first, P) :].nan_to_num().max().item()] if first < P else []))
                qr = q[b, t, h].double()
                prob = torch.softmax(kr @ qr * scale, dim=0)
                o[b, t, h] = prob @ vr
                a[b, t, h] = prob @ vr.abs()
                reach[b, t, h] = (kr.abs() @ qr.abs()).max() * scale
    return o, a, reach, top
