"""The paged 8-bit K/V cache in 64 bits, one page, head and query at a time.

A plain restatement of what include/csahca.h says of the ``csahca_kv8_*`` entry
points, in numpy (torch only carries float8 and bfloat16 tensors in and out).
Caches are CPU torch tensors in the layout of ``csahca_amd.kv8_layout``.
"""
from __future__ import annotations

import numpy as np
import torch

GROUP = 16
LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def _e4m3_values() -> np.ndarray:
    """The 256 codes: 1 sign, 4 exponent (bias 7), 3 mantissa bits; 0x7f / 0xff NaN."""
    c = np.arange(256)
    e, m = c >> 3 & 15, c & 7
    mag = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    mag[(c & 127) == 127] = np.nan
    return np.where(c & 128, -mag, mag)


E4M3 = _e4m3_values()
_MIDDLES = (E4M3[:126] + E4M3[1:127]) / 2


def decode(codes: np.ndarray, fmt) -> np.ndarray:
    """uint8 codes to fp64."""
    return E4M3[codes] if fmt == torch.float8_e4m3fn else codes.view(np.int8).astype(np.float64)


def encode(x: np.ndarray, fmt) -> np.ndarray:
    """fp64 values to uint8 codes: clamped, to nearest, ties to even; NaN to NaN or, in int8, to 0."""
    nan = np.isnan(x)
    y = np.clip(np.where(nan, 0.0, x), -LARGEST[fmt], LARGEST[fmt])
    if fmt == torch.int8:
        return np.rint(y).astype(np.int8).view(np.uint8)
    a = np.abs(y)
    code = np.searchsorted(_MIDDLES, a, side="left")
    tie = (code < 126) & (a == _MIDDLES[np.minimum(code, 125)])
    code = code + (tie & (code % 2 == 1))
    code = code | np.where(np.signbit(y), 128, 0)
    return np.where(nan, 127, code).astype(np.uint8)


def scale_for(amax: float, fmt) -> float:
    """The least power of two in 2^-120 .. 2^120 that holds amax."""
    e = -120
    while e < 120 and amax > LARGEST[fmt] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def _codes(t: torch.Tensor) -> np.ndarray:
    return t.view(torch.uint8).numpy()


def _rows(tile: np.ndarray) -> np.ndarray:
    """A (page, head) tile of either cache as [page, D] (a copy)."""
    return tile.copy() if tile.ndim == 2 else tile.transpose(0, 2, 1).reshape(-1, tile.shape[1])


def _tile(rows: np.ndarray, like: np.ndarray) -> np.ndarray:
    return rows if like.ndim == 2 else rows.reshape(like.shape[0], GROUP, -1).transpose(0, 2, 1)


def page_of(table: np.ndarray, b: int, pos: int, page: int, pages: int) -> int:
    j = pos // page
    if pos < 0 or j >= table.shape[1]:
        return -1
    p = int(table[b, j])
    return p if 0 <= p < pages else -1


def write(k, v, cache, table, start, counts=None):
    """A new cache (CPU tensors) with the tokens written."""
    cache = tuple(t.clone() for t in cache)
    table = table.numpy()
    pages, heads, page, _ = cache[0].shape
    fmt = cache[0].dtype
    B, _, N, _ = k.shape
    for x, data, scale in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        codes, scale, x = _codes(data), scale.numpy(), x.double().numpy()
        for b in range(B):
            first = int(start[b])
            count = N if counts is None else min(max(int(counts[b]), 0), N)
            if first < 0:
                continue
            for j in range(first // page, (first + count - 1) // page + 1 if count else 0):
                lo, hi = max(first - j * page, 0), min(first + count - j * page, page)
                p = page_of(table, b, j * page, page, pages)
                if hi <= lo or p < 0:
                    continue
                for h in range(heads):
                    new = x[b, h, j * page + lo - first : j * page + hi - first]
                    fin = np.abs(new[np.isfinite(new)])
                    s = scale_for(fin.max() if fin.size else 0.0, fmt)
                    rows = _rows(codes[p, h])
                    old = float(scale[p, h])
                    if lo > 0:
                        if s > old:
                            rows[:lo] = encode(decode(rows[:lo], fmt) * (old / s), fmt)
                        else:
                            s = old
                    rows[lo:hi] = encode(new * (1.0 / s), fmt)
                    codes[p, h] = _tile(rows, codes[p, h])
                    scale[p, h] = s
    return cache


def token(cache, table, b, h, pos):
    """(k, v) of one position in fp64, or None where it has no page."""
    pages, _, page, _ = cache[0].shape
    p = page_of(table, b, pos, page, pages)
    if p < 0:
        return None
    r = pos % page
    k = decode(_codes(cache[0])[p, h, r], cache[0].dtype) * float(cache[2][p, h])
    v = decode(_codes(cache[1])[p, h, r // GROUP, :, r % GROUP], cache[1].dtype) * float(cache[3][p, h])
    return k, v


def read(cache, table, lengths, max_tokens, start=None):
    """fp64 (k, v) [batch, heads, max_tokens, D]."""
    table = table.numpy()
    B, H, D = table.shape[0], cache[0].shape[1], cache[0].shape[3]
    out = np.zeros((2, B, H, max_tokens, D))
    for b in range(B):
        first = 0 if start is None else int(start[b])
        for n in range(max_tokens):
            pos = first + n
            if not 0 <= pos < int(lengths[b]):
                continue
            for h in range(H):
                kv = token(cache, table, b, h, pos)
                if kv is not None:
                    out[0, b, h, n], out[1, b, h, n] = kv
    return out[0], out[1]


def _softmax_v(q, ks, vs, scale):
    """(out, sum of p |v|, largest scale * sum |q k|) of one query over the given tokens."""
    D = q.shape[0]
    if not ks:
        return np.zeros(D), np.zeros(D), 0.0
    k, v = np.stack(ks), np.stack(vs)
    s = k @ q * scale
    with np.errstate(all="ignore"):
        p = np.exp(s - s.max())
        p = p / p.sum()
    return p @ v, p @ np.abs(v), float(np.max(np.abs(k) @ np.abs(q)) * abs(scale))


def attend(q, cache, table, lengths, scale=None, chunks=None, chunk_size=None):
    """fp64 attention of q [B, Q, heads, D] (or [B, heads, D]) over all tokens,
    or over the listed ``chunks`` [B, kv_heads, k]; with it the same sum over
    |v| and the largest sum |q k| of each row, for error bounds."""
    shape, D = tuple(q.shape), q.shape[-1]
    q = q.double().numpy().reshape(shape[0], -1, shape[-2], D)
    table = table.numpy()
    B, Q, heads, _ = q.shape
    _, H, page, _ = cache[0].shape
    scale = D ** -0.5 if scale is None else scale
    out, mass, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:-1])
    for b in range(B):
        n = min(max(int(lengths[b]), 0), table.shape[1] * page)
        for h in range(H):
            have = {}
            if chunks is None:
                at = list(range(n))
            else:
                at = [int(c) * chunk_size + t for c in chunks[b, h] if 0 <= int(c) <= n // chunk_size
                      for t in range(chunk_size)]
                at = [pos for pos in at if pos < n]
            for pos in set(at):
                have[pos] = token(cache, table, b, h, pos)
            for i in range(Q):
                seen = [have[pos] for pos in at if have[pos] is not None and pos < n - Q + 1 + i]
                for g in range(heads // H):
                    r = h * (heads // H) + g
                    out[b, i, r], mass[b, i, r], size[b, i, r] = _softmax_v(
                        q[b, i, r], [kv[0] for kv in seen], [kv[1] for kv in seen], scale)
    return out.reshape(shape), mass.reshape(shape), size.reshape(shape[:-1])
