"""Plain restatement of a paged KV cache held in 8 bits, in numpy.

Codes are e4m3 bytes ``[P, 2, page, Hkv, D]``; each block -- the tokens of one page,
K or V, one head -- has a power-of-two scale as an e8m0 byte ``[P, 2, Hkv]``: a code
stands for ``code * 2**(byte - 127)``.  A block's exponent is the least ``E >= -100``
with ``amax <= 448 * 2**E``.  No reference counterpart (its cache holds the model's
type); the definition is this package's own.
"""

from __future__ import annotations

import math

import numpy as np

LEAST_EXP = -100
# the largest e4m3 value times a power of two that the 16-bit type holds
LARGEST = {"float16": 61440.0, "bfloat16": 1.875 * 2.0 ** 127}


def _code_values() -> np.ndarray:
    out = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.nan if (c & 127) == 127 else (8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9
        out[c] = -v if c & 128 else v
    return out


CODE_VALUES = _code_values()
_POSITIVE = CODE_VALUES[:127]                            # 0 .. 448, ascending
_MIDDLES = (_POSITIVE[1:] + _POSITIVE[:-1]) / 2


def encode(x: np.ndarray) -> np.ndarray:
    """The code nearest to each value (ties to the even code), |x| <= 448; NaN and
    infinities are NaN."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    lo = np.searchsorted(_MIDDLES, a, side="left")       # a tie goes to the lower code ...
    tie = (lo < 126) & (a == _MIDDLES[np.minimum(lo, 125)])
    lo = lo + (tie & (lo % 2 == 1))                      # ... or to the upper one where that is even
    out = lo | np.where(np.signbit(x), 128, 0)
    return np.where(np.isfinite(x), out, 127).astype(np.uint8)


def exponent(amax: float) -> int:
    e = LEAST_EXP
    while amax > math.ldexp(448.0, e):
        e += 1
    return e


def values(codes: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """float64 values of a layer."""
    return CODE_VALUES[codes] * np.exp2(scale.astype(np.float64) - 127.0)[:, :, None, :, None]


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray) -> np.ndarray:
    """HF's rotate_half form on float32 heads ``[n, H, D]`` with tables ``[n, D]``."""
    h = x.shape[-1] // 2
    turned = np.concatenate([-x[..., h:], x[..., :h]], axis=-1)
    return x * cos[:, None] + turned * sin[:, None]


def append(codes: np.ndarray, scale: np.ndarray, pages, slots, k: np.ndarray, v: np.ndarray, dtype: str) -> int:
    """One call's entries, ``k`` / ``v`` ``[n, Hkv, D]`` float32 (k rotated), written in place;
    returns how many were skipped."""
    num_pages, _, page_size, heads, _ = codes.shape
    ok = [i for i in range(len(pages)) if 0 <= pages[i] < num_pages and 0 <= slots[i] < page_size]
    of_page = {}
    for i in ok:
        of_page.setdefault(int(pages[i]), []).append(i)
    for p, mine in of_page.items():
        first = min(int(slots[i]) for i in mine)
        for sel, rows in ((0, k), (1, v)):
            for h in range(heads):
                x = np.abs(rows[mine, h])
                x = np.minimum(x[np.isfinite(x)], LARGEST[dtype])
                e = exponent(float(x.max()) if x.size else 0.0)
                if first > 0:
                    old = int(scale[p, sel, h]) - 127
                    e = max(e, old)
                    if e > old:
                        before = CODE_VALUES[codes[p, sel, :first, h]] * 2.0 ** (old - e)
                        codes[p, sel, :first, h] = encode(before)
                scale[p, sel, h] = e + 127
                for i in mine:                           # in order: the last of a slot is kept
                    r = rows[i, h].astype(np.float64)
                    r = np.where(np.isfinite(r), np.clip(r, -LARGEST[dtype], LARGEST[dtype]), r)
                    codes[p, sel, int(slots[i]), h] = encode(r * 2.0 ** -e)
    return len(pages) - len(ok)
