"""Plain float64 forms of the FP8 paged serving operators: E4M3 rounding, residual + RMS normalisation + codes, the paged cache and the
attention that reads it.  numpy only; one loop per sequence and page, written from the definitions."""
from __future__ import annotations

import numpy as np

LEAST_EXPONENT = -120           # of a page's scale


def e4m3_values() -> np.ndarray:
    """What the 256 codes stand for: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7f and 0xff are NaN, there are no infinities."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 0x7f) == 0x7f, np.nan, v)
    return np.where(c >= 128, -v, v)


_VALUES = e4m3_values()


def e4m3_decode(codes: np.ndarray) -> np.ndarray:
    return _VALUES[codes.astype(np.uint8)]


def e4m3_round(v: np.ndarray) -> np.ndarray:
    """The nearest E4M3 value, ties to even, magnitudes beyond 448 to 448; NaN stays."""
    v = np.asarray(v, dtype=np.float64)
    a = np.minimum(np.abs(v), 448.0)
    _, e = np.frexp(np.maximum(a, 2.0 ** -6))
    step = np.ldexp(1.0, e - 4)
    out = np.minimum(np.rint(a / step) * step, 448.0)
    return np.where(np.isnan(v), np.nan, np.copysign(out, v))


def page_scale(amax) -> np.ndarray:
    """The least power of two s with amax / s <= 448, not below 2 ** -120."""
    amax = np.asarray(amax, dtype=np.float64)
    m, e = np.frexp(np.maximum(amax, 1e-300))
    e = np.where(amax > 0, e - 9 + (m > 0.875), LEAST_EXPONENT)
    return np.ldexp(1.0, np.maximum(e, LEAST_EXPONENT))


def add_norm(total: np.ndarray, weight: np.ndarray, eps: float, quant_eps: float, pow2: bool):
    """Normalized rows and block scales of rows already summed; [rows, dim] -> (normalized [rows, dim], scales [rows, dim / 128])."""
    t = total.astype(np.float64)
    n = t / np.sqrt((t * t).mean(1, keepdims=True) + eps) * weight.astype(np.float64)
    s = np.maximum(np.abs(n).reshape(len(n), -1, 128).max(2), quant_eps) / 448.0
    if pow2:
        m, e = np.frexp(s)
        s = np.ldexp(1.0, np.where(m == 0.5, e - 1, e))
    return n, s


def rotary_rows(positions: int, dim: int, rope_dim: int, base: float = 10000.0):
    half = rope_dim // 2
    angle = np.arange(positions)[:, None] * base ** (-np.arange(half) / max(half, 1))
    rest = np.zeros((positions, dim - rope_dim))
    return (np.concatenate([np.cos(angle), np.cos(angle), rest + 1], 1).astype(np.float32),
            np.concatenate([-np.sin(angle), np.sin(angle), rest], 1).astype(np.float32))


def turn(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, rope_dim: int) -> np.ndarray:
    """x [tokens, heads, dim], cos / sin [tokens, dim]."""
    half = rope_dim // 2
    x = x.astype(np.float64)
    swapped = np.concatenate([x[..., half:rope_dim], x[..., :half], x[..., rope_dim:]], -1)
    return x * cos[:, None].astype(np.float64) + swapped * sin[:, None].astype(np.float64)


def append(keys, values, key_codes, value_codes, key_scales, value_scales, table, lengths, cu_steps):
    """keys (turned already), values [tokens, kv_heads, dim] float64; codes uint8, key [pool, kv_heads, page, dim], value [pool, kv_heads, dim, page].  Returns
    new copies of the four cache arrays, the codes as values (float64)."""
    pool, kv_heads, page, dim = key_codes.shape
    out = [e4m3_decode(key_codes), e4m3_decode(value_codes).transpose(0, 1, 3, 2).copy(), key_scales.astype(np.float64), value_scales.astype(np.float64)]
    for s, length in enumerate(lengths):
        n = cu_steps[s + 1] - cu_steps[s]
        places = [(i, length - n + i) for i in range(n) if length - n + i >= 0]
        for p in sorted({at // page for _, at in places}):
            here = [(i, at) for i, at in places if at // page == p]
            if p >= table.shape[1] or not 0 <= table[s, p] < pool:
                continue
            which, held = table[s, p], here[0][1] - p * page
            for rows, codes, scales in ((keys, out[0], out[2]), (values, out[1], out[3])):
                new = np.stack([rows[cu_steps[s] + i] for i, _ in here], 1)                  # [kv_heads, tokens, dim]
                finite = np.where(np.isfinite(new), np.abs(new), 0.0).max((1, 2))
                scale = page_scale(finite)
                if held:
                    scale = np.maximum(scale, scales[which])
                    codes[which, :, :held] = e4m3_round(codes[which, :, :held] * (scales[which] / scale)[:, None, None])
                codes[which, :, held:held + len(here)] = e4m3_round(np.where(np.isfinite(new), new, np.nan) / scale[:, None, None])
                scales[which] = scale
    return out[0], out[1].transpose(0, 1, 3, 2), out[2], out[3]


def attention(q, key_codes, value_codes, key_scales, value_scales, table, lengths, cu_steps, scale: float):
    """q [tokens, heads, dim].  Returns (outputs, bound): outputs float64 [tokens, heads, dim], zeros where no key is seen, and per output what its error is
    measured in: a dict of float64 arrays, `spread` the weighted mean of |v|, `score` the largest scale * sum |q k| of its keys, `keys` how
    many there are, `top` the largest |v| over the sum of weights."""
    pool, kv_heads, page, dim = key_codes.shape
    tokens, heads, _ = q.shape
    out = np.zeros((tokens, heads, dim))
    note = dict(spread=np.zeros((tokens, heads, dim)), score=np.zeros((tokens, heads, 1)), keys=np.zeros((tokens, heads, 1)), top=np.zeros((tokens, heads, 1)))
    for s, length in enumerate(lengths):
        n = cu_steps[s + 1] - cu_steps[s]
        held = min(length, table.shape[1] * page)
        place = [(p, table[s, p // page]) for p in range(max(held, 0))]
        place = np.array([(p, w) for p, w in place if 0 <= w < pool], dtype=np.int64).reshape(-1, 2)
        at, which = place[:, 0], place[:, 1]
        k = e4m3_decode(key_codes[which, :, at % page]) * key_scales[which][:, :, None]      # [keys, kv_heads, dim]
        v = e4m3_decode(value_codes[which, :, :, at % page]) * value_scales[which][:, :, None]
        for i in range(n):
            sees = at <= length - n + i
            if not sees.any():
                continue
            for h in range(heads):
                kv = h // (heads // kv_heads)
                row = q[cu_steps[s] + i, h].astype(np.float64)
                score = k[sees, kv] @ row * scale
                w = np.exp(score - score.max()) if np.isfinite(score).all() else np.full(score.shape, np.nan)
                t = cu_steps[s] + i, h
                with np.errstate(invalid="ignore"):
                    out[t] = w @ v[sees, kv] / w.sum()
                    note["spread"][t] = w @ np.abs(v[sees, kv]) / w.sum()
                    note["score"][t] = (np.abs(k[sees, kv]) @ np.abs(row)).max() * abs(scale)
                    note["keys"][t] = sees.sum()
                    note["top"][t] = np.nanmax(np.abs(v[sees, kv]), initial=0.0) / w.sum()
    return out, note
