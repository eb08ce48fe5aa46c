"""Oracle of the append-with-rotation operators: the rotation in numpy, in float32 operation by operation and in 64 bits."""

from __future__ import annotations

import numpy as np

import rpa_testlib as tl
from rpa_testlib import BF16, F16, F32, FP8, INT8, orc


def table(rows, rope, base=10000.0):
    """cos | sin of the angles, from 64 bits."""
    angle = np.arange(rows)[:, None] * base ** (-np.arange(0, rope, 2) / rope)
    return np.concatenate([np.cos(angle), np.sin(angle)], axis=1).astype(np.float32)


def token_positions(ctx, qsl, n_live, T):
    """Cache position of every token, -1 where it belongs to no sequence."""
    pos = np.full(T, -10 ** 9, np.int64)
    for i in range(n_live):
        for r in range(qsl[i + 1] - qsl[i]):
            if qsl[i] + r < T:
                pos[qsl[i] + r] = ctx[i] - (qsl[i + 1] - qsl[i]) + r
    return pos


def rotate(x, rows, rope, neox, dtype=np.float32):
    """x [T, heads, D] turned by table rows [T, rope], each product and sum rounded to ``dtype``."""
    x, rows = x.astype(dtype), rows.astype(dtype)
    h = rope // 2
    c, s = rows[:, None, :h], rows[:, None, h:]
    y = x.copy()
    first, second = (slice(0, h), slice(h, rope)) if neox else (slice(0, rope, 2), slice(1, rope, 2))
    a, b = x[..., first], x[..., second]
    y[..., first] = (a * c).astype(dtype) - (b * s).astype(dtype)
    y[..., second] = (b * c).astype(dtype) + (a * s).astype(dtype)
    return y


def encode(x, tag):
    """float32 values -> storage bits, rounded to nearest even (fp8: the bare cast)."""
    if tag == BF16:
        return orc.f32_to_bf16_bits(x)
    if tag == F16:
        return x.astype(np.float16)
    if tag == FP8:
        return orc.cast_e4m3fn_ref(x)
    return x.astype(np.float32)


def decode(raw, tag):
    if tag == BF16:
        return orc.bf16_bits_to_f32(raw)
    if tag in (FP8, INT8):
        return orc.decode_codes(raw, tag)
    return raw.astype(np.float32)


def batch(rng, q_lens, past, page_size, pad_rows=0, pad_tokens=0, spare=3, max_pages=None):
    """(ctx, block tables, qsl, num_seqs, T, P) of sequences with ``past`` tokens ahead of their new ones."""
    q_lens, past = np.asarray(q_lens, np.int32), np.asarray(past, np.int32)
    n = len(q_lens)
    S = n + pad_rows
    ctx = np.zeros(S, np.int32)
    ctx[:n] = q_lens + past
    need = [-(-int(c) // page_size) for c in ctx[:n]]
    M = max_pages or max(max(need), 1)
    P = sum(need) + spare
    perm = rng.permutation(np.arange(P))
    bt = np.zeros((S, M), np.int32)
    k = 0
    for i, m in enumerate(need):
        bt[i, :m] = perm[k:k + m]
        k += m
    qsl = np.zeros(S + 1, np.int32)
    qsl[1:n + 1] = np.cumsum(q_lens)
    qsl[n + 1:] = qsl[n]
    return ctx, bt, qsl, np.array([n], np.int32), int(qsl[n]) + pad_tokens, P


def append_scaled(key, value, codes, scales, ctx, bt, qsl, n_live, kv):
    """The scaled 8-bit write in float32: of each page a sequence writes to, the scale grows to ``amax * (1 / qmax)`` where
    that is more (1 where both are 0; a page that starts with new tokens has no old scale), what the page holds is coded
    again if it grew, the new tokens are coded.  Returns (codes, scales)."""
    codes, scales, pg = codes.copy(), scales.copy(), codes.shape[1]
    unit = np.float32(1.0) / np.float32(orc.QMAX[kv])
    for i in range(n_live):
        q0, q1, end = int(qsl[i]), int(qsl[i + 1]), int(ctx[i])
        pos = max(end - (q1 - q0), 0)
        while pos < end:
            j, first = divmod(pos, pg)
            n, page, t0 = min(end, (j + 1) * pg) - pos, int(bt[i, j]), q0 + pos - (end - (q1 - q0))
            for c in range(2 * key.shape[1]):
                x = (value if c & 1 else key)[t0:t0 + n, c >> 1]
                old = scales[page, c] if first else np.float32(0.0)
                new = max(old, np.float32(np.abs(x).max()) * unit) or np.float32(1.0)
                if first and new > old:
                    codes[page, :first, c] = orc.quantise_codes((orc.decode_codes(codes[page, :first, c], kv) * old) / new, kv)
                codes[page, first:first + n, c] = orc.quantise_codes(x / new, kv)
                scales[page, c] = new
            pos += n
    return codes, scales


def dev(a, gpu):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).to(gpu)


def raw_of(t, tag):
    """Storage bits of a device tensor, as the encoders above return them."""
    import torch

    t = t.contiguous().cpu()
    if tag == BF16:
        return t.view(torch.int16).numpy().view(np.uint16)
    if tag == FP8:
        return t.view(torch.uint8).numpy()
    return t.numpy()


__all__ = ["tl", "orc", "BF16", "F16", "F32", "FP8", "INT8", "table", "token_positions", "rotate", "encode", "decode", "batch", "append_scaled", "dev", "raw_of"]
