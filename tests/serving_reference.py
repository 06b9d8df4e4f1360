"""Plain 64-bit forms of the serving operators (include/holo_b200.h:
cuda_attention_packed, cuda_kv4_*), for the tests: numpy on the host, from the
definitions.  Values of the 4-bit cache are placed and read one by one, by the
layout's description."""
import numpy as np


def half_at(hd, side, pos, dim):
    """Byte offset in a block, and shift, of the 4-bit code of value `dim` of position `pos` (side 0 keys, 1 values)."""
    b, r, nb = dim // 32, dim % 32, hd // 32
    if side == 0:
        word, nib = pos * 4 * nb + (r // 8) * nb + b, r % 8
        return word * 4 + nib // 2, 4 * (nib % 2)
    g, nib = r // 4, r % 4
    half = ((((g // 2) * 8 + pos // 2) * 2 + g % 2) * 2 + pos % 2) * nb + b
    return 8 * hd + half * 2 + nib // 2, 4 * (nib % 2)


def scale_at(hd, side, pos, dim):
    return (16 + side) * hd + 2 * (pos * (hd // 32) + dim // 32)


def quantise(x):
    """(codes, fp16 scales) of x [..., hd], in the arithmetic that the format defines (fp32, rounded after each operation)."""
    x = np.asarray(x, np.float32).reshape(*np.shape(x)[:-1], -1, 32)
    with np.errstate(all="ignore"):
        first = np.argmax(np.abs(x) == np.abs(x).max(-1, keepdims=True), axis=-1)
        m = np.take_along_axis(x, first[..., None], -1)
        d = (m / np.float32(-8)).astype(np.float16)
        d = np.where(np.isfinite(x).all(-1, keepdims=True), d, np.float16(np.nan))
        w = d.astype(np.float32)
        q = np.where(w == 0, np.float32(0), np.rint(x / w))
        codes = np.clip(np.nan_to_num(q, nan=0.0) + 8, 0, 15).astype(np.int64)
    return codes.reshape(*codes.shape[:-2], -1), d[..., 0]


def values(codes, scales):
    with np.errstate(all="ignore"):
        w = scales.astype(np.float64)[..., None]
        return ((codes.reshape(*scales.shape, 32) - 8) * w).reshape(codes.shape)


def place(pool, layer, page, kvh, at, hd, side, codes, scales):
    """Writes one position's codes [hd] and scales [hd / 32] of a head into pool (numpy uint8, the cache's layout)."""
    blk = pool[layer, page, kvh, at // 16]
    pos = at % 16
    for dim in range(hd):
        byte, shift = half_at(hd, side, pos, dim)
        blk[byte] = (int(blk[byte]) & ~(15 << shift) & 255) | (int(codes[dim]) << shift)
        if dim % 32 == 0:
            o = scale_at(hd, side, pos, dim)
            blk[o:o + 2] = np.frombuffer(np.float16(scales[dim // 32]).tobytes(), np.uint8)


def fetch(pool, layer, page, kvh, at, hd, side):
    """One position's values [hd] of a head, 64-bit."""
    blk, pos = pool[layer, page, kvh, at // 16], at % 16
    dims = np.arange(hd)
    where = [half_at(hd, side, pos, d) for d in dims]
    codes = np.array([int(blk[o]) >> s & 15 for o, s in where])
    scales = np.array([np.frombuffer(blk[scale_at(hd, side, pos, d):][:2].tobytes(), np.float16)[0] for d in dims[::32]])
    return values(codes, scales)


def attend(q, k, v, scale, causal=False):
    """softmax(scale q k^T) v in 64 bits: q [n][hd], k and v [m][hd]; causal: query i sees the keys up to i + m - n.
    No keys: zeros.  Also each row's log of its sum of exps."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    if k.shape[0] == 0:
        return np.zeros((len(q), v.shape[1])), np.full(len(q), -np.inf)
    w = q @ k.T * scale
    if causal:
        w = np.where(np.arange(len(k)) > np.arange(len(q))[:, None] + len(k) - len(q), -np.inf, w)
    m = w.max(1, keepdims=True)
    p = np.exp(w - m)
    return p / p.sum(1, keepdims=True) @ v, (m + np.log(p.sum(1, keepdims=True)))[:, 0]


# Bound on |out - exact|, from the format of the steps.  u is the unit roundoff of the rows' type (the softmax weights are
# rounded to 11 bits or more, but for bfloat16 prompts to 8, and the result once to the type); scores are sums of hd products
# with operands good to 2^-22 of the largest, so they are off by at most hd * 2^-22 * max|q| max|k| * scale, and the weights by
# twice that relatively; exp and the sums of n weights add (n + 8) * 2^-23.
UNIT = {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -9}


def bound(q, k, v, scale, dtype):
    if k.shape[0] == 0:
        return 0.0
    s = k.shape[1] * 2.0 ** -22 * float(np.abs(q).max()) * float(np.abs(k).max()) * scale
    return float(np.abs(v).max()) * (2 * s + (k.shape[0] + 8) * 2.0 ** -23 + 2 * UNIT[dtype])
