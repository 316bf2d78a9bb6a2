"""Plain restatement of the 4-bit pools for the tests: the quantiser's rule in fp32 as it is
defined, what a pool's bytes stand for, and attention over them in float64."""
from __future__ import annotations

import numpy as np

F = np.float32


def quantise(x: np.ndarray):
    """Rows x [..., D] fp32 -> (codes uint8 [..., D], scale fp32 [...], zero point [...])."""
    x = np.where(np.isnan(x), F(0), x).astype(F)
    x = np.clip(x, F(-1e36), F(1e36))
    lo = np.minimum(x.min(-1), F(0))
    hi = np.maximum(x.max(-1), F(0))
    r = ((hi - lo) / F(15)).astype(F)
    s = ((r.view(np.uint32) + np.uint32(0x7FFFF)) & np.uint32(0xFFF80000)).view(F)
    s = np.maximum(s, F(2.0 ** -100))
    z = np.rint((-lo / s).astype(F))
    n = np.clip(np.rint((x / s[..., None]).astype(F)) + z[..., None], 0, 15).astype(np.uint8)
    return n, s, z.astype(np.int64)


def values(n, s, z):
    return (n.astype(np.float64) - z[..., None]) * s[..., None].astype(np.float64)


def pack_k(n: np.ndarray) -> np.ndarray:
    """Codes [..., D] of a token -> its K row's bytes [..., D/2]."""
    return n[..., 0::2] | (n[..., 1::2] << 4)


def pack_v(n: np.ndarray) -> np.ndarray:
    """Codes [..., D] of a token -> its column of the V tile [..., D/2]."""
    h = n.shape[-1] // 2
    return n[..., :h] | (n[..., h:] << 4)


def pool_values(kv, layer: int = 0, spans: bool = False):
    """What every slot of a 4-bit KVCache stands for: K, V float64 [blocks, Hkv, bs, D], and with
    spans=True the ranges 15 s of its keys and values [blocks, Hkv, bs]."""
    nb, h, bs, d = kv.num_blocks, kv.num_kv_heads, kv.block_size, kv.head_dim
    k = kv.k_pool(layer).cpu().numpy().reshape(nb, h, bs, d // 2)
    v = kv.v_pool(layer).cpu().numpy().reshape(nb, h, d // 2, bs).swapaxes(2, 3)
    kn = np.stack([k & 15, k >> 4], -1).reshape(nb, h, bs, d)
    vn = np.concatenate([v & 15, v >> 4], -1)
    (ks, kz), (vs, vz) = [[t.cpu().numpy() for t in pair] for pair in kv.scales(layer)]
    both = values(kn, ks, kz), values(vn, vs, vz)
    return both + (15.0 * ks, 15.0 * vs) if spans else both


def attention(q, K, V, ctx, rows, tables, scale, out, span):
    """q [B, R, Hq, D] float64; K, V from pool_values; rows past a sequence's count keep `out`.
    Returns (out float64, sum over visible keys of p |v| of each element: what an error of the
    probabilities is relative to). `span`: 15 s of every slot's values [blocks, Hkv, bs]; its sum
    over visible keys, weighted by p, is returned third: what codes and zero points, summed apart,
    are rounded relative to. Fourth, what the probabilities' smallest step is worth at most:
    n keys times the largest range among the sequence's, kept below 2^13 times the visible ones'."""
    B, R, Hq, D = q.shape
    nb, H, bs, _ = K.shape
    out, mag, reach, least = out.astype(np.float64).copy(), *(np.zeros(q.shape) for _ in range(3))
    for b in range(B):
        c = min(max(int(ctx[b]), 0), tables.shape[1] * bs)
        n = int(rows[b])
        if n > R or n <= 0 or n > c:
            continue
        t = np.arange(c)
        blk = tables[b, t // bs]
        ok = (blk >= 0) & (blk < nb)
        safe = np.where(ok, blk, 0)
        for h in range(H):
            k, v, w = K[safe, h, t % bs], V[safe, h, t % bs], span[safe, h, t % bs]
            for g in range(Hq // H):
                for j in range(n):
                    see = ok & (t <= c - n + j)
                    i = h * (Hq // H) + g
                    if not see.any():
                        out[b, j, i] = 0
                        continue
                    s = (k[see] @ q[b, j, i]) * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[b, j, i] = p @ v[see]
                    mag[b, j, i] = p @ np.abs(v[see])
                    reach[b, j, i] = p @ w[see]
                    least[b, j, i] = see.sum() * min(w[ok].max(), 2.0 ** 13 * w[see].max())
    return out, mag, reach, least


def attention_tolerance(q, K, k_span, scale, ref, mag, reach, least, q_dtype, out_dtype):
    """Largest deviations a right kernel may have, by arithmetic (half steps: bf16 2^-8 relative,
    fp16 2^-11, fp32 2^-24):
      - scores: dots of D products in fp32, the queries to 21 bits at least: an error of
        2^-20 sum |q| |k| scale, twice in a probability (its own score, the maximum's), and the
        exponent's argument rounded to fp32 (2^-22 of the largest score);
      - probabilities to fp16 unless queries or outputs are fp32 (then to 21 bits), their sums
        in fp32 (sqrt of 2^15 terms, 2^-16);
      - unless queries or outputs are fp32, codes and zero points are summed apart, in fp32, 32
        products to a step aligned to the largest and cut at 2^-24 of it (33 * 2^-24 < 2^-18): 2^-18
        of the sum of p 15 s_v for each of the two sums, and for the scores of 15 s_k sum |q|;
      - p s_v in f16 in units of B 2^-10, B a power of two less than twice the largest s_v: its last
        part ends at 2^-24, so half a step of 2^-35 B, 2^-34 of the largest range, for each key;
      - the output's own rounding."""
    fine = "f32" in (q_dtype, out_dtype)
    qf = np.where(np.isfinite(q), q, 0)
    one = np.abs(qf).sum(-1).max() * abs(scale)
    peak = np.sqrt((K ** 2).sum(-1).max()) * np.sqrt((qf ** 2).sum(-1).max()) * abs(scale)
    score = 2.0 ** -20 * min(np.abs(K).max() * one, 40 * peak) + (0 if fine else 2 * 2.0 ** -18 * k_span.max() * one)
    rel = 2 * score + 2.0 ** -22 * peak + (2.0 ** -16 if fine else 2.0 ** -11 + 2.0 ** -16)
    half = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[out_dtype]
    tiny = 2.0 ** -25 if out_dtype == "f16" else 1e-38
    return rel * mag + (0 if fine else 2 * 2.0 ** -18 * reach) + 2.0 ** -34 * least + half * np.abs(ref) + tiny
