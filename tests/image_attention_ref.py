"""64-bit restatement of the image-token attention operators' formulas, and the roundings their tolerances count.

The tests' oracle (NumPy, loops over heads and blocks): qkv_norm_rope, block_select, block_attention."""
import numpy as np

BLOCK_Q = 128
BF16 = np.dtype([("bfloat16", "<u2")])
KINDS = {"f32": np.dtype(np.float32), "f16": np.dtype(np.float16), "bf16": BF16}
#: Half a step of rounding to nearest, relative to the value; and the largest error below the smallest normal value.
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def narrow(a, kind):
    """Rounds a float array to a storage type (to nearest, ties to even)."""
    a = np.asarray(a, np.float32)
    if kind != "bf16":
        return a.astype(KINDS[kind])
    u = a.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    r = np.where(np.isnan(a), np.uint16(0x7FC0), r)
    return np.ascontiguousarray(r).view(BF16)


def wide(a):
    """A storage array's values in 64 bits."""
    a = np.asarray(a)
    if a.dtype == BF16:
        return (a.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def norm_rope(x, gamma, eps, norm, positions, axis_dims, theta, halves):
    """x [n, tokens, heads, dim] in 64 bits; positions [n or 1, tokens, 3] or None. Returns (y, size): size is the
    length of the pair that each channel turns with, by which a rotation's error is measured."""
    y = x.copy()
    dim = x.shape[-1]
    if norm:
        y = y / np.sqrt(np.mean(y * y, -1, keepdims=True) + eps) * (1.0 if gamma is None else gamma.astype(np.float64))
    size = np.abs(y)
    first = 0
    for a, d in enumerate(axis_dims if positions is not None else ()):
        for i in range(d // 2):
            angle = positions[..., a].astype(np.float64)[:, :, None] * float(theta) ** (-2.0 * i / d)
            c, s = np.cos(angle), np.sin(angle)
            e0, e1 = (first + i, first + d // 2 + i) if halves else (first + 2 * i, first + 2 * i + 1)
            a0, a1 = y[..., e0].copy(), y[..., e1].copy()
            y[..., e0], y[..., e1] = a0 * c - a1 * s, a1 * c + a0 * s
            size[..., e0] = size[..., e1] = np.hypot(a0, a1)
        first += d
    return y, size


def select(q, k, topk, block_k, mask=None):
    """q [n, nq, heads, dim], k [n, nk, kv_heads, dim] in 64 bits -> index [n, heads, q blocks, topk]."""
    n, nq, heads, _ = q.shape
    nk, group = k.shape[1], heads // k.shape[2]
    q_blocks, k_blocks = -(-nq // BLOCK_Q), -(-nk // block_k)
    index = np.full((n, heads, q_blocks, topk), -1, np.int32)
    for b in range(n):
        keep = np.ones(nk, bool) if mask is None else mask[b] != 0
        for h in range(heads):
            means = []
            for j in range(k_blocks):
                rows = k[b, j * block_k:(j + 1) * block_k, h // group][keep[j * block_k:(j + 1) * block_k]]
                means.append(rows.sum(0) / len(rows) if len(rows) else None)
            live = [j for j in range(k_blocks) if means[j] is not None]
            for i in range(q_blocks):
                mean = q[b, i * BLOCK_Q:(i + 1) * BLOCK_Q, h].mean(0)
                score = {j: float(mean @ means[j]) for j in live}
                best = sorted(sorted(live, key=lambda j: (not np.isnan(score[j]), -score[j], j))[:topk])
                index[b, h, i, :len(best)] = best
    return index


def attention(q, k, v, index, block_k, mask, scale, kind):
    """(out, tolerance) of block_attention in 64 bits, for inputs that the storage type `kind` holds.

    The tolerance counts, in units of the row's Σ p |v| / Σ p:
      * the error of a logit, e = 2^-19 · scale · max_j Σ |q_i k_ji|: an f32 dot product in which at most 16 partial
        sums are rounded or truncated (2^-23 each, 2^-19 in all), which covers the two-part split of f32 operands too
        (2^-21); it moves every weight by a factor within e, and the quotient by 2 e;
      * the exponential, its argument's rounding (2^-23 of at most 2^7 before the weight underflows) and the sums:
        2^-16 + 2^-24 · blocks;
      * for 16-bit types the weights' rounding (half a step) before the product with v, and at the end the result's;
      * f16 weights below 2^-14 have an absolute error of 2^-25 each, counted against the row's sum of weights."""
    n, nq, heads, dim = q.shape
    nk, group = k.shape[1], heads // k.shape[2]
    k_blocks = -(-nk // block_k)
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(n):
        keep = np.ones(nk, bool) if mask is None else mask[b] != 0
        for h in range(heads):
            for i in range(-(-nq // BLOCK_Q)):
                keys = [j for blk in index[b, h, i] if 0 <= blk < k_blocks
                        for j in range(blk * block_k, min(nk, (blk + 1) * block_k)) if keep[j]]
                if not keys:
                    continue
                rows = slice(i * BLOCK_Q, (i + 1) * BLOCK_Q)
                qh, kh, vh = q[b, rows, h], k[b, keys, h // group], v[b, keys, h // group]
                logit = qh @ kh.T * scale
                p = np.exp(logit - logit.max(1, keepdims=True))
                total = p.sum(1, keepdims=True)
                o = p @ vh / total
                spread = p @ np.abs(vh) / total
                e = 2.0 ** -19 * abs(scale) * (np.abs(qh) @ np.abs(kh).T).max(1, keepdims=True)
                weights = 0.0 if kind == "f32" else HALF_STEP[kind]
                t = (2 * e + 2.0 ** -16 + 2.0 ** -24 * index.shape[-1] + weights) * spread
                if kind == "f16":
                    t += 2.0 ** -25 * np.abs(vh).sum(0)[None] / total
                out[b, rows, h], tol[b, rows, h] = o, t + HALF_STEP[kind] * (np.abs(o) + t) + TINY[kind]
    return out, tol
