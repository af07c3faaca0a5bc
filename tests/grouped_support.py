"""Products grouped by expert by their definitions, in 64 bits (include/skl-gfx950.h states the rules): what the GPU tests of these operators
compare with. Nothing here shares code with the library."""
import numpy as np

import mx_support as mx

U = mx.U  # half a unit in the last place of fp32, relative


def bits(x, kind):
    """The 16-bit (f32: 32-bit) patterns of the nearest values of `kind`."""
    x = np.asarray(x, np.float32)
    if kind == "f32":
        return x.copy()
    return mx.to_bf16(x) if kind == "bf16" else x.astype(np.float16).view(np.uint16)


def values(b, kind):
    if kind == "f32":
        return np.asarray(b, np.float64)
    return mx.of_bf16(b).astype(np.float64) if kind == "bf16" else np.asarray(b, np.uint16).view(np.float16).astype(np.float64)


def group_rows(ids, per_row, groups):
    """(offsets, order, rows, place); order and rows as long as what belongs to a group."""
    ids = np.asarray(ids, np.int64)
    order = np.concatenate([np.flatnonzero(ids == g) for g in range(groups)]).astype(np.int64) if len(ids) else np.zeros(0, np.int64)
    offsets = np.concatenate(([0], np.cumsum([np.count_nonzero(ids == g) for g in range(groups)])))
    place = np.full(len(ids), -1, np.int64)
    place[order] = np.arange(len(order))
    return offsets, order, order // per_row, place


def cut(offsets, total, groups):
    """(first, end) of every group's rows, cut off at 0 and total."""
    if offsets is None:
        return [(0, total)]
    o = np.clip(np.asarray(offsets, np.int64), 0, total)
    return [(int(o[e]), int(max(o[e], o[e + 1]))) for e in range(groups)]


def gathered(a, index, count):
    """Rows 0 .. count - 1 of a through an index: zeros where it points outside."""
    if index is None:
        return a[:count]
    index = np.asarray(index, np.int64)
    out = np.zeros((count, a.shape[1]))
    good = (index >= 0) & (index < len(a))
    out[good] = a[index[good]]
    return out


def gamma(k):
    """A fp32 sum of k exact products in any order, scaled and added to, is within this times the sum of magnitudes: the bound of the reference's
    fp32-accumulation tests (test/gemm/gemm_f32rcprc_f32rcprc_f32rcprc.c)."""
    return 2.0 * np.expm1((k + 2) * np.log1p(U))


def rounded(value, bound, kind):
    """The bound behind a rounding to `kind`: half a step - relative to the value 2^-8 for bf16, 2^-11 for f16 - of what is rounded, which lies within `bound` of value,
    or half the smallest number."""
    if kind == "f32":
        return bound
    half, least = (2.0 ** -8, 2.0 ** -134) if kind == "bf16" else (2.0 ** -11, 2.0 ** -25)
    return bound + half * (np.abs(value) + bound) + least


def product(a, b, c, alpha, beta, groups, index=None):
    """(result, bound) of alpha a[rows] b[e] + beta c on the rows (first, end) of `groups`, and which rows those are. b: one (k, n) matrix per group."""
    m, n = c.shape
    rows = gathered(a, index, m)
    want, bound, inside = c.copy(), np.zeros((m, n)), np.zeros(m, bool)
    for (first, end), w in zip(groups, b):
        if end > first:
            x = rows[first:end]
            want[first:end] = alpha * (x @ w) + (beta * c[first:end] if beta else 0.0)
            bound[first:end] = gamma(w.shape[0]) * (abs(alpha) * (np.abs(x) @ np.abs(w)) + (abs(beta) * np.abs(c[first:end]) if beta else 0.0))
            inside[first:end] = True
    return want, bound, inside


def over(a, b, c, alpha, beta, groups, index_a=None, index_b=None, total=None):
    """(result, bound) of alpha a[rows]^T b[rows] + beta c[e] for every group."""
    x, y = gathered(a, index_a, total), gathered(b, index_b, total)
    want, bound = np.empty(c.shape), np.empty(c.shape)
    for e, (first, end) in enumerate(groups):
        u, v = x[first:end], y[first:end]
        want[e] = alpha * (u.T @ v) + (beta * c[e] if beta else 0.0)
        bound[e] = gamma(end - first) * (abs(alpha) * (np.abs(u).T @ np.abs(v)) + (abs(beta) * np.abs(c[e]) if beta else 0.0))
    return want, bound


def u4_weights(q, scales, zeros, group_k):
    """The (k, n) matrix of codes q (n, k), scales (n, groups) in 64 bits and zeros likewise or None."""
    at = np.arange(q.shape[1]) // group_k
    z = 8.0 if zeros is None else zeros[:, at].astype(np.float64)
    return ((q.astype(np.float64) - z) * scales[:, at]).T


def u4_store(q, ld, fill=0xA5):
    """Packed codes of (n, k), rows ld values apart, `fill` where nothing of them lies."""
    n, k = q.shape
    out = np.full((n - 1) * (ld // 2) + (k + 1) // 2, fill, np.uint8)
    padded = np.zeros((n, k + k % 2), np.uint8)
    padded[:, :k] = q
    if k % 2:
        padded[:, k] = fill & 15
    for j in range(n):
        out[j * (ld // 2):j * (ld // 2) + (k + 1) // 2] = padded[j, 0::2] | (padded[j, 1::2] << 4)
    return out
