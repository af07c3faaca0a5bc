"""MXFP4 and the mixture-of-experts layer by their definitions, in 64 bits (include/skl-gfx950.h states the rules): what the GPU tests of
these operators compare with. Nothing here shares code with the library."""
import numpy as np

import ofp4_support

MAGNITUDES = ofp4_support.E2M1_VALUES[:8]
U = 2.0 ** -24  # half a unit in the last place of fp32, relative


def quantise(x):
    """(codes, scale bytes) of the rows of x, codes as one number per value."""
    x = np.asarray(x, np.float64)
    m, k = x.shape
    blocks = -(-k // 32)
    padded = np.zeros((m, blocks * 32))
    padded[:, :k] = x
    padded = padded.reshape(m, blocks, 32)
    finite = np.isfinite(padded).all(axis=2)
    largest = np.abs(np.where(finite[:, :, None], padded, 0.0)).max(axis=2)
    exponent = np.frexp(largest)[1] - 1  # floor(log2), any number for 0
    s = np.where(largest > 0, np.maximum(exponent - 2, -126), -126)
    with np.errstate(invalid="ignore"):
        v = np.ldexp(np.where(finite[:, :, None], padded, 0.0), -s[:, :, None])
    a = np.minimum(np.abs(v), 6.0)
    distance = np.abs(a[..., None] - MAGNITUDES)
    nearest = distance.min(axis=-1, keepdims=True)
    near = distance == nearest                               # one code, or the two beside a midpoint
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(axis=-1), even.argmax(axis=-1), near.argmax(axis=-1)).astype(np.uint8)
    code |= np.signbit(v).astype(np.uint8) << 3
    code = np.where(finite[:, :, None], code, 0).astype(np.uint8).reshape(m, -1)[:, :k]
    return code, np.where(finite, s + 127, 255).astype(np.uint8)


def values(code, scales, k=None):
    """What codes (one number per value) and their scale bytes stand for."""
    k = code.shape[1] if k is None else k
    v = ofp4_support.E2M1_VALUES[code[:, :k]]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return v * s.repeat(32, axis=1)[:, :k]


def store(code, scales, ld, lds, fill=0xA5):
    """The flat arrays of an MXFP4 matrix, rows ld values and lds bytes apart, `fill` where nothing of it lies."""
    m, k = code.shape
    out = np.full((m - 1) * (ld // 2) + (k + 1) // 2, fill, np.uint8)
    sc = np.full((m - 1) * lds + scales.shape[1], fill, np.uint8)
    padded = np.zeros((m, k + k % 2), np.uint8)
    padded[:, :k] = code
    if k % 2:
        padded[:, k] = fill & 15  # the half byte behind an odd row is not part of the matrix
    for i in range(m):
        out[i * (ld // 2):i * (ld // 2) + (k + 1) // 2] = padded[i, 0::2] | (padded[i, 1::2] << 4)
        sc[i * lds:i * lds + scales.shape[1]] = scales[i]
    return out, sc


def loaded(flat, sc, m, k, ld, lds):
    """The codes and scale bytes in the flat arrays."""
    code = np.zeros((m, k), np.uint8)
    scales = np.zeros((m, -(-k // 32)), np.uint8)
    for i in range(m):
        row = flat[i * (ld // 2):i * (ld // 2) + (k + 1) // 2]
        code[i] = np.stack((row & 15, row >> 4), axis=1).reshape(-1)[:k]
        scales[i] = sc[i * lds:i * lds + scales.shape[1]]
    return code, scales


def to_bf16(x):
    """The nearest bf16 values' bits of fp32 numbers (no NaN among them)."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def of_bf16(bits):
    return (np.asarray(bits, np.uint32) << 16).view(np.float32)


def product_bound(a, b, alpha, beta, c):
    """(alpha a b^T + beta c in 64 bits, elementwise bound): a fp32 sum of K exact products in any order, scaled and added to; the bound of the
    reference's fp32-accumulation tests (test/gemm/gemm_f32rcprc_f32rcprc_f32rcprc.c) without anything on top."""
    gamma = 2.0 * np.expm1((a.shape[1] + 2) * np.log1p(U))
    return alpha * (a @ b.T) + beta * c, gamma * (abs(alpha) * (np.abs(a) @ np.abs(b).T) + abs(beta) * np.abs(c))


def activation(v, act):
    from scipy.special import erf
    if act == 0:
        return v
    if act == 1:
        return np.maximum(v, 0.0)
    return v / (1.0 + np.exp(-v)) if act == 2 else 0.5 * v * (1.0 + erf(v / np.sqrt(2.0)))


def moe(x, router, gate, up, down, top, act, normalise, beta, residual, chosen):
    """(y, weights, bound of y, bound of the weights relative to them) for x (t, h), router (e, h), gate and up (e, i, h), down (e, h, i) in 64
    bits. `chosen`, the experts that the library chose (t, top), are checked first: in descending order of their logits and none of the
    others above them, each to within what fp32 sums may be off; logits further apart than that leave one choice.

    Bounds, with sums of n fp32 products off by at most (n + 2) u times the sum of magnitudes, u = 2^-24:
      a logit                 dl = (h + 2) u |x| |r|
      a weight                relative e^(2 dl) - 1 and (e + 16) u for the exponentials, their sum and the quotient (expf: 2 ulp)
      gate, up                dg, du as dl
      f = act(gate)           |f'| <= 1.13 (GELU), so 1.13 dg, and its own rounding: 4 ulp, GELU 40 ulp of |f| and 2^-22 absolute (its values far
                              below zero, see skl_device.hpp)
      h = f up w              |up w| df + |f w| du + |f up| dw, + 2^-16 |h| for the two bf16 terms and 3 u |h|
      y                       sum |down| dh, + (top (i + 8) + 16) u sum |h| |down| - two products per value and the waves' sums -, + 2 u |beta residual|
    """
    t, h = x.shape
    inter = gate.shape[1]
    logits = x @ router.T
    dl = (h + 2) * U * (np.abs(x) @ np.abs(router).T)
    ids = chosen
    assert ids.min() >= 0 and ids.max() < logits.shape[1] and all(len(set(row)) == top for row in ids.tolist())
    picked = np.take_along_axis(logits, ids, axis=1)
    picked_off = np.take_along_axis(dl, ids, axis=1)
    assert np.all(picked[:, 1:] <= picked[:, :-1] + picked_off[:, 1:] + picked_off[:, :-1]), "not in descending order"
    others = np.ones(logits.shape, bool)
    np.put_along_axis(others, ids, False, axis=1)
    assert np.all(~others | (logits - dl <= picked[:, -1:] + picked_off[:, -1:])), "a larger logit was not chosen"
    ex = np.exp(picked - picked[:, :1])
    total = ex.sum(axis=1, keepdims=True) if normalise else np.exp(logits - picked[:, :1]).sum(axis=1, keepdims=True)
    weights = ex / total
    off = dl.max(axis=1, keepdims=True)
    dw = (np.expm1(2 * off) + (logits.shape[1] + 16) * U) * np.ones_like(weights)
    y = np.zeros((t, h)) if residual is None else beta * residual
    bound = 2 * U * np.abs(y)
    for e in range(router.shape[0]):
        token, slot = np.nonzero(ids == e)
        if not len(token):
            continue
        xs = x[token]
        w, w_off = weights[token, slot][:, None], (weights * dw)[token, slot][:, None]
        g, u = xs @ gate[e].T, xs @ up[e].T
        dg, du = (h + 2) * U * (np.abs(xs) @ np.abs(gate[e]).T), (h + 2) * U * (np.abs(xs) @ np.abs(up[e]).T)
        f = activation(g, act)
        df = 1.13 * dg + (40 if act == 3 else 4) * 2 * U * np.abs(f) + (2.0 ** -22 if act == 3 else 0.0)
        hidden = f * u * w
        dh = np.abs(u * w) * df + np.abs(f * w) * du + np.abs(f * u) * w_off + (2.0 ** -16 + 3 * U) * np.abs(hidden)
        y[token] += hidden @ down[e].T
        bound[token] += dh @ np.abs(down[e]).T + (top * (inter + 8) + 16) * U * (np.abs(hidden) @ np.abs(down[e]).T)
    return y, weights, bound, dw
