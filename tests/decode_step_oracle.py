"""The decode-step operators in 64 bits and whole numbers, for the tests (numpy, no device)."""

import math

import numpy as np


def to_bf16(x):
    """fp32 -> (bfloat16 bits as uint16, the values they stand for), round to nearest even."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    h = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    h = np.where(np.isnan(x), np.uint16(0x7FC0), h)
    return h, (h.astype(np.uint32) << 16).view(np.float32)


def rms_norm(x, r, scale, eps):
    """(s in fp32, y in 64 bits)."""
    s = x if r is None else (x + r).astype(np.float32)
    d = s.astype(np.float64)
    return s, d / np.sqrt((d * d).mean(axis=1, keepdims=True) + np.float64(np.float32(eps))) * scale.astype(np.float64)


def quantize_rows(y):
    """int8 codes and multipliers of fp32 rows, in the library's 32-bit arithmetic."""
    m = np.abs(y).max(axis=1)
    a = np.where(m > 0, np.float32(127) / np.where(m > 0, m, np.float32(1)), np.float32(1)).astype(np.float32)
    return np.clip(np.rint(y * a[:, None]), -127, 127).astype(np.int8), a


def lora(x, q, a, w, mult, bias, la, lb, scale, rank, slot, relu=False):
    """The layer in 64 bits, and a bound on what 32-bit arithmetic in any order may differ by.

    Per product of the base: one rounding each of a w, its reciprocal, the accumulator (exact below 2^24), the product
    and the addition of the bias.  A sum of n fp32 products in any order, fused or not, is off by at most n half steps of
    the sum of magnitudes (each partial result is rounded once, each product at most once).
    """
    h = 2.0 ** -24
    base = (q.astype(np.float64) @ w.astype(np.float64).T) / (a.astype(np.float64)[:, None] * mult.astype(np.float64))
    y = base + bias
    bound = h * (4 * np.abs(base) + np.abs(y))
    for m in range(len(x)):
        s = slot[m]
        if s < 0 or rank[s] == 0:
            continue
        k, r = x.shape[1], rank[s]
        A, B, X = la[s, :r].astype(np.float64), lb[s, :, :r].astype(np.float64), x[m].astype(np.float64)
        c = np.float64(scale[s])
        t, size = A @ X, np.abs(A) @ np.abs(X)
        off = (k + 8) * h * size                  # of t, with the split of x and the gain
        d = c * (B @ t)
        y[m] += d
        bound[m] += abs(c) * (np.abs(B) @ off + (r + 8) * h * (np.abs(B) @ (np.abs(t) + off))) + 2 * h * np.abs(y[m])
    if relu:
        y = np.maximum(y, 0.0)
    return y, bound


def sample(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """(place, logprob) of one row: masses as whole multiples of 2^-44, sums in whole numbers."""
    l = np.array(logits, np.float32) + np.float32(0)
    temperature, top_p, min_p, u = (float(np.float32(v)) for v in (temperature, top_p, min_p, u))
    if l.size == 0:
        return -1, -math.inf
    l = np.where(np.isnan(l), np.float32(-np.inf), l)
    top = int(np.argmax(l))
    if l[top] == -np.inf:
        return 0, -math.inf
    valid = temperature >= 0 and top_p >= 0 and 0 <= min_p <= 1 and 0 <= u < 1
    if not valid or temperature == 0 or top_k == 1 or top_p == 0:
        return top, 0.0
    with np.errstate(all="ignore"):
        y = np.where(l == l[top], 0.0, (l.astype(np.float64) - np.float64(l[top])) * (math.log2(math.e) / temperature))
        y = np.where(l == -np.inf, -np.inf, y)
        mass = np.where(y >= -45.5, np.rint(np.exp2(np.where(y >= -45.5, y, 0.0)) * 2.0 ** 44), 0.0).astype(np.uint64)
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        upto = np.cumsum(mass[order], dtype=np.uint64)
        need = max(1, -(-int(upto[-1]) * int(top_p * 2.0 ** 64) // 2 ** 64))
        order = order[:int(np.searchsorted(upto, np.uint64(need))) + 1]
    if min_p > 0:
        order = order[y[order] >= math.log2(min_p)]
    ids = np.sort(order)
    upto = np.cumsum(mass[ids], dtype=np.uint64)
    total = int(upto[-1])
    need = (total * int(u * 2.0 ** 32) >> 32) + 1
    at = int(ids[int(np.searchsorted(upto, np.uint64(need)))])
    return at, float(y[at] * math.log(2.0) - math.log(total * 2.0 ** -44))
