"""The operators over a paged cache in whole numbers and 64 bits, for the tests (numpy, no device)."""

import math

import numpy as np

H = 2.0 ** -24  # half a step of fp32


def plan(lengths, new, held, page, table, free, count, cap):
    """One request after the other, with lists.  Returns a dict of the state and the rows' maps."""
    lengths, held, table, free = (np.array(a, np.int64) for a in (lengths, held, table, free))
    requests, width = table.shape
    pages, err, ended = len(free), 0, np.asarray(new) < 0
    if not 0 <= count <= pages:
        count, err = 0, 1
    for b in range(requests):
        if ended[b]:
            if not 0 <= held[b] <= width:
                held[b], err = 0, 1
            for j in range(held[b]):
                if count < pages:
                    free[count] = table[b, j]
                    count += 1
                else:
                    err = 1
            held[b] = lengths[b] = 0
    slot, request, position, cu, served, going = [], [], [], [0], 0, True
    for b in range(requests):
        n = int(new[b])
        if not ended[b]:
            good = 0 <= held[b] <= width and 0 <= lengths[b] <= held[b] * page
            err = err or int(not good)
            need = max(0, -(-(lengths[b] + n) // page) - held[b]) if good else 0
            going = (going and good and need <= count and len(slot) + n <= cap and lengths[b] + n <= width * page)
        if going:
            served += 1
        if going and not ended[b]:
            for _ in range(need):
                count -= 1
                table[b, held[b]] = free[count]
                err = err or int(not 0 <= free[count] < pages)
                held[b] += 1
            for p in range(lengths[b], lengths[b] + n):
                there = 0 <= table[b, p // page] < pages
                err = err or int(not there)
                slot.append(table[b, p // page] * page + p % page if there else -1)
                request.append(b)
                position.append(p)
            lengths[b] += n
        cu.append(len(slot))
    pad = lambda x: np.array(x + [-1] * (cap - len(x)), np.int64)  # noqa: E731
    return dict(lengths=lengths, held=held, table=table, free=free, count=count, cu=np.array(cu), slot=pad(slot),
                request=pad(request), position=pad(position), served=served, err=err)


def visible(length, n, i, window, sinks):
    """Keys that row i of n sees."""
    p = length - n + i
    j = np.arange(max(0, p + 1))
    return j[(j > p - window) | (j < sinks)] if window else j


def attention(q, k, v, length, window=0, sinks=0, scale=1.0):
    """Rows q [n, heads, d] of one request over k, v [length, kv_heads, d], in 64 bits: (out, bound).

    The bound, for fp32 arithmetic in any order with h = 2^-24.  A score is a sum of at most 3 d exact products (fp32
    queries come as three exact parts), each addition off by at most a step, 2 h, of the sum of magnitudes |q||k|; scale
    log2(e) and the reference's subtraction add 6 h of the largest score; exp2 is within a step, 2 h: a weight is off by
    the factor e = exp(off of its score) (1 + 2 h).  Sums over the visible keys, in any order and with three parts a
    weight, are off by at most (3 keys + 16) steps, 2 h each, of the sum of magnitudes (16: joins and rescalings).
    """
    n, heads, d = q.shape
    group = heads // k.shape[1]
    out, bound = np.zeros((n, heads, d)), np.zeros((n, heads, d))
    for i in range(n):
        see = visible(length, n, i, window, sinks)
        if len(see) == 0:
            continue
        for hq in range(heads):
            kk, vv, qq = k[see, hq // group].astype(np.float64), v[see, hq // group].astype(np.float64), q[i, hq].astype(np.float64)
            s = scale * (kk @ qq)
            off = scale * (3 * d + 2) * 2 * H * (np.abs(kk) @ np.abs(qq)) + 6 * H * (np.abs(s).max() + np.abs(s))
            w = np.exp(s - s.max())
            e = np.expm1(off) + 2 * H
            out[i, hq] = (w @ vv) / w.sum()
            steps = (3 * len(see) + 16) * 2 * H
            size = (w * (1 + e)) @ np.abs(vv) / w.sum()
            bound[i, hq] = (w * e) @ np.abs(vv) / w.sum() + (w @ e) / w.sum() * size + 2 * steps * size + 2 * H * np.abs(out[i, hq])
    return out, bound


def masses(logits, temperature, top_k, top_p, min_p):
    """What a row's settings keep, by id: integer masses (temperature 0: 1 at the maximum), and their sum."""
    l = np.array(logits, np.float32) + np.float32(0)
    l = np.where(np.isnan(l), np.float32(-np.inf), l)
    temperature, top_p, min_p = (float(np.float32(x)) for x in (temperature, top_p, min_p))
    kept, top = np.zeros(len(l), np.uint64), int(np.argmax(l))
    if l[top] == -np.inf:
        return kept, 0
    valid = temperature >= 0 and top_p >= 0 and 0 <= min_p <= 1
    if not valid or temperature == 0 or top_k == 1 or top_p == 0:
        kept[top] = 1
        return kept, 1
    with np.errstate(all="ignore"):
        y = np.where(l == l[top], 0.0, (l.astype(np.float64) - np.float64(l[top])) * (math.log2(math.e) / temperature))
        y = np.where(l == -np.inf, -np.inf, y)
        mass = np.where(y >= -45.5, np.rint(np.exp2(np.where(y >= -45.5, y, 0.0)) * 2.0 ** 44), 0.0).astype(np.uint64)
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if l[top] == np.inf:
        order = order[l[order] == np.inf]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        upto = np.cumsum(mass[order], dtype=np.uint64)
        need = max(1, -(-int(upto[-1]) * int(top_p * 2.0 ** 64) // 2 ** 64))
        order = order[:int(np.searchsorted(upto, np.uint64(need))) + 1]
    if min_p > 0:
        order = order[y[order] >= math.log2(min_p)]
    kept[order] = mass[order]
    return kept, int(kept.sum())


def verify(rows, drafts, draft_rows, settings, u, u_draw, why=None):
    """One request: logits rows [n + 1, V], n drafts, draft logits [n, V] (None: looked up; a row None: out of range),
    settings (temperature, top_k, top_p, min_p).  Returns (tokens of the n + 1 rows, accepted)."""
    n, v = len(rows) - 1, len(rows[0])
    share = lambda x: x[0].astype(np.float64) / x[1] if x[1] else np.zeros(v)  # noqa: E731
    token = [-1] * (n + 1)
    for i in range(n + 1):
        got = masses(rows[i], *settings)
        p = share(got)
        left = p
        if i < n:
            t, number = int(drafts[i]), float(np.float32(u[i]))
            q, known = np.zeros(v), True
            if draft_rows is None:
                if 0 <= t < v:
                    q[t] = 1.0
            elif draft_rows[i] is None:
                known = False
            else:
                q = share(masses(draft_rows[i], *settings))
            if known and 0 <= t < v and 0 <= number < 1 and number * q[t] < p[t]:
                token[i] = t
                continue
            left = np.maximum(p - q, 0.0)
        if not got[1]:
            token[i] = 0
            return token, i
        w = np.rint(left * 2.0 ** 51).astype(np.uint64)
        if not w.sum():
            w = np.rint(p * 2.0 ** 51).astype(np.uint64)
        number = float(np.float32(u_draw))
        number = number if 0 <= number < 1 else 0.0
        upto = np.cumsum(w, dtype=np.uint64)
        need = (int(upto[-1]) * int(number * 2.0 ** 32) >> 32) + 1
        token[i] = int(np.searchsorted(upto, np.uint64(need)))
        return token, i


class Cache:
    """Requests' keys and values in pages: caches as the operators lay them out, tables, and what is in them."""

    def __init__(self, rng, lengths, kv_heads, d, page, bf16, width=None, spare=3, stale=None, values="normal"):
        from decode_step_oracle import to_bf16

        held = [-(-n // page) for n in lengths]
        pages = sum(held) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(lengths), width or max(max(held), 1)), -1, np.int32)
        dt = np.uint16 if bf16 else np.float32
        fill = 0 if stale is None else stale  # what slots hold that no key was put into
        one = to_bf16(np.float32([fill]))[0][0] if bf16 else np.float32(fill)
        self.k_cache = np.full((pages, kv_heads, page, d), one, dt)
        self.v_cache = np.full((pages, kv_heads, d, page), one, dt)
        self.k, self.v, at = [], [], 0
        for b, n in enumerate(lengths):
            mine = order[at:at + held[b]]
            at += held[b]
            self.table[b, :held[b]] = mine
            if values == "whole":  # sums of them are exact
                k, v = (rng.integers(-8, 9, size=(n, kv_heads, d)).astype(np.float32) for _ in range(2))
            else:
                k, v = (rng.standard_normal((n, kv_heads, d)).astype(np.float32) for _ in range(2))
            if bf16:
                (kb, k), (vb, v) = to_bf16(k), to_bf16(v)
            else:
                kb, vb = k, v
            self.k.append(k)
            self.v.append(v)
            for j in range(held[b]):
                part = slice(j * page, min(n, (j + 1) * page))
                m = part.stop - part.start
                self.k_cache[mine[j], :, :m] = kb[part].transpose(1, 0, 2)
                self.v_cache[mine[j], :, :, :m] = vb[part].transpose(1, 2, 0)
