"""Plain 64-bit forms of the paged cache's operators, and bounds for their rounding errors."""
import math

import torch

MANTISSA = {torch.float32: 24, torch.bfloat16: 8, torch.float16: 11}      # half a step is 2^-MANTISSA of the value


def sees(parents, N):
    """[N, N] bool: which drafts each draft of one request reads."""
    m = torch.zeros(N, N, dtype=torch.bool)
    for i in range(N):
        p = i - 1 if parents is None else int(parents[i])
        if p < -1:
            continue
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def cached_rows(cache, table_row, length):
    """(rows [length, H_kv, D], there [length]): a page outside the cache is not there."""
    pages, page = cache.shape[:2]
    ids = table_row[:(length + page - 1) // page].long().tolist()
    rows = [cache[i] if 0 <= i < pages else torch.zeros_like(cache[0]) for i in ids]
    ok = torch.tensor([0 <= i < pages for i in ids], dtype=torch.bool).repeat_interleave(page)[:length]
    flat = torch.cat(rows)[:length] if rows else cache.new_zeros(0, *cache.shape[2:])
    return flat, ok


def attention(q, k, v, kc, vc, table, lengths, parents=None, scale=None):
    """(out, lse, bound on |out - exact|, bound on |lse - exact|) in 64 bits, on the CPU.

    Rounding errors counted: a score is a sum of K products in fp32, times a constant: |ds| <= (K + 4) 2^-24 scale sum |q||k|; the
    exponent's own rounding and the exponential, 2^-20 together (a hardware exponential is good to 2 units of 2^-23; the maximum
    subtracted is the same number everywhere); a sum of n terms in fp32 in any order: n 2^-24; in 16 bits the weights are rounded to the
    type, half a step each, and the result once more."""
    dt = q.dtype
    q, k, v, kc, vc, table, lengths = (x.cpu() for x in (q, k, v, kc, vc, table, lengths))
    parents = parents.cpu() if parents is not None else None
    B, N, H, K = q.shape
    Hkv, V = k.shape[2], v.shape[3]
    scale = K ** -0.5 if scale is None else scale
    u = 2.0 ** -MANTISSA[dt]
    out, tol = torch.zeros(B, N, H, V, dtype=torch.float64), torch.zeros(B, N, H, V, dtype=torch.float64)
    lse, ltol = torch.full((B, N, H), -math.inf, dtype=torch.float64), torch.zeros(B, N, H, dtype=torch.float64)
    for b in range(B):
        ck, ok = cached_rows(kc, table[b], int(lengths[b]))
        cv, _ = cached_rows(vc, table[b], int(lengths[b]))
        m = sees(parents[b] if parents is not None else None, N)
        for i in range(N):
            if not m[i, i]:
                continue
            kk, vv = torch.cat([ck[ok], k[b][m[i]]]).double(), torch.cat([cv[ok], v[b][m[i]]]).double()
            for h in range(H):
                kh, vh = kk[:, h // (H // Hkv)], vv[:, h // (H // Hkv)]
                s = scale * (kh @ q[b, i, h].double())
                lse[b, i, h] = s.logsumexp(0)
                w = s.softmax(0)
                out[b, i, h] = w @ vh
                n = len(s)
                ds = ((K + 4) * 2.0 ** -24 * abs(scale) * (kh.abs() @ q[b, i, h].double().abs())).max() + s.abs().max() * 2.0 ** -22 + 2.0 ** -20
                each = 2 * ds + n * 2.0 ** -23 + (u if dt != torch.float32 else 0)
                tol[b, i, h] = u * out[b, i, h].abs() + each * (w @ vh.abs()) + 2.0 ** -24 * (dt == torch.float16)
                ltol[b, i, h] = ds + n * 2.0 ** -24 + (lse[b, i, h].abs() + 1) * 2.0 ** -22
    return out, lse, tol, ltol


def plan(lengths, counts, table, pool, top, page, n):
    """The plan, one request after another; lists and ints."""
    lengths, counts, pool, table = list(lengths), list(counts), list(pool), [list(r) for r in table]
    B, M = len(lengths), len(table[0])
    slots, taken = [[-1] * n for _ in range(B)], [0] * B
    for b in range(B):
        if counts[b] < 0:
            for j in range(-(-lengths[b] // page)):
                pool[top] = table[b][j]
                table[b][j] = -1
                top += 1
            lengths[b] = 0
    have, asked = top, 0
    for b in range(B):
        if counts[b] <= 0 or counts[b] > n or lengths[b] + counts[b] > M * page:
            continue
        held = -(-lengths[b] // page)
        need = -(-(lengths[b] + counts[b]) // page) - held
        asked += need
        if need and asked > have:
            continue
        for j in range(need):
            table[b][held + j] = pool[have - 1 - (asked - need) - j]
        top -= need
        for i in range(counts[b]):
            pos = lengths[b] + i
            slots[b][i] = table[b][pos // page] * page + pos % page
        taken[b] = counts[b]
        lengths[b] += counts[b]
    return slots, taken, lengths, table, pool, top
