"""Definitions in 64 bits, with plain loops, of the operators of a serving step: rotary positions, the
rotated append to a paged cache, attention with a shared prefix, sampling from filtered logits."""
import math

import torch


def rotate(x, pos, f, interleaved, scale):
    """x [..., H, D] float64 (pos [...]): the first 2 len(f) values of each head turned."""
    y, h = x.clone(), f.numel()
    a = pos.double()[..., None, None] * f.double()
    c, s = torch.cos(a) * scale, torch.sin(a) * scale
    lo, hi = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
    u, v = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = u * c - v * s, v * c + u * s
    return y


def rotate_bound(x, f, interleaved, scale, dtype):
    """Half a step of the result's type, and 1e-6 of a pair's size: the angle as a 32-bit fraction of a half turn
    (pi 2^-24 = 1.9e-7), sine and cosine within 2 steps (1.2e-7 each), two products and a sum (1.8e-7)."""
    h, z = f.numel(), x.abs()
    pair = torch.zeros_like(z)
    lo, hi = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
    pair[..., lo] = pair[..., hi] = (z[..., lo] + z[..., hi]) * scale
    y = torch.maximum(pair, z)
    return y * (torch.finfo(dtype).eps / 2 + 1e-6) + torch.finfo(dtype).smallest_normal


def append(qkv, kc, vc, tables, lens, cu, f, interleaved, scale, offset=0, bias=None):
    """Returns q and the new caches, all float64."""
    nblk, hkv, page, d = kc.shape
    x = qkv.double() if bias is None else qkv.double() + bias.double()
    x = x.reshape(qkv.shape[0], -1, d)
    hq = x.shape[1] - 2 * hkv
    q, kc, vc = torch.zeros(x.shape[0], hq, d, dtype=torch.float64), kc.double().clone(), vc.double().clone()
    c = list(range(len(lens) + 1)) if cu is None else cu.tolist()
    for b in range(len(lens)):
        for i, r in enumerate(range(c[b], c[b + 1])):
            p = int(lens[b]) + i
            y = x[r, :hq + hkv]
            if f is not None:
                y = rotate(y, torch.tensor(p + offset), f, interleaved, scale)
            q[r] = y[:hq]
            if 0 <= p < tables.shape[1] * page and 0 <= int(tables[b, p // page]) < nblk:
                kc[int(tables[b, p // page]), :, p % page] = y[hq:]
                vc[int(tables[b, p // page]), :, p % page] = x[r, hq + hkv:]
    return q, kc, vc


def attention(q, kc, vc, tables, lens, ptable, plen, cu, scale):
    """Row by row: (out, lse, sum of p |v|), float64."""
    t, hq, d = q.shape
    nblk, hkv, page, _ = kc.shape
    out, size = torch.zeros(t, hq, d, dtype=torch.float64), torch.zeros(t, hq, d, dtype=torch.float64)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64)
    c = list(range(len(lens) + 1)) if cu is None else cu.tolist()

    def places(table, n):
        return [(int(table[j // page]), j % page) for j in range(max(0, min(n, len(table) * page)))]
    pre = [] if ptable is None else [(b, s) for b, s in places(ptable, plen) if 0 <= b < nblk]
    for b in range(len(lens)):
        n = c[b + 1] - c[b]
        mine = places(tables[b], int(lens[b]))
        for i in range(n):
            see = pre + [(k, s) for j, (k, s) in enumerate(mine) if j <= len(mine) - n + i and 0 <= k < nblk]
            if not see:
                continue
            at, sl = torch.tensor([k for k, _ in see]), torch.tensor([s for _, s in see])
            keys, vals = kc[at, :, sl].double(), vc[at, :, sl].double()          # [l, hkv, d]
            for h in range(hq):
                w = keys[:, h // (hq // hkv)] @ q[c[b] + i, h].double() * scale
                p = torch.softmax(w, 0)
                v = vals[:, h // (hq // hkv)]
                out[c[b] + i, h], size[c[b] + i, h] = p @ v, p @ v.abs()
                lse[c[b] + i, h] = torch.logsumexp(w, 0)
    return out, lse, size


def attention_bound(out, size, dtype):
    """Each probability is rounded to the type for the product with the values (half a step of each p |v|), the
    result is rounded once; 1e-4 of sum p |v| for the 32-bit scores (128 products of size 1 to 10 are within 8e-5),
    exponents and sums."""
    half = torch.finfo(dtype).eps / 2
    return size * (half + 1e-4) + out.abs() * half + 1e-7


def sample(x, u, t, k, p, m):
    """One row: (token, share)."""
    x = [float(v) for v in x.double()]
    tokens = [i for i, v in enumerate(x) if v == v and v > -math.inf]
    if not tokens:
        return -1, 0.0
    order = sorted(tokens, key=lambda i: (-x[i], i))
    if not t > 0:
        return order[0], 1.0
    top = x[order[0]]
    w = {i: 1.0 if x[i] == top else (0.0 if top == math.inf else math.exp((x[i] - top) / t)) for i in order}
    if k > 0:
        order = order[:k]
    if p < 1:
        mass, run, kept = math.fsum(w[i] for i in order), 0.0, []
        for i in order:
            if kept and not run < p * mass:
                break
            kept.append(i)
            run += w[i]
        order = kept
    m = min(m, 1.0) if m > 0 else 0.0
    order = sorted(i for i in order if w[i] >= m)
    total, run = math.fsum(w[i] for i in order), 0.0
    for i in order:
        run += w[i]
        if run > max(u, 0.0) * total and w[i] > 0:
            return i, w[i] / total
    last = [i for i in order if w[i] > 0][-1]
    return last, w[last] / total
