"""Attention over a paged KV cache for a batch with a shared prefix, on csrc/prefix_attn.hip, and the
composite that other devices, head dims and 32-bit caches take.

Reference: paddle/phi/kernels/fusion/gpu/block_multi_head_attention_kernel.cu (its pre-cache: a prefix per
sequence).
"""
import ctypes
import math

import torch

from . import _native as N

HEAD_DIMS = (64, 128, 256)


def _hip(t):
    from . import use_hip
    return use_hip(t)


def _pages(cache, table, n):
    """[Hkv, n, D] keys or values of the first n places of a page table, and which of the places exist."""
    page = cache.shape[2]
    j = torch.arange(n, device=cache.device)
    blk = table.long()[j // page]
    has = (blk >= 0) & (blk < cache.shape[0])
    x = cache[blk.clamp(0, cache.shape[0] - 1), :, j % page].transpose(0, 1).float()
    return torch.where(has[None, :, None], x, torch.zeros_like(x)), has


def composite(q, key_cache, value_cache, tables, lens, ptable, plen, cu, most, scale):
    """The definition, sequence by sequence, in 32 bits; a sequence of more than ``most`` new tokens is NaN."""
    T, Hq, D = q.shape
    Hkv, page = key_cache.shape[1], key_cache.shape[2]
    G = Hq // Hkv
    B = lens.shape[0]
    out = torch.zeros(T, Hq, D, dtype=torch.float32, device=q.device)
    lse = torch.full((T, Hq), float('-inf'), device=q.device)
    c = list(range(B + 1)) if cu is None else cu.tolist()
    np_ = 0 if ptable is None else max(0, min(int(plen), ptable.numel() * page))
    kp = vp = None
    if np_:
        kp, hp = _pages(key_cache, ptable, np_)
        vp, _ = _pages(value_cache, ptable, np_)
    for b in range(B):
        r0, n = c[b], c[b + 1] - c[b]
        if n > most:
            out[max(r0, 0):max(r0 + n, 0)] = lse[max(r0, 0):max(r0 + n, 0)] = float('nan')
            continue
        if n <= 0 or r0 < 0 or r0 + n > T:
            continue
        L = max(0, min(int(lens[b]), tables.shape[1] * page))
        k, h = _pages(key_cache, tables[b], L)
        v, _ = _pages(value_cache, tables[b], L)
        see = (torch.arange(L, device=q.device)[None] <= (L - n + torch.arange(n, device=q.device))[:, None]) & h[None]
        if np_:
            k, v = torch.cat([kp, k], 1), torch.cat([vp, v], 1)
            see = torch.cat([hp[None].expand(n, -1), see], 1)
        if k.shape[1] == 0:
            continue
        qq = q[r0:r0 + n].float().view(n, Hkv, G, D).permute(1, 2, 0, 3)                     # [Hkv, G, n, D]
        s = torch.matmul(qq, k[:, None].transpose(-1, -2).contiguous()) * scale
        s = s.masked_fill(~see, float('-inf'))
        m = s.amax(-1, keepdim=True)
        e = torch.where(see, torch.exp(s - torch.where(m == float('-inf'), torch.zeros_like(m), m)), torch.zeros_like(s))
        l_ = e.sum(-1, keepdim=True)
        bad = ~torch.isfinite(v)
        o = torch.matmul(e, torch.where(bad, torch.zeros_like(v), v)[:, None])
        if bool(bad.any()):  # an infinity or NaN reaches the rows that see its key, and no other
            for x in (float('inf'), float('-inf'), float('nan')):
                hit = torch.isnan(v) if x != x else v == x
                o = torch.where(torch.matmul(e, hit.float()[:, None]) > 0, o + x, o)
        o = torch.where(l_ == 0, torch.zeros_like(o), o / l_)
        out[r0:r0 + n] = o.permute(2, 0, 1, 3).reshape(n, Hq, D)
        lse[r0:r0 + n] = (m + torch.log(l_)).squeeze(-1).permute(2, 0, 1).reshape(n, Hq)
    return out.to(q.dtype), lse


def supported(q, key_cache, value_cache):
    """Whether the kernel takes these tensors (else the composite does)."""
    return (_hip(q) and q.dtype in (torch.bfloat16, torch.float16) and key_cache.dtype == q.dtype
            and value_cache.dtype == q.dtype and q.shape[2] in HEAD_DIMS)


def _rows16(t):
    """t with unit inner stride, its other strides and its address multiples of 16 bytes."""
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def attend(q, key_cache, value_cache, tables, lens, ptable, plen, cu, most, scale, want_lse):
    """q [T, Hq, D]; caches [blocks, Hkv, page, D] of equal strides; tables [B, n] / lens [B] / ptable [m] / cu
    [B + 1] int32; plen an int or a one-element int32 tensor.  Returns (out, lse or None)."""
    T, Hq, D = q.shape
    nblk, Hkv, page, _ = key_cache.shape
    B = lens.shape[0]
    most = max(1, min(most, T))
    if not supported(q, key_cache, value_cache):
        with torch.no_grad():
            o, lse = composite(q, key_cache, value_cache, tables, lens, ptable, plen, cu, most, scale)
        return o, lse if want_lse else None
    out = torch.empty(T, Hq, D, dtype=q.dtype, device=q.device)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=q.device) if want_lse else None
    if T == 0 or Hq == 0:
        return out, lse
    if B == 0:
        return out.zero_(), None if lse is None else lse.fill_(float('-inf'))
    q = _rows16(q)
    dev = isinstance(plen, torch.Tensor)
    cap = 0 if ptable is None else ptable.numel() * page
    plan = (ctypes.c_int * 5)()
    N.check(N.lib.pa_prefix_attn_plan(T, B, Hq, Hkv, D, most, int(cu is not None), cap if dev else min(int(plen), cap),
                                      tables.shape[1] * page, plan), 'prefix_attn_plan')
    # this call's own workspace: two streams or two captured graphs never share one
    ws = torch.empty(plan[4] * T * Hq * (D + 2), dtype=torch.float32, device=q.device) if plan[4] else None
    with N.device_of(q):
        N.check(N.lib.pa_prefix_attn(
            N.ptr(q), N.ptr(key_cache), N.ptr(value_cache), q.stride(0), q.stride(1),
            (ctypes.c_longlong * 3)(*key_cache.stride()[:3]), N.ptr(tables), tables.stride(0), tables.shape[1],
            N.ptr(ptable), 0 if ptable is None else ptable.numel(), N.ptr(plen) if dev else None,
            0 if dev else min(int(plen), cap), nblk, page, N.ptr(lens), N.ptr(cu), N.ptr(out), N.ptr(lse), N.ptr(ws),
            plan, T, B, Hq, Hkv, D, most, float(scale), N.dtcode(q.dtype), N.stream()), 'prefix_attn')
    return out, lse
