"""Rotary positions from frequencies and the rotated append to a paged KV cache, on csrc/rotary_paged.hip,
with composites of elementary operations for tensors off the GPU.

Reference: paddle/phi/kernels/fusion/gpu/fused_rope_kernel.cu, block_attn.h (the cache writes of
block_multihead_attention).
"""
import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import _native as N

MAX_PAIRS = 256  # rotated pairs of a head (csrc/rotary_paged.hip kMaxPairs)
FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _hip(t):
    from . import use_hip
    return use_hip(t)


def _alignment(ts):
    """Elements (at most 8) that divide every address and every stride but the last of the tensors."""
    a = 8
    for t in ts:
        if t is not None and t.numel():
            a = math.gcd(a, t.data_ptr() // t.element_size())
            if t.is_contiguous():
                a = math.gcd(a, t.shape[-1])
            else:
                a = math.gcd(a, *(s for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1))
    return a


def _even(t):
    """t, copied where its address or a stride is odd (contiguous() leaves a view at an odd address as it is)."""
    return t if t is None or _alignment((t,)) % 2 == 0 else t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    return (ctypes.c_longlong * 3)(*t.stride()[:3])


def rotate(x, cos, sin, interleaved):
    """The composite: the first 2 * cos.shape[-1] values of each head of x [..., H, D] turned in 32 bits by the
    angles [..., pairs], rounded once."""
    h = cos.shape[-1]
    c, s, f = cos[..., None, :], sin[..., None, :], x.float()
    if interleaved:
        a, b = f[..., 0:2 * h:2], f[..., 1:2 * h:2]
        r = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = f[..., :h], f[..., h:2 * h]
        r = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([r, f[..., 2 * h:]], -1).to(x.dtype)


def angles(pos, inv_freq, scale):
    a = pos.double()[..., None] * inv_freq.double()
    return (a.cos() * scale).float(), (a.sin() * scale).float()


def _launch(q, k, inv_freq, pos, interleaved, scale, sign):
    B, S, Hq, D = q.shape
    q = q if q.stride(3) == 1 else q.contiguous()
    if k is not None and k.stride(3) != 1:
        k = k.contiguous()
    a = _alignment((q, k))
    if interleaved and a % 2:
        q, k = _even(q), _even(k)
        a = _alignment((q, k))
    yq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    yk = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    f = inv_freq.double().contiguous()
    with N.device_of(q):
        N.check(N.lib.pa_rope_freq(N.ptr(q), N.ptr(k), N.ptr(yq), N.ptr(yk), _strides(q),
                                   None if k is None else _strides(k), B, S, Hq, 0 if k is None else k.shape[2], D,
                                   f.numel(), int(interleaved), N.ptr(f), scale, N.ptr(pos),
                                   0 if pos is None else pos.stride(0), 0 if pos is None else pos.stride(1),
                                   int(pos is not None and pos.dtype == torch.int64), sign, a,
                                   N.dtcode(q.dtype), N.stream()), 'rope_freq')
    return yq, yk


def _tangents():
    """Whether tensors may carry tangents (forward-mode differentiation)."""
    return forward_ad._current_level >= 0


class _RopeFreq(torch.autograd.Function):
    """Linear in (q, k): the backward pass is the forward one with the angles' sign turned, so it has a
    backward pass of its own, and a tangent is turned as its input is."""

    @staticmethod
    def forward(ctx, q, k, inv_freq, pos, interleaved, scale, sign):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(inv_freq, pos)
        ctx.how = (interleaved, scale, sign)
        if _tangents():
            ctx.save_for_forward(inv_freq, pos)
            ctx.like = q, k
        return _launch(q, k, inv_freq, pos, interleaved, scale, sign)

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        inv_freq, pos = ctx.saved_tensors
        q, k = ctx.like
        tq = torch.zeros_like(q) if tq is None else tq
        tk = torch.zeros_like(k) if tk is None and k is not None else tk
        ctx.like = None
        return (_RopeFreq.apply if torch.is_grad_enabled() else _launch)(tq, tk, inv_freq, pos, *ctx.how)

    @staticmethod
    def backward(ctx, dq, dk):
        inv_freq, pos = ctx.saved_tensors
        interleaved, scale, sign = ctx.how
        turn = _RopeFreq.apply if torch.is_grad_enabled() else _launch
        gq = gk = None
        if dq is not None:
            gq, gk = turn(dq, dk, inv_freq, pos, interleaved, scale, -sign)
        elif dk is not None:
            gk, _ = turn(dk, None, inv_freq, pos, interleaved, scale, -sign)
        return gq, gk, None, None, None, None, None


def rope_freq(q, k, inv_freq, pos, interleaved, scale):
    """q [B, S, Hq, D], k [B, S, Hk, D] or None; inv_freq [pairs]; pos [B, S] integers or None (0 .. S - 1)."""
    if _hip(q):
        wanted = _tangents() or torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))
        return (_RopeFreq.apply if wanted else _launch)(q, k, inv_freq, pos, interleaved, float(scale), 1.0)
    p = torch.arange(q.shape[1], device=q.device)[None] if pos is None else pos
    cos, sin = angles(p, inv_freq, scale)
    return rotate(q, cos, sin, interleaved), None if k is None else rotate(k, cos, sin, interleaved)


def paged_append(qkv, key_cache, value_cache, tables, lens, cu, inv_freq, interleaved, scale, bias=None, offset=0):
    """q rows of qkv [T, (Hq + 2 Hkv) D] turned and returned [T, Hq, D]; keys turned and values written into the
    pages of sequence b at places lens[b], lens[b] + 1, ...; the angle's position is the place + offset."""
    nblk, Hkv, page, D = key_cache.shape
    T, B = qkv.shape[0], lens.shape[0]
    Hq = qkv.shape[1] // D - 2 * Hkv
    pairs = 0 if inv_freq is None else inv_freq.numel()
    if _hip(qkv):
        qkv = qkv if qkv.stride(1) == 1 else qkv.contiguous()
        a = _alignment((qkv, key_cache, value_cache, bias))
        if interleaved and a % 2:
            if _alignment((key_cache, value_cache)) % 2:
                raise ValueError("interleaved pairs need caches of even strides")
            qkv, bias = _even(qkv), _even(bias)
            a = _alignment((qkv, key_cache, value_cache, bias))
        q = torch.empty(T, Hq, D, dtype=qkv.dtype, device=qkv.device)
        f = None if inv_freq is None else inv_freq.double().contiguous()
        dev = isinstance(offset, torch.Tensor)
        with N.device_of(qkv):
            N.check(N.lib.pa_paged_append(
                N.ptr(qkv), qkv.stride(0), N.ptr(bias), N.ptr(q), N.ptr(key_cache), N.ptr(value_cache),
                _strides(key_cache), N.ptr(tables), tables.stride(0), tables.shape[1], nblk, page, N.ptr(lens), N.ptr(cu),
                N.ptr(offset) if dev else None, int(dev and offset.dtype == torch.int64), 0 if dev else int(offset), T, B, Hq, Hkv, D, pairs, int(interleaved),
                N.ptr(f), float(scale), a, N.dtcode(qkv.dtype), N.stream()), 'paged_append')
        return q
    with torch.no_grad():
        return _append_composite(qkv, key_cache, value_cache, tables, lens, cu, inv_freq, interleaved, scale, bias, offset)


def _append_composite(qkv, key_cache, value_cache, tables, lens, cu, inv_freq, interleaved, scale, bias, offset):
    nblk, Hkv, page, D = key_cache.shape
    T, B = qkv.shape[0], lens.shape[0]
    Hq = qkv.shape[1] // D - 2 * Hkv
    x = qkv.reshape(T, Hq + 2 * Hkv, D)
    x = x.float() + bias.float().reshape(1, Hq + 2 * Hkv, D) if bias is not None else x
    c = torch.arange(B + 1) if cu is None else cu.long().cpu()
    q = torch.zeros(T, Hq, D, dtype=qkv.dtype, device=qkv.device)
    for b in range(B):
        r0, r1 = max(int(c[b]), 0), min(int(c[b + 1]), T)
        if r1 <= r0:
            continue
        place = int(lens[b]) + torch.arange(r1 - r0, device=qkv.device)
        rows = x[r0:r1]
        qk = rows[:, :Hq + Hkv].to(torch.float32)
        if inv_freq is not None:
            qk = rotate(qk, *angles(place + int(offset), inv_freq, scale), interleaved)
        q[r0:r1] = qk[:, :Hq].to(q.dtype)
        col = torch.div(place, page, rounding_mode='floor')
        has = (place >= 0) & (col < tables.shape[1])
        blk = tables[b].long()[col.clamp(0, tables.shape[1] - 1)]
        has &= (blk >= 0) & (blk < nblk)
        at, slot = blk[has], (place % page)[has]
        key_cache[at, :, slot] = qk[has, Hq:].to(key_cache.dtype)
        value_cache[at, :, slot] = rows[has, Hq + Hkv:].to(value_cache.dtype)
    return q
