"""Sampling of one token per row from filtered logits on csrc/sampling.hip, and its composite.

Reference: paddle/phi/kernels/gpu/top_p_sampling_kernel.cu.
"""
import torch

from . import _native as N


def _hip(t):
    from . import use_hip
    return use_hip(t)


def composite(x, u, temperature, top_k, top_p, min_p):
    """The definition in 64 bits; the settings are scalars or [rows, 1] tensors."""
    rows, V = x.shape
    xd = x.double()
    xd = torch.where(torch.isnan(xd), torch.full_like(xd, float('-inf')), xd)

    def setting(v, dt):
        return v.to(dt).reshape(-1, 1).expand(rows, 1) if isinstance(v, torch.Tensor) else \
            torch.full((rows, 1), v, dtype=dt, device=x.device)
    t, p, m = (setting(v, torch.float64) for v in (temperature, top_p, min_p))
    k = setting(top_k, torch.int64)
    m = torch.where(m > 0, m.clamp(max=1.0), torch.zeros_like(m))
    u = u.double().reshape(rows, 1)
    u = torch.where(u >= 0, u, torch.zeros_like(u))
    greedy = ~(t > 0)
    w, at = torch.sort(xd, dim=-1, descending=True, stable=True)
    top, token = w[:, :1], w > float('-inf')
    w = torch.exp((w - top) / torch.where(greedy, torch.ones_like(t), t))
    w = torch.where(torch.isinf(top), (xd.gather(1, at) == top).double(), w)  # +inf beside anything finite
    col = torch.arange(V, device=x.device)[None]
    w = torch.where(token & (col < torch.where(greedy, torch.ones_like(k), torch.where(k > 0, k, V))), w, 0.0)
    kept = (w.cumsum(-1) - w < p * w.sum(-1, keepdim=True)) | (p >= 1) | (col == 0)
    w = torch.where(kept & (w >= m), w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, at, w)
    total = w.sum(-1, keepdim=True)
    c = w.cumsum(-1)
    last = torch.where(w > 0, col, torch.full_like(col, -1)).amax(-1, keepdim=True)
    hit = (c > u * total) & (w > 0)
    ids = torch.where(hit.any(-1, keepdim=True), hit.int().argmax(-1, keepdim=True), last)
    probs = torch.where(ids >= 0, w.gather(1, ids.clamp(min=0)) / total, torch.zeros_like(total))
    return probs.float(), ids


def sample(x, u, temperature, top_k, top_p, min_p):
    """x [rows, V]; u [rows]; the settings scalars or [rows] tensors (fp32, top_k int32).  Returns (probs fp32, ids int64), [rows, 1]."""
    rows, V = x.shape
    if not _hip(x):
        with torch.no_grad():
            return composite(x, u, temperature, top_k, top_p, min_p)
    x = x if x.stride(1) == 1 else x.contiguous()
    u = (u if u.dtype in (torch.float32, torch.float64) else u.float()).contiguous()
    keep = []

    def setting(v):
        if not isinstance(v, torch.Tensor):
            return None, v
        keep.append(v.contiguous())
        return N.ptr(keep[-1]), 0
    (tp, t0), (kp, k0), (pp, p0), (mp, m0) = (setting(v) for v in (temperature, top_k, top_p, min_p))
    ids = torch.empty(rows, 1, dtype=torch.int64, device=x.device)
    probs = torch.empty(rows, 1, dtype=torch.float32, device=x.device)
    if rows == 0:
        return probs, ids
    # this call's own workspace: two streams or two captured graphs never share one
    ws = torch.empty(rows * N.lib.pa_sample_ws_bytes(V), dtype=torch.uint8, device=x.device)
    with N.device_of(x):
        N.check(N.lib.pa_sample(N.ptr(x), x.stride(0), rows, V, N.ptr(u), int(u.dtype == torch.float64), tp, kp, pp, mp,
                                float(t0), int(k0), float(p0), float(m0), N.ptr(ids), N.ptr(probs), N.ptr(ws), N.dtcode(x.dtype),
                                N.stream()), 'sample')
    return probs, ids
