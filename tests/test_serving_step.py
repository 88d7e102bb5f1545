"""Operators of a serving step over a paged KV cache (rotary positions from frequencies, the rotated append,
attention with a shared prefix, sampling from filtered logits) against their definitions in 64 bits, on the CPU's
composites and, with the gpu mark, on the HIP kernels; their refusals; and a run of them together."""
import math

import pytest
import torch

import paddle
import paddle.incubate.nn.functional as IF

import serving_oracle as O

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def near(got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    off = (got - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off - bound).max()):.3g} over the bound, worst {float(off.max()):.3g}"


def frequencies(pairs, base=10000.0):
    return base ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))


# ------------------------------------------------------------------------------------------ rotary
@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('shape,rot,dtype', [
    ((2, 5, 4, 2, 64), 64, BF), ((1, 1, 1, 1, 64), 32, HF), ((3, 7, 5, 1, 80), 20, FF), ((1, 130, 3, 3, 128), 128, FF),
    ((2, 3, 8, 2, 96), 24, BF), ((1, 9, 2, 1, 256), 256, HF), ((1, 4, 2, 2, 6), 2, FF), ((2, 1025, 2, 1, 64), 64, BF),
    ((1, 3, 1, 1, 512), 512, BF), ((1, 2, 3, 1, 64), 0, BF)])
def test_rotary_both_ways(dev, interleaved, shape, rot, dtype):
    B, S, hq, hk, D = shape
    g = torch.Generator().manual_seed(S * D + rot)
    qkv = torch.randn(B, S, hq + 2 * hk, D, generator=g).to(dtype)
    gq, gk = torch.randn(B, S, hq, D, generator=g).to(dtype), torch.randn(B, S, hk, D, generator=g).to(dtype)
    f, pos, scale = frequencies(rot // 2), torch.randint(0, 1 << 20, (B, S), generator=g), 1.25
    base = qkv.to(dev)
    q, k = base[:, :, :hq].detach().requires_grad_(), base[:, :, hq:hq + hk].detach().requires_grad_()
    yq, yk = IF.fused_partial_rotary_embedding(q, k, f.to(dev), pos.to(dev), interleaved, scale)
    dq, dk = torch.autograd.grad([yq._t, yk._t], [q, k], [gq.to(dev), gk.to(dev)])
    for got, x, sign in ((yq._t, qkv[:, :, :hq], 1), (yk._t, qkv[:, :, hq:hq + hk], 1), (dq, gq, -1), (dk, gk, -1)):
        x = x.double()
        near(got, O.rotate(x, pos * sign, f, interleaved, scale), O.rotate_bound(x, f, interleaved, scale, dtype))
    # one of the outputs alone, without k, and the gradient of the gradient
    only = torch.autograd.grad(IF.fused_partial_rotary_embedding(q, k, f.to(dev), pos.to(dev), interleaved, scale)[1]._t,
                               k, gk.to(dev))[0]
    assert torch.equal(only, dk)
    alone, none = IF.fused_partial_rotary_embedding(q, None, f.to(dev), pos.to(dev), interleaved, scale)
    assert none is None and torch.equal(alone._t, yq._t)


@pytest.mark.parametrize('dev', DEVICES)
def test_rotary_positions_and_layouts(dev):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 6, 3, 32, generator=g)
    f = frequencies(8)

    def run(t, pos=None, freq=f):
        return IF.fused_partial_rotary_embedding(t.to(dev), None, freq.to(dev), None if pos is None else pos.to(dev))[0]._t.cpu()
    want = run(x, torch.arange(6)[None].expand(2, 6).contiguous())
    assert torch.equal(run(x), want)                                            # default positions
    assert torch.equal(run(x, torch.arange(6, dtype=torch.int32)), want)        # [S], 32-bit
    assert torch.equal(run(x, torch.arange(6)[None]), want)                     # [1, S]
    assert torch.equal(run(x[1]), want[1])                                      # packed tokens
    for strided in (x.transpose(0, 1).contiguous().transpose(0, 1), x.flip(0).flip(0)[:, :, ::1],
                    torch.cat([x, x], -1)[..., :32], torch.cat([x[..., :1], x], -1)[..., 1:],
                    x.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(run(strided), want)
    near(run(x, torch.full((6,), -5)), O.rotate(x.double(), torch.full((2, 6), -5), f, False, 1.0),
         O.rotate_bound(x.double(), f, False, 1.0, FF))
    single = f.float()                                                          # frequencies of 32 bits, as they are
    near(run(x, torch.full((6,), 10 ** 6), single), O.rotate(x.double(), torch.full((2, 6), 10 ** 6), single, False, 1.0),
         O.rotate_bound(x.double(), f, False, 1.0, FF))
    assert run(x[:0]).shape == (0, 6, 3, 32) and run(x[:, :0]).shape == (2, 0, 3, 32)


@pytest.mark.parametrize('dev', DEVICES)
def test_rotary_gradient_against_differences(dev):
    """Linear in its input: a central difference over a unit step is exact but for 32-bit rounding."""
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn(1, 3, 2, 16, generator=g).to(dev).requires_grad_(), torch.randn(1, 3, 2, 16, generator=g).to(dev)
    f = frequencies(6).to(dev)

    def value(t):
        return (IF.fused_partial_rotary_embedding(t, None, f, None, True, 0.5)[0]._t * w).sum()
    grad = torch.autograd.grad(value(x), x)[0]
    e = torch.zeros_like(x)
    for i in range(0, x.numel(), 7):
        e.view(-1)[i] = 1.0
        with torch.no_grad():
            d = (value(x + e) - value(x - e)) / 2
        e.view(-1)[i] = 0.0
        assert abs(float(d - grad.view(-1)[i])) <= 1e-4   # sums of 96 products of size 1 to 10, each within 2^-24
    # the gradient of the gradient: dx = R^T w is linear in w, so d (dx . c) / dw = R c
    w.requires_grad_()
    out = IF.fused_partial_rotary_embedding(x, None, f, None, True, 0.5)[0]._t
    dx = torch.autograd.grad(out, x, w, create_graph=True)[0]
    c = torch.randn(x.shape, generator=g).to(dev)
    want = IF.fused_partial_rotary_embedding(c, None, f, None, True, 0.5)[0]._t
    assert torch.allclose(torch.autograd.grad(dx, w, c)[0], want, atol=1e-5)


def test_rotary_inv_freq_forms():
    f, s = IF.rotary_inv_freq(8, 100.0)
    assert s == 1.0 and f._t.dtype == torch.float64
    want = 100.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8)
    assert torch.allclose(f._t.cpu(), want, rtol=1e-14)
    f, s = IF.rotary_inv_freq(8, 100.0, dict(type='linear', factor=4.0))
    assert torch.allclose(f._t.cpu(), want / 4, rtol=1e-14) and s == 1.0
    f, _ = IF.rotary_inv_freq(8, 100.0, dict(type='ntk', factor=4.0))
    assert float(f._t[0]) == 1.0 and math.isclose(float(f._t[-1]), float(want[-1]) / 4, rel_tol=1e-12)
    plain = IF.rotary_inv_freq(64, 10000.0)[0]._t.cpu()
    for kind in ('wavelength', 'yarn'):
        f, s = IF.rotary_inv_freq(64, 10000.0, dict(type=kind, factor=8.0, original_max_position=4096))
        r = f._t.cpu() / plain
        assert math.isclose(float(r[0]), 1.0, rel_tol=1e-12) and math.isclose(float(r[-1]), 0.125, rel_tol=1e-12)
        assert bool((r[1:] <= r[:-1] + 1e-12).all())
        assert math.isclose(s, 0.1 * math.log(8.0) + 1.0 if kind == 'yarn' else 1.0)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0),
                dict(rotary_dim=8, scaling=dict(type='none')), dict(rotary_dim=8, scaling=dict(type='yarn', factor=2.0)),
                dict(rotary_dim=8, scaling=dict(type='linear', factor=0.0)), dict(rotary_dim=2, scaling=dict(type='ntk'))):
        with pytest.raises(ValueError):
            IF.rotary_inv_freq(**bad)


@pytest.mark.parametrize('dev', DEVICES)
def test_rotary_refusals(dev):
    x, f = torch.randn(1, 2, 2, 16, device=dev), frequencies(4).to(dev)
    bad = [dict(q=x[0, 0]), dict(q=x.double()), dict(inv_freq=f[None]), dict(inv_freq=f.half()), dict(inv_freq=None),
           dict(inv_freq=frequencies(9).to(dev)), dict(k=x.half()), dict(k=x[..., :8]), dict(k=x[:, :1]),
           dict(position_ids=torch.zeros(3, dtype=torch.int64, device=dev)),
           dict(position_ids=torch.zeros(2, device=dev)), dict(q=torch.randn(1, 2, 2, 15, device=dev), interleaved=True)]
    for b in bad:
        with pytest.raises(ValueError):
            IF.fused_partial_rotary_embedding(**dict(dict(q=x, inv_freq=f), **b))


# ------------------------------------------------------------------------------------------ paged caches
def paged(g, lens, page, hkv, d, dtype, spare=0, fill=None, extra_cols=0):
    """Random caches and a table of shuffled blocks for these lengths, -1 behind each sequence's own."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g)
    tables = torch.full((len(lens), max(need + [1]) + extra_cols), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n].int()
        at += n
    shape = (max(total, 1), hkv, page, d)
    kc, vc = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
    if fill is not None:
        kc.fill_(fill), vc.fill_(fill)
    return kc, vc, tables, order[at:].int()


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('hq,hkv,d,rot,page,past,new,dtype', [
    (4, 2, 64, 64, 16, [0, 5, 31], None, BF), (3, 1, 80, 40, 8, [7], None, HF), (6, 6, 64, 16, 4, [0, 3, 9], [5, 0, 2], FF),
    (8, 2, 128, 128, 64, [60, 0, 200], [9, 70, 1], BF), (2, 2, 32, 0, 3, [4, 1], [1, 8], HF),
    (0, 2, 64, 64, 16, [3, 2], None, BF), (5, 1, 96, 36, 16, [11] * 9, [300] * 9, BF)])
def test_append(dev, interleaved, hq, hkv, d, rot, page, past, new, dtype):
    g = torch.Generator().manual_seed(hq * d + len(past))
    n = [1] * len(past) if new is None else new
    kc, vc, tables, _ = paged(g, [a + b for a, b in zip(past, n)], page, hkv, d, dtype, spare=2)
    T = sum(n)
    rows = torch.randn(T + 3, (hq + 2 * hkv) * d + 8, generator=g).to(dtype)
    cu = None if new is None else torch.tensor([0] + n).cumsum(0).int()
    qkv = rows[:T + (0 if new is None else 3), :-8]         # strided rows; with offsets, rows behind the last sequence
    f = frequencies(rot // 2) if rot else None
    bias = torch.randn((hq + 2 * hkv) * d, generator=g).to(dtype) if len(past) == 3 else None
    lens = torch.tensor(past, dtype=torch.int32)
    wq, wk, wv = O.append(qkv, kc, vc, tables, lens, cu, f, interleaved, 1.1, 7, bias)
    dk, dv = kc.to(dev), vc.to(dev)
    q, k2, v2 = IF.paged_rotary_append(rows.to(dev)[:qkv.shape[0], :-8], dk, dv, tables.to(dev), lens.to(dev),
                                       None if cu is None else cu.to(dev), None if f is None else f.to(dev), interleaved,
                                       1.1, None if bias is None else bias.to(dev), 7)
    assert k2._t.data_ptr() == dk.data_ptr() and v2._t.data_ptr() == dv.data_ptr()
    # a pair's size is at most 8 here (sums of two normal values with a bias, times 1.1)
    step = torch.finfo(dtype).eps / 2
    near(q._t, wq, wq.abs() * step + 1e-5)
    near(dk, wk, wk.abs() * step + 1e-5)
    near(dv, wv, wv.abs() * step + (0 if bias is None else 1e-6))
    same = wv == vc.double()
    assert torch.equal(dv.cpu()[same], vc[same])            # what no new token owns is left as it was
    if cu is not None:
        assert float(q._t[T:].abs().sum()) == 0.0
    # the prefix's length on the device
    q3, _, _ = IF.paged_rotary_append(rows.to(dev)[:qkv.shape[0], :-8], dk, dv, tables.to(dev), lens.to(dev),
                                      None if cu is None else cu.to(dev), None if f is None else f.to(dev), interleaved,
                                      1.1, None if bias is None else bias.to(dev), torch.tensor([7], device=dev))
    assert torch.equal(q3._t, q._t)


@pytest.mark.parametrize('dev', DEVICES)
def test_append_without_a_place(dev):
    """Blocks that are not the cache's and places past the table: the queries are turned, nothing is stored."""
    g = torch.Generator().manual_seed(1)
    kc = torch.randn(4, 1, 4, 16, generator=g)
    vc = torch.randn(4, 1, 4, 16, generator=g)
    tables = torch.tensor([[0, -1], [1, 7], [2, 3], [3, 2]], dtype=torch.int32)
    lens = torch.tensor([4, 5, 8, -1], dtype=torch.int32)   # block -1, block 7 of 4, past two blocks, before the first
    qkv = torch.randn(4, 3 * 16, generator=g)
    dk, dv = kc.to(dev), vc.to(dev)
    q, _, _ = IF.paged_rotary_append(qkv.to(dev), dk, dv, tables.to(dev), lens.to(dev), inv_freq=frequencies(8).to(dev))
    assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)
    want = O.rotate(qkv.double().view(4, 3, 16)[:, :1], lens, frequencies(8), False, 1.0)
    near(q._t, want, want.abs() * 2 ** -24 + 1e-5)


@pytest.mark.parametrize('dev', DEVICES)
def test_append_refusals(dev):
    z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device=dev)  # noqa: E731
    i = lambda *s: z(*s, t=torch.int32)  # noqa: E731
    good = dict(qkv=z(2, 4 * 16), key_cache=z(3, 1, 4, 16), value_cache=z(3, 1, 4, 16), block_tables=i(2, 3), seq_lens=i(2))
    IF.paged_rotary_append(**good)
    bad = [dict(qkv=z(2, 4 * 16).half()), dict(qkv=z(2, 16)), dict(qkv=z(2, 50)), dict(qkv=z(3, 4 * 16)),
           dict(value_cache=z(3, 1, 4, 8)), dict(key_cache=z(3, 4, 16)), dict(block_tables=i(2)), dict(seq_lens=i(3)),
           dict(seq_lens=z(2)), dict(cu_seqlens_q=i(2)), dict(block_tables=i(2, 0)), dict(qkv_bias=z(5)),
           dict(inv_freq=frequencies(9).to(dev)), dict(position_offset=i(2)),
           dict(value_cache=z(3, 4, 1, 16).transpose(1, 2)[:, :, :, :]), dict(block_tables=torch.zeros(2, 3, device=dev))]
    for b in bad:
        if 'value_cache' in b and b['value_cache'].stride() == good['key_cache'].stride():
            continue
        with pytest.raises(ValueError):
            IF.paged_rotary_append(**dict(good, **b))


# ------------------------------------------------------------------------------------------ shared prefix
def attention_case(dev, hq, hkv, d, page, plen, own, new, dtype, seed=0, scale=None, behind=0, sharp=1.0, device_len=False):
    g = torch.Generator().manual_seed(seed * 1000 + d + plen)
    kc, vc, tables, common = paged(g, own, page, hkv, d, dtype, spare=-(-plen // page), extra_cols=1)
    n = [1] * len(own) if new is None else new
    cu = None if new is None else torch.tensor([0] + n).cumsum(0).int()
    q = (torch.randn(sum(n) + behind, hq, d, generator=g) * sharp).to(dtype)
    lens = torch.tensor(own, dtype=torch.int32)
    scale_ = 1.0 / math.sqrt(d) if scale is None else scale
    want, lse, size = O.attention(q, kc, vc, tables, lens, common if plen else None, plen, cu, scale_)
    got, glse = IF.shared_prefix_attention(
        q.to(dev), kc.to(dev), vc.to(dev), tables.to(dev), lens.to(dev), common.to(dev) if plen else None,
        (torch.tensor(plen, device=dev) if device_len else plen) if plen else None,
        None if cu is None else cu.to(dev), None if new is None else max(n + [1]), scale, True)
    near(got._t, want, O.attention_bound(want, size, dtype))
    near(torch.where(torch.isinf(lse), torch.zeros_like(lse), glse._t.double().cpu()),
         torch.where(torch.isinf(lse), torch.zeros_like(lse), lse), 1e-3)
    assert torch.equal(torch.isinf(glse._t.cpu()), torch.isinf(lse))


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('hq,hkv,d,page,plen,own,new,dtype', [
    (4, 1, 64, 16, 33, [1, 20, 7], None, BF),            # one token each
    (8, 8, 128, 64, 100, [65, 1], None, BF),             # heads that share nothing
    (7, 1, 128, 32, 300, [40, 129], None, HF),           # odd group
    (20, 1, 64, 16, 64, [31, 32, 33], None, BF),         # a group beyond one row tile
    (16, 2, 256, 16, 70, [15, 260], None, BF),
    (4, 2, 64, 5, 21, [13, 4], None, HF),                # pages that fit no tile
    (2, 1, 128, 1, 3, [40, 2], None, BF),                # pages of one token
    (4, 2, 64, 16, 0, [17, 50], None, BF),               # no prefix: straight to the output
    (4, 2, 128, 16, 600, [9], None, BF),                 # several ranges of the prefix
    (6, 2, 64, 16, 40, [12, 40, 3, 9], [5, 33, 3, 0], BF),   # ragged chunks, one sequence without new tokens
    (8, 1, 128, 64, 130, [90, 70], [90, 3], HF),
    (4, 4, 256, 8, 17, [30, 18], [18, 17], BF),
    (16, 1, 64, 16, 16, [6, 2], [4, 2], BF),
    (16, 2, 64, 16, 200, [3, 40] * 20, None, BF),        # prefix items of many rows
    (8, 1, 128, 64, 333, [5] * 33, None, HF),
    (8, 1, 128, 5, 203, [5] * 17, None, BF),
    (16, 1, 256, 8, 130, [2, 33] * 5, None, BF),
    (12, 2, 128, 32, 1200, [30, 40], [30, 25], BF)])
def test_attention(dev, hq, hkv, d, page, plen, own, new, dtype):
    attention_case(dev, hq, hkv, d, page, plen, own, new, dtype, behind=0 if new is None else 2)


@pytest.mark.parametrize('dev', DEVICES)
def test_attention_empty_and_long_parts(dev):
    attention_case(dev, 4, 2, 64, 16, 0, [0, 5, 0], None, BF)             # rows that see nothing
    attention_case(dev, 4, 2, 64, 16, 9, [0, 5], None, BF)                # rows that see the prefix alone
    attention_case(dev, 4, 2, 64, 16, 0, [2, 3], [4, 3], BF)              # more new tokens than keys
    attention_case(dev, 4, 2, 64, 16, 5, [2, 3], [4, 3], BF, device_len=True)
    attention_case(dev, 2, 1, 64, 16, 37, [33, 64], None, BF, scale=0.37, sharp=4.0)   # sharp rows
    attention_case(dev, 2, 1, 128, 16, 64, [2100, 3], None, HF)           # more pages than a wave's window
    attention_case(dev, 2, 1, 64, 1, 150, [170, 3], None, HF)
    attention_case(dev, 16, 1, 128, 1, 150, [0, 3] * 5, None, BF)
    attention_case(dev, 32, 2, 64, 16, 4500, [0, 3] * 5, None, BF, device_len=True)


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('dtype', [BF, HF])
def test_attention_what_lies_behind_the_keys(dev, dtype):
    """NaN and infinities in unused slots, unallocated blocks, and in later tokens of the same call."""
    g = torch.Generator().manual_seed(5)
    hq, hkv, d, page = 4, 2, 64, 16
    own, n = [21, 40, 9], [3, 40, 2]
    kc, vc, tables, common = paged(g, own, page, hkv, d, dtype, spare=4)
    cu, lens = torch.tensor([0, 3, 43, 45], dtype=torch.int32), torch.tensor(own, dtype=torch.int32)
    tables[1, 1] = -1                                       # keys 16 .. 31 of sequence 1 are nowhere
    q = torch.randn(45, hq, d, generator=g).to(dtype)
    scale = 1 / math.sqrt(d)
    want, _, size = O.attention(q, kc, vc, tables, lens, common, 50, cu, scale)
    used = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for t, m in [(common, 50)] + [(tables[b], own[b]) for b in range(3)]:
        for j in range(m):
            if int(t[j // page]) >= 0:
                used[int(t[j // page]), j % page] = True
    for fill in (float('nan'), float('inf')):
        k2, v2 = kc.clone(), vc.clone()
        k2.transpose(1, 2)[~used], v2.transpose(1, 2)[~used] = fill, fill
        got = IF.shared_prefix_attention(q.to(dev), k2.to(dev), v2.to(dev), tables.to(dev), lens.to(dev), common.to(dev),
                                         50, cu.to(dev), 40)._t
        near(got, want, O.attention_bound(want, size, dtype))
    # the last new token of sequence 1 has a NaN and infinities among its values: its own rows alone take them
    last = (int(tables[1, 39 // page]), 39 % page)
    v2 = vc.clone()
    v2[last[0], :, last[1], 3], v2[last[0], :, last[1], 5], v2[last[0], :, last[1], 6] = \
        float('nan'), float('inf'), float('-inf')
    got = IF.shared_prefix_attention(q.to(dev), kc.to(dev), v2.to(dev), tables.to(dev), lens.to(dev), common.to(dev), 50,
                                     cu.to(dev), 40)._t.cpu()
    rows = torch.ones(45, dtype=torch.bool)
    rows[42] = False
    near(got[rows], want[rows], O.attention_bound(want, size, dtype)[rows])
    assert bool(got[42, :, 3].isnan().all()) and bool((got[42, :, 5] == float('inf')).all())
    assert bool((got[42, :, 6] == float('-inf')).all())
    near(got[42, :, 8:], want[42, :, 8:], O.attention_bound(want, size, dtype)[42, :, 8:])
    # a NaN among the keys that a row sees reaches that row and no other
    k2 = kc.clone()
    k2[last[0], :, last[1]] = float('nan')
    got = IF.shared_prefix_attention(q.to(dev), k2.to(dev), vc.to(dev), tables.to(dev), lens.to(dev), common.to(dev), 50,
                                     cu.to(dev), 40)._t.cpu()
    near(got[rows], want[rows], O.attention_bound(want, size, dtype)[rows])
    assert bool(got[42].isnan().all())


@pytest.mark.parametrize('dev', DEVICES)
def test_attention_lengths_beyond_tables_and_strides(dev):
    g = torch.Generator().manual_seed(6)
    hq, hkv, d, page = 4, 2, 64, 16
    both = torch.randn(6, 2, hkv, page, d, generator=g).to(BF)          # keys and values of a block side by side
    kc, vc = both[:, 0], both[:, 1]
    tables, lens = torch.tensor([[0, 5], [3, 1]], dtype=torch.int32), torch.tensor([99, -4], dtype=torch.int32)
    wide = torch.randn(2, 3 * hq, d, generator=g).to(BF)
    q = wide[:, hq:2 * hq]
    want, _, size = O.attention(q, kc, vc, tables, torch.tensor([32, 0]), torch.tensor([2]), 11, None, 0.125)
    b2, w2 = both.to(dev), wide.to(dev)
    got = IF.shared_prefix_attention(w2[:, hq:2 * hq], b2[:, 0], b2[:, 1], tables.to(dev), lens.to(dev),
                                     torch.tensor([2], device=dev), 11)
    near(got._t, want, O.attention_bound(want, size, BF))
    whole = IF.shared_prefix_attention(w2[:, hq:2 * hq], b2[:, 0], b2[:, 1], tables.to(dev), lens.to(dev),
                                       torch.tensor([2, 4], device=dev))
    want, _, size = O.attention(q, kc, vc, tables, torch.tensor([32, 0]), torch.tensor([2, 4]), 32, None, 0.125)
    near(whole._t, want, O.attention_bound(want, size, BF))


@pytest.mark.gpu
@pytest.mark.parametrize('page', [64, 16, 3])
def test_offsets_beyond_32_bits(page):
    """Pages around and behind 2^31 and 2^32 bytes of a cache, appended to and read."""
    g = torch.Generator().manual_seed(8)
    hq, hkv, d = 4, 1, 128
    size = hkv * page * d * 2
    nblk = (9 << 29) // size                                            # 4.5 GiB
    used = [(1 << 31) // size - 1, (1 << 31) // size, (1 << 31) // size + 1, (1 << 32) // size - 1, (1 << 32) // size,
            (1 << 32) // size + 1, nblk - 1, 0]
    kc, vc = (torch.empty(nblk, hkv, page, d, dtype=BF, device='cuda') for _ in range(2))
    small = torch.randn(2, len(used), hkv, page, d, generator=g).to(BF)
    at = torch.tensor(used, device='cuda')
    kc[at], vc[at] = small[0].cuda(), small[1].cuda()
    table = torch.tensor([[4, 1, 6], [2, 3, 7]], dtype=torch.int32)     # indexes into `used`
    common = torch.tensor([0, 5], dtype=torch.int32)
    there = torch.tensor(used, dtype=torch.int32)
    past = torch.tensor([2 * page - 1, 3 * page - 1], dtype=torch.int32)
    qkv = torch.randn(2, (hq + 2) * d, generator=g).to(BF)
    f = frequencies(64)
    wq, wk, wv = O.append(qkv, small[0], small[1], table, past, None, f, False, 1.0, 2 * page)
    q, _, _ = IF.paged_rotary_append(qkv.cuda(), kc, vc, there[table.long()].cuda(), past.cuda(), inv_freq=f.cuda(),
                                     position_offset=2 * page)
    step = torch.finfo(BF).eps / 2
    near(q._t, wq, wq.abs() * step + 1e-5)
    near(kc[at], wk, wk.abs() * step + 1e-5)
    assert torch.equal(vc[at].cpu().double(), wv)
    now = kc[at].cpu(), vc[at].cpu()
    want, _, bound = O.attention(q._t.cpu(), *now, table, past + 1, common, 2 * page, None, d ** -0.5)
    got = IF.shared_prefix_attention(q, kc, vc, there[table.long()].cuda(), (past + 1).cuda(), there[common.long()].cuda())
    near(got._t, want, O.attention_bound(want, bound, BF))


@pytest.mark.parametrize('dev', DEVICES)
def test_attention_refusals(dev):
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=dev)  # noqa: E731
    i = lambda *s: z(*s, t=torch.int32)  # noqa: E731
    good = dict(query=z(2, 4, 64), key_cache=z(3, 2, 4, 64), value_cache=z(3, 2, 4, 64), block_tables=i(2, 3), seq_lens=i(2))
    IF.shared_prefix_attention(**good)
    bad = [dict(query=z(2, 256)), dict(query=z(2, 3, 64)), dict(query=z(2, 4, 32)), dict(query=z(2, 4, 64).half()),
           dict(query=z(3, 4, 64)), dict(block_tables=i(2)), dict(seq_lens=i(1)), dict(cu_seqlens_q=i(4)),
           dict(prefix_len=3), dict(prefix_blocks=i(2), prefix_len=9), dict(prefix_blocks=i(2), prefix_len=-1),
           dict(prefix_blocks=z(2)), dict(prefix_blocks=i(2, 1)), dict(scale=0.0), dict(scale=-1.0), dict(scale=float('nan')),
           dict(cu_seqlens_q=i(3), max_seqlen_q=0), dict(value_cache=z(3, 2, 8, 64)[:, :, ::2])]
    for b in bad:
        with pytest.raises(ValueError):
            IF.shared_prefix_attention(**dict(good, **b))
    over = IF.shared_prefix_attention(**dict(good, query=z(4, 4, 64), cu_seqlens_q=torch.tensor([0, 3, 4], device=dev,
                                                                                               dtype=torch.int32),
                                             seq_lens=torch.tensor([5, 5], device=dev), max_seqlen_q=3))
    assert bool(torch.isfinite(over._t).all())
    none = IF.shared_prefix_attention(z(0, 4, 64), good['key_cache'], good['value_cache'], i(0, 3), i(0))
    assert none._t.shape == (0, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize('cu', [[0, 5, 3, 8], [-3, 2, 4, 8], [0, 9, 9, 12], [2 ** 31 - 1, -2 ** 31, 5, 8], [0, 0, 0, 0]])
def test_offsets_that_do_not_fit(cu):
    """Offsets that fall, start before the first row or end behind the last: nothing outside the tensors is read or
    written (the queries of a sequence with such offsets are not defined), the caches' other places stay."""
    g = torch.Generator().manual_seed(9)
    kc, vc, tables, common = paged(g, [40, 40, 40], 16, 2, 64, BF, spare=3)
    qkv = torch.randn(8, 8 * 64, generator=g).to(BF).cuda()
    cu, lens, old = torch.tensor(cu, dtype=torch.int32).cuda(), torch.tensor([4, 5, 6], dtype=torch.int32).cuda(), kc.clone()
    dk, dv, tables = kc.cuda(), vc.cuda(), tables.cuda()
    q, _, _ = IF.paged_rotary_append(qkv, dk, dv, tables, lens, cu, frequencies(8).cuda())
    common = common.cuda()
    assert q._t.shape == (8, 4, 64) and torch.equal(dk[common.long()].cpu(), old[common.cpu().long()])
    out = IF.shared_prefix_attention(q, dk, dv, tables, lens, common, 40, cu, 8)
    torch.cuda.synchronize()
    assert out._t.shape == (8, 4, 64)
    if int(cu.abs().sum()) == 0:
        assert float(out._t.float().abs().sum()) == 0.0


# ------------------------------------------------------------------------------------------ sampling
def sampling_case(dev, x, u, t, k, p, m):
    probs, ids = paddle.filtered_sampling(x.to(dev), u.to(dev), *(v.to(dev) if isinstance(v, torch.Tensor) else v
                                                                  for v in (t, k, p, m)))
    assert probs._t.dtype == torch.float32 and ids._t.dtype == torch.int64 and ids._t.shape == (x.shape[0], 1)
    at = lambda v, r: v[r].item() if isinstance(v, torch.Tensor) else v  # noqa: E731
    for r in range(x.shape[0]):
        token, share = O.sample(x[r], float(u[r]), at(t, r), at(k, r), at(p, r), at(m, r))
        assert int(ids._t[r, 0]) == token, (r, int(ids._t[r, 0]), token)
        assert abs(float(probs._t[r, 0]) - share) <= share * 2 ** -23 + 1e-9


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('vocab,dtype', [(1, FF), (2, BF), (63, HF), (64, FF), (1000, BF), (5003, FF), (9000, HF)])
def test_sampling_settings(dev, vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    rows = 12
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    u = torch.rand(rows, generator=g, dtype=torch.float64)
    one = torch.ones(rows)
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 5, 1.0, 0.0), (1.0, 40, 0.8, 0.05), (0.0, 3, 0.5, 0.5),
                       (1.0, 1, 1.0, 0.0), (2.0, 0, 1.0, 0.2), (0.9, 0, 0.0, 0.0), (0.05, 7, 0.99, 0.0),
                       (torch.rand(rows, generator=g) + 0.1, torch.randint(0, 30, (rows,), generator=g),
                        torch.rand(rows, generator=g), torch.rand(rows, generator=g) * 0.2),
                       (one * 0.5, one.long() * vocab, one, one), (1.0, 10 ** 6, 1.5, -1.0)):
        sampling_case(dev, x, u, t, k, p, m)
    sampling_case(dev, x, u.float(), 0.8, 20, 0.95, 0.01)


@pytest.mark.parametrize('dev', DEVICES)
def test_sampling_ties_and_masks(dev):
    g = torch.Generator().manual_seed(2)
    inf, nan = float('inf'), float('nan')
    flat = torch.zeros(8, 700)
    flat[:, 5] = -0.0
    u = torch.tensor([0.0, 0.1, 0.25, 0.5, 0.75, 0.9, 0.999999, 0.3], dtype=torch.float64)
    for k, p in ((0, 1.0), (9, 1.0), (0, 0.5), (64, 0.25), (3, 0.34), (0, 0.0)):
        sampling_case(dev, flat, u, 1.0, k, p, 0.0)                     # equal logits: the lowest indexes
    few = torch.randint(0, 3, (8, 700), generator=g).float()
    for k, p in ((0, 0.9), (300, 1.0), (250, 0.7), (1, 0.5)):
        sampling_case(dev, few, u, 0.9, k, p, 0.0)
    masked = torch.randn(8, 700, generator=g)
    masked[torch.rand(8, 700, generator=g) < 0.97] = -inf
    masked[0], masked[1, 3], masked[2] = -inf, nan, nan
    masked[3, 10:20] = torch.finfo(FF).min                              # the lowest value is a token
    masked[4], masked[4, 13] = -inf, -3.0                               # one token left
    masked[5, [7, 400]] = inf
    masked[6] = torch.finfo(FF).min
    for k, p, m in ((0, 1.0, 0.0), (4, 1.0, 0.0), (0, 0.8, 0.0), (0, 1.0, 0.3), (5, 0.9, 0.1)):
        sampling_case(dev, masked, u, 1.0, k, p, m)
    sampling_case(dev, masked, u, 0.0, 0, 1.0, 0.0)
    sampling_case(dev, masked.bfloat16(), u, 1.0, 3, 0.9, 0.0)
    for edge in (1.0, 2.0, -1.0):                                       # numbers outside [0, 1): the ends
        sampling_case(dev, masked, torch.full((8,), edge), 1.0, 0, 0.9, 0.0)


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('vocab,dtype', [(8192, FF), (8193, BF), (20001, FF), (40000, HF)])
def test_sampling_large_vocabularies(dev, vocab, dtype):
    """Several chunks; borders in bins of few tokens, and of more than the kernel ranks (flat rows, many ties)."""
    g = torch.Generator().manual_seed(vocab)
    rows = 8
    x = torch.randn(rows, vocab, generator=g) * 2.5
    x[:, ::997] += 6.0
    x[1] = 0.25                                                         # one value
    x[2] = torch.randint(0, 2, (vocab,), generator=g).float()           # two values
    x[3, vocab // 2:] = float('-inf')
    x[4] *= 0.01                                                        # nearly flat
    x[5], x[5, vocab - 1] = float('-inf'), 1.0                          # the last token alone
    x[6] -= 1e4
    x[7, 17] = float('inf')
    x = x.to(dtype)
    u = torch.rand(rows, generator=g, dtype=torch.float64)
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.0, vocab // 3, 1.0, 0.0), (1.0, vocab // 3, 0.7, 0.0),
                       (0.8, 50, 0.95, 0.02), (1.0, 0, 1.0, 0.9), (3.0, 0, 0.999, 1e-3), (0.01, 5000, 0.999, 0.0),
                       (0.0, 0, 1.0, 0.0), (1e-40, 0, 1.0, 0.0), (float('inf'), 0, 0.5, 0.0)):
        sampling_case(dev, x, u, t, k, p, m)


@pytest.mark.gpu
@pytest.mark.parametrize('vocab,settings', [(150001, ((1.0, 0, 0.9, 0.0), (0.8, 700, 0.95, 0.0), (1.0, 0, 1.0, 0.0))),
                                            (600007, ((1.0, 0, 0.5, 0.0), (0.7, 900, 1.0, 0.001), (2.0, 0, 1.0, 0.0)))])
def test_sampling_vocabularies_of_many_chunks(vocab, settings):
    """More parts than are looked through at a time (131072 tokens), more chunks than the shifts held (524288)."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(2, vocab, generator=g) * 2.5
    x[1, vocab - 400:] += 4.0                        # the candidates lie in the last chunk
    for t, k, p, m in settings:
        sampling_case('cuda', x, torch.tensor([0.37, 0.992], dtype=torch.float64), t, k, p, m)


@pytest.mark.parametrize('dev', DEVICES)
def test_sampling_strided_rows_and_empty(dev):
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(5, 1300, generator=g)
    u = torch.rand(5, generator=g)
    probs, ids = paddle.filtered_sampling(wide.to(dev)[:, 3:1204], u.to(dev).reshape(5, 1), 0.9, 50, 0.9)
    p2, i2 = paddle.filtered_sampling(wide[:, 3:1204].contiguous().to(dev), u.to(dev), 0.9, 50, 0.9)
    assert torch.equal(ids._t, i2._t) and torch.equal(probs._t, p2._t)
    p3, i3 = paddle.filtered_sampling(wide.to(dev).t().contiguous().t()[:, 3:1204], u.to(dev), 0.9, 50, 0.9)
    assert torch.equal(ids._t, i3._t)
    p4, i4 = paddle.filtered_sampling(torch.empty(0, 10, device=dev), torch.empty(0, device=dev))
    assert i4._t.shape == (0, 1) and p4._t.shape == (0, 1)


@pytest.mark.parametrize('dev', DEVICES)
def test_sampling_settings_of_other_types(dev):
    g = torch.Generator().manual_seed(10)
    x, u = torch.randn(4, 300, generator=g), torch.rand(4, generator=g)
    nan = float('nan')

    def run(*settings):
        probs, ids = paddle.filtered_sampling(x.to(dev), u.to(dev), *(v.to(dev) if isinstance(v, torch.Tensor) else v
                                                                      for v in settings))
        return ids._t.cpu().reshape(-1).tolist(), probs._t.cpu()
    full = lambda v, t: torch.full((4,), v, dtype=t)  # noqa: E731
    plain = run(0.8, 0, 0.9, 0.01)
    for k in (2 ** 40 + 3, -2 ** 40 + 3, full(2 ** 40 + 3, torch.int64), full(-2 ** 40 + 3, torch.int64)):  # all
        assert run(0.8, k, 0.9, 0.01)[0] == plain[0]
    for t in (torch.float64, torch.float32):
        same = run(full(0.75, t), full(7, torch.int64), full(0.5, t), full(0.125, t))
        want = run(0.75, 7, 0.5, 0.125)
        assert same[0] == want[0] and torch.equal(same[1], want[1])
    first = x.argmax(-1).tolist()
    assert run(nan, 0, 1.0, 0.0)[0] == first and run(1.0, 0, nan, 0.0)[0] == first and run(1.0, 0, full(nan, FF), 0.0)[0] == first
    assert run(0.8, 0, 0.9, nan)[0] == run(0.8, 0, 0.9, 0.0)[0]
    paddle_u = paddle.filtered_sampling(x.to(dev), full(nan, FF).to(dev))[1]._t.cpu().reshape(-1).tolist()
    assert paddle_u == [0] * 4
    # columns and expanded numbers as settings
    wide = torch.rand(4, 3, generator=g) + 0.5
    want = [O.sample(x[r], float(u[r]), float(wide[r, 1]), 9, 0.875, 0.0)[0] for r in range(4)]
    assert run(wide[:, 1], torch.tensor(9, dtype=torch.int32).expand(4), torch.tensor([0.875]).expand(4), 0.0)[0] == want


@pytest.mark.parametrize('dev', DEVICES)
def test_sampling_refusals(dev):
    x, u = torch.randn(3, 9, device=dev), torch.rand(3, device=dev)
    for bad in ((x[0], u), (x.double(), u), (x[:, :0], u), (x, u[:2]), (x, u.long()), (x, 0.5)):
        with pytest.raises(ValueError):
            paddle.filtered_sampling(*bad)
    for bad in (dict(temperature=u[:2]), dict(top_k=u), dict(top_p=torch.zeros(3, dtype=torch.int64, device=dev)),
                dict(min_p=u[None, :2])):
        with pytest.raises(ValueError):
            paddle.filtered_sampling(x, u, **bad)


# ------------------------------------------------------------------------------------------ together
class Step:
    """A layer of attention between an embedding and logits, over a paged cache behind a shared prefix.  Everything
    but the four operators is a lookup, so that runs can be compared bit by bit."""

    def __init__(self, dev, dtype, prompts, steps, plen, hq=4, hkv=2, d=64, page=16, vocab=200):
        g = torch.Generator().manual_seed(7)
        total = [n + steps for n in prompts]
        self.kc, self.vc, self.tables, self.common = (t.to(dev) for t in
                                                      paged(g, total, page, hkv, d, dtype, spare=-(-plen // page)))
        self.embed = torch.randn(vocab, (hq + 2 * hkv) * d, generator=g).to(dtype).to(dev)
        self.pick = torch.randint(0, hq * d, (vocab,), generator=g).to(dev)     # logits: values of the output
        self.u = torch.rand(steps, len(prompts), generator=g).to(dev)
        self.f, self.scale, self.plen = frequencies(d // 4).to(dev), 1.07, plen
        self.prompts = [torch.randint(0, vocab, (n,), generator=g).to(dev) for n in prompts]
        self.top_k = torch.tensor([0, 5, 40][:len(prompts)], device=dev, dtype=torch.int32)

    def append(self, tokens, lens, cu=None):
        return IF.paged_rotary_append(self.embed[tokens], self.kc, self.vc, self.tables, lens, cu, self.f, True, self.scale,
                                      position_offset=self.plen)[0]

    def attend(self, q, lens, cu=None, most=None):
        return IF.shared_prefix_attention(q, self.kc, self.vc, self.tables, lens, self.common, self.plen, cu, most)

    def sample(self, out, u):
        x = out._t.reshape(out.shape[0], -1)[:, self.pick] * 9
        return x, *paddle.filtered_sampling(x, u, 0.7, self.top_k, 0.9, 0.01)

    def prefill(self):
        """The prompts' keys and values; each one's last token goes to the first step."""
        n = torch.tensor([len(p) - 1 for p in self.prompts], dtype=torch.int32)
        cu = torch.cat([torch.zeros(1, dtype=torch.int32), n.cumsum(0).int()]).to(self.kc.device)
        none = torch.zeros(len(n), dtype=torch.int32, device=self.kc.device)
        if int(cu[-1]):
            self.append(torch.cat([p[:-1] for p in self.prompts]), none, cu)
        return n.to(self.kc.device), torch.stack([p[-1] for p in self.prompts])


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('dtype', [BF, HF, FF])
def test_decode_loop(dev, dtype):
    """Prompts appended in one ragged call, then single tokens: every step against the definitions on what the caches
    held before it, and the caches at the end against one call of the whole sequences."""
    steps, prompts, plen = 4, [5, 1, 20], 33
    s = Step(dev, dtype, prompts, steps, plen)
    start = s.kc.clone(), s.vc.clone()
    lens, tokens = s.prefill()
    said = [list(p.cpu()) for p in s.prompts]
    for i in range(steps):
        old, f = (s.kc.cpu(), s.vc.cpu()), s.f.cpu()
        q = s.append(tokens, lens)
        wq, wk, wv = O.append(s.embed[tokens].cpu(), *old, s.tables.cpu(), lens.cpu(), None, f, True, s.scale, plen)
        half = torch.finfo(dtype).eps / 2
        near(q._t, wq, wq.abs() * half + 1e-5)
        near(s.kc, wk, wk.abs() * half + 1e-5)
        assert torch.equal(s.vc.cpu().double(), wv)
        lens = lens + 1
        out = s.attend(q, lens)
        want, _, size = O.attention(q._t.cpu(), s.kc.cpu(), s.vc.cpu(), s.tables.cpu(), lens.cpu(), s.common.cpu(), plen, None,
                                    1 / math.sqrt(q.shape[2]))
        near(out._t, want, O.attention_bound(want, size, dtype))
        x, probs, ids = s.sample(out, s.u[i])
        for b in range(len(prompts)):
            token, share = O.sample(x[b].cpu(), float(s.u[i, b]), 0.7, int(s.top_k[b]), 0.9, 0.01)
            assert int(ids._t[b, 0]) == token
            assert abs(float(probs._t[b, 0]) - share) <= share * 2 ** -23 + 1e-9
            said[b].append(ids._t[b, 0].cpu())
        tokens = ids._t[:, 0]
    whole = Step(dev, dtype, prompts, steps, plen)
    whole.kc.copy_(start[0]), whole.vc.copy_(start[1])
    n = torch.tensor([len(t) - 1 for t in said], dtype=torch.int32)
    whole.append(torch.cat([torch.stack(t[:-1]) for t in said]).to(dev), torch.zeros_like(n).to(dev),
                 torch.cat([torch.zeros(1, dtype=torch.int32), n.cumsum(0).int()]).to(dev))
    assert torch.equal(whole.kc, s.kc) and torch.equal(whole.vc, s.vc)


def run_steps(s, lens, tokens, replay=None):
    """Steps one after the other, in place on (lens, tokens, u): what is said, and the last outputs."""
    said = []
    u = s.u[0].clone()

    def step():
        q = s.append(tokens, lens)
        lens.add_(1)
        out = s.attend(q, lens)
        _, probs, ids = s.sample(out, u)
        tokens.copy_(ids._t[:, 0])
        return out._t, probs._t
    if replay is not None:
        replay(step)
    for i in range(s.u.shape[0]):
        u.copy_(s.u[i])
        outs = step() if replay is None else replay(None)
        said.append((tokens.clone(), outs[0].clone(), outs[1].clone()))
    return said


class Captured:
    def __init__(self, s, lens, tokens):
        self.keep = (s, lens, tokens)

    def __call__(self, step):
        if step is not None:
            s, lens, tokens = self.keep
            was = s.kc.clone(), s.vc.clone(), lens.clone(), tokens.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.outs = step()
            for t, v in zip((s.kc, s.vc, lens, tokens), was):   # (the step that warmed up)
                t.copy_(v)
            return None
        self.graph.replay()
        return self.outs


@pytest.mark.gpu
def test_captured_steps_replay():
    """Steps replayed from a graph, with eager steps of another batch and synchronizations between, give what eager
    steps give; two graphs and an eager batch at once on three streams as well."""
    def fresh():
        s = Step('cuda', BF, [5, 1, 20], 6, 40)
        return s, *s.prefill()
    want = run_steps(*fresh())

    def same(got):
        for w, g in zip(want, got, strict=True):
            for a, b in zip(w, g):
                assert torch.equal(a, b)
    same(run_steps(*fresh()))                                   # the same again, bit by bit
    s, lens, tokens = fresh()
    cap = Captured(s, lens, tokens)

    def between(step):
        if step is None:
            same(run_steps(*fresh()))
            torch.cuda.synchronize()
        return cap(step)
    same(run_steps(s, lens, tokens, between))
    torch.cuda.synchronize()
    # at once
    runs = []
    for k in range(3):
        s, lens, tokens = fresh()
        u, got = s.u[0].clone(), []
        cap = Captured(s, lens, tokens) if k < 2 else None

        def step(s=s, lens=lens, tokens=tokens, u=u):
            q = s.append(tokens, lens)
            lens.add_(1)
            out = s.attend(q, lens)
            _, probs, ids = s.sample(out, u)
            tokens.copy_(ids._t[:, 0])
            return out._t, probs._t
        if cap is not None:
            cap(step)
        runs.append((s, tokens, u, got, (lambda cap=cap: cap(None)) if cap is not None else step, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for i in range(6):
        for s, tokens, u, got, go, stream in runs:
            with torch.cuda.stream(stream):
                u.copy_(s.u[i])
                outs = go()
                got.append((tokens.clone(), outs[0].clone(), outs[1].clone()))
    torch.cuda.synchronize()
    for r in runs:
        same(r[3])


@pytest.mark.gpu
def test_rotary_captured_both_ways():
    """Forward and backward in one graph, of leaves that no eager graph holds, replayed between eager calls."""
    g = torch.Generator().manual_seed(5)
    mk = lambda: torch.randn(2, 65, 6, 64, generator=g).to(BF).cuda()  # noqa: E731
    f = frequencies(16).cuda()
    x, dy = mk().requires_grad_(), mk()

    def both(x, dy):
        q, k = IF.fused_partial_rotary_embedding(x[:, :, :4], x[:, :, 4:], f)
        return torch.cat([q._t.detach(), k._t.detach()], 2), torch.autograd.grad([q._t, k._t], x, [dy[:, :, :4], dy[:, :, 4:]])[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(x, dy)
    for _ in range(4):
        a, b = mk(), mk()
        with torch.no_grad():
            x.copy_(a), dy.copy_(b)
        graph.replay()
        want = both(a.requires_grad_(), b)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_answers_do_not_change_between_calls():
    """Sums by atomics are of integers, joins have one order."""
    g = torch.Generator().manual_seed(6)
    x = (torch.randn(9, 60000, generator=g) * 2).to(BF).cuda()
    u = torch.rand(9, generator=g).cuda()
    kc, vc, tables, common = paged(g, [70, 300, 5] * 8, 16, 2, 128, BF, spare=80)
    q = torch.randn(24, 16, 128, generator=g).to(BF).cuda()
    lens = torch.tensor([70, 300, 5] * 8, dtype=torch.int32).cuda()
    args = q, kc.cuda(), vc.cuda(), tables.cuda(), lens, common.cuda(), 1270
    first = None
    for _ in range(5):
        got = [t._t for t in (*paddle.filtered_sampling(x, u, 0.9, 0, 0.95), *paddle.filtered_sampling(x, u, 1.5, 3000, 0.9, 1e-4),
                              *IF.shared_prefix_attention(*args, return_lse=True))]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))
