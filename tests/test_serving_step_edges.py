"""Operators of a serving step at the edges of what their documentation allows: other orders of a cache, far strides,
wide integers, long tables, extreme scores."""
import math

import pytest
import torch

import paddle.incubate.nn.functional as IF

import serving_oracle as O
from test_serving_step import BF, DEVICES, FF, HF, frequencies, near, paged


# ------------------------------------------------------------------------------------------ orders of a cache
def slot_major(cache):
    """The same cache in [block, slot, head, D] storage, seen as [block, head, slot, D]."""
    return cache.transpose(1, 2).contiguous().transpose(1, 2)


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('hq,hkv,d,page,plen,own,new,dtype', [
    (8, 4, 128, 64, 300, [70, 129, 1], None, BF),            # whole pages a tile, few rows
    (12, 3, 64, 32, 130, [65, 40], [65, 3], HF),
    (4, 2, 256, 64, 100, [64, 3], None, BF),
    (32, 2, 128, 64, 333, [5, 70] * 8, None, BF),            # prefix items of many rows: pages of a tile, ...
    (32, 2, 64, 16, 333, [5, 70] * 8, None, HF),             # ... of an instruction's rows, ...
    (32, 2, 128, 5, 203, [5, 30] * 8, None, BF),             # ... and of neither
    (16, 2, 256, 64, 200, [2, 33] * 8, None, BF),
    (4, 2, 64, 5, 21, [13, 4], None, HF)])
def test_slot_major_caches(dev, hq, hkv, d, page, plen, own, new, dtype):
    """Appended to and read: slots Hkv * D apart, heads D apart."""
    g = torch.Generator().manual_seed(hq * d + page)
    n = [1] * len(own) if new is None else new
    kc, vc, tables, common = paged(g, own, page, hkv, d, dtype, spare=-(-plen // page))
    cu = None if new is None else torch.tensor([0] + n).cumsum(0).int()
    lens, f = torch.tensor(own, dtype=torch.int32), frequencies(d // 4)
    past = lens - torch.tensor(n, dtype=torch.int32)
    qkv = torch.randn(sum(n), (hq + 2 * hkv) * d, generator=g).to(dtype)
    wq, wk, wv = O.append(qkv, kc, vc, tables, past, cu, f, False, 1.0, plen)
    dk, dv = slot_major(kc.to(dev)), slot_major(vc.to(dev))
    assert dk.stride() == (page * hkv * d, d, hkv * d, 1)
    up = lambda t: None if t is None else t.to(dev)  # noqa: E731
    q, k2, _ = IF.paged_rotary_append(up(qkv), dk, dv, up(tables), up(past), up(cu), up(f), position_offset=plen)
    assert k2._t.data_ptr() == dk.data_ptr()
    step = torch.finfo(dtype).eps / 2
    near(q._t, wq, wq.abs() * step + 1e-5)
    near(dk, wk, wk.abs() * step + 1e-5)
    assert torch.equal(dv.cpu().double(), wv)
    want, _, size = O.attention(q._t.cpu(), dk.cpu(), dv.cpu(), tables, lens, common, plen, cu, 1 / math.sqrt(d))
    got = IF.shared_prefix_attention(q, dk, dv, up(tables), up(lens), up(common), plen, up(cu), max(n))
    near(got._t, want, O.attention_bound(want, size, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [1, 20])                    # prefix items of few rows and of many
@pytest.mark.parametrize('page,stride', [(64, 70_000_000), (16, (1 << 27) + 8), (64, (1 << 25) + 8), (64, 1 << 25)])
def test_slot_strides_beyond_32_bits(page, stride, rows):
    """Slots so far apart that a tile's rows lie up to 9 GB behind each other: a [slot, block, head, D] storage of many
    blocks, of which a few are used."""
    g = torch.Generator().manual_seed(page + rows)
    hq, hkv, d, nblk = 8, 1, 128, 6
    room = torch.empty(page * stride, dtype=BF, device='cuda')
    small = torch.randn(2, nblk, hkv, page, d, generator=g).to(BF)
    kc, vc = (room.as_strided((nblk, hkv, page, d), (hkv * d, d, stride, 1), i * nblk * hkv * d) for i in (0, 1))
    kc.copy_(small[0]), vc.copy_(small[1])
    tables = torch.tensor([[4, 1], [2, 3]] * rows, dtype=torch.int32)
    common, past = torch.tensor([0, 5], dtype=torch.int32), torch.tensor([page, 2 * page - 2] * rows, dtype=torch.int32)
    q = torch.randn(2 * rows, hq, d, generator=g).to(BF)
    want, _, size = O.attention(q, *small, tables, past, common, 2 * page - 3, None, d ** -0.5)
    got = IF.shared_prefix_attention(q.cuda(), kc, vc, tables.cuda(), past.cuda(), common.cuda(), 2 * page - 3)
    near(got._t, want, O.attention_bound(want, size, BF))
    qkv = torch.randn(2, (hq + 2) * d, generator=g).to(BF)
    wq, wk, wv = O.append(qkv, *small, tables[:2], past[:2], None, None, False, 1.0)
    IF.paged_rotary_append(qkv.cuda(), kc, vc, tables[:2].cuda(), past[:2].cuda())
    assert torch.equal(kc.cpu().double(), wk) and torch.equal(vc.cpu().double(), wv)


# ------------------------------------------------------------------------------------------ what a call does not allow
@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('d,dtype', [(64, BF), (128, HF), (64, FF), (80, BF)])   # kernel and composite
def test_more_new_tokens_than_max_seqlen_q(dev, d, dtype):
    """Rows of such a sequence are NaN, the others as ever; a row behind the last sequence is zero."""
    g = torch.Generator().manual_seed(d)
    n, own = [3, 2, 4, 0, 1], [5, 9, 4, 3, 20]
    kc, vc, tables, common = paged(g, own, 16, 2, d, dtype, spare=2)
    cu, lens = torch.tensor([0] + n).cumsum(0).int(), torch.tensor(own, dtype=torch.int32)
    q = torch.randn(sum(n) + 2, 4, d, generator=g).to(dtype)
    want, lse, size = O.attention(q, kc, vc, tables, lens, common, 20, cu, d ** -0.5)
    args = [t.to(dev) for t in (q, kc, vc, tables, lens, common)]
    out, l2 = (t._t.cpu() for t in IF.shared_prefix_attention(*args, 20, cu.to(dev), 2, return_lse=True))
    over = torch.tensor([0, 1, 2, 5, 6, 7, 8])
    fits = torch.tensor([3, 4, 9])
    assert bool(out[over].isnan().all()) and bool(l2[over].isnan().all())
    near(out[fits], want[fits], O.attention_bound(want, size, dtype)[fits])
    near(l2[fits], lse[fits], 1e-3)
    assert float(out[10:].float().abs().sum()) == 0.0 and bool((l2[10:] == -math.inf).all())


# ------------------------------------------------------------------------------------------ 64-bit integers
@pytest.mark.parametrize('dev', DEVICES)
def test_integers_beyond_32_bits(dev):
    """Blocks, lengths and offsets of 64 bits mean what they say: none comes back around as a small one."""
    g = torch.Generator().manual_seed(12)
    big, page, d = 1 << 32, 16, 64
    kc, vc = (torch.randn(6, 1, page, d, generator=g).to(BF) for _ in range(2))
    tables = torch.tensor([[0, 1], [2, 3], [4, 5]])
    wild = torch.tensor([[0, 1], [2 + big, 3], [4, 5 - big]])                  # two blocks that are not the cache's
    lens, f = torch.tensor([17, 5, 20]), frequencies(8)
    qkv = torch.randn(3, 4 * d, generator=g).to(BF)
    up = lambda t: t.to(dev)  # noqa: E731

    def append(tables, lens, offset=0):
        k, v = up(kc.clone()), up(vc.clone())
        q = IF.paged_rotary_append(up(qkv), k, v, up(tables), up(lens), None, up(f), position_offset=offset)[0]
        return q._t.cpu(), k.cpu(), v.cpu()
    known = torch.tensor([[0, 1], [-1, 3], [4, -1]])
    for a, b in zip(append(wild, lens), append(known, lens)):
        assert torch.equal(a, b)
    _, k, v = append(tables, torch.tensor([17, 5 + big, 20 - big]))            # places past the table and before it
    _, k1, v1 = append(torch.tensor([[0, 1], [-1, -1], [-1, -1]]), lens)
    assert torch.equal(k, k1) and torch.equal(v, v1)
    # the length of a prefix before the positions; 1.3e10 radians in 64 bits are good to 3e-6 on either side
    x, far = qkv.double().view(3, 4, d)[:, :2], 3 * big
    for offset in (far, up(torch.tensor([far])), up(torch.tensor(7)), up(torch.tensor([7], dtype=torch.int32))):
        want = O.rotate(x, lens + int(offset), f, False, 1.0)
        near(append(tables, lens, offset)[0], want, O.rotate_bound(x, f, False, 1.0, BF) + 1e-5 * x.abs().amax())

    def attend(tables, lens, prefix, plen, **kw):
        return IF.shared_prefix_attention(up(qkv.view(3, 4, d)), up(kc), up(vc), up(tables), up(lens), up(prefix), plen, **kw)._t.cpu()
    assert torch.equal(attend(wild, lens, torch.tensor([3, 1 + big]), 30), attend(known, lens, torch.tensor([3, -1]), 30))
    assert torch.equal(attend(tables, torch.tensor([17 + big, 5, 20 - big]), torch.tensor([3]), up(torch.tensor(big + 2))),
                       attend(tables, torch.tensor([32, 5, 0]), torch.tensor([3]), 16))
    assert torch.equal(attend(tables, lens, torch.tensor([3]), up(torch.tensor(2 - big))), attend(tables, lens, torch.tensor([3]), 0))
    # offsets of rows that do not fit the call: no sequence's
    none = attend(tables, lens, torch.tensor([3]), 16, cu_seqlens_q=up(torch.tensor([0, 0, 3, 3]) + big), max_seqlen_q=3)
    assert float(none.float().abs().sum()) == 0.0


# ------------------------------------------------------------------------------------------ what has a gradient
@pytest.mark.parametrize('dev', DEVICES)
def test_frequencies_that_want_a_gradient(dev):
    """Frequencies are constants on every device: where a gradient would be lost the call is refused."""
    x, f = torch.randn(1, 3, 2, 16, device=dev), frequencies(4).to(dev)
    learned = f.clone().requires_grad_()
    for q in (x, x.clone().requires_grad_()):
        with pytest.raises(ValueError, match='inv_freq'):
            IF.fused_partial_rotary_embedding(q, q, learned)
        want = IF.fused_partial_rotary_embedding(q, q, f)
        for got in (IF.fused_partial_rotary_embedding(q, q, learned.detach()),):
            assert all(torch.equal(a._t, b._t) for a, b in zip(got, want))
    with torch.no_grad():
        got = IF.fused_partial_rotary_embedding(x, None, learned)[0]
    assert torch.equal(got._t, IF.fused_partial_rotary_embedding(x, None, f)[0]._t)
    assert not got._t.requires_grad


@pytest.mark.parametrize('dev', DEVICES)
def test_rotary_forward_mode(dev):
    """The tangent of a rotation is the rotated tangent, whether the inputs want gradients or not."""
    from torch.autograd import forward_ad
    g = torch.Generator().manual_seed(13)
    mk = lambda h: torch.randn(2, 5, h, 16, generator=g).to(dev)  # noqa: E731
    f, (q, k, tq, tk) = frequencies(6).to(dev), (mk(3), mk(2), mk(3), mk(2))
    turn = lambda q, k: [None if t is None else t._t for t in IF.fused_partial_rotary_embedding(q, k, f, interleaved=True)]  # noqa: E731
    (wq, wk), (vq, vk) = turn(q, k), turn(tq, tk)
    for wanted in (False, True):
        q.requires_grad_(wanted), k.requires_grad_(wanted)
        with forward_ad.dual_level():
            for a, b, ta, tb in ((forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk), vq, vk),
                                 (forward_ad.make_dual(q, tq), k, vq, None), (q, forward_ad.make_dual(k, tk), None, vk),
                                 (forward_ad.make_dual(q, tq), None, vq, None)):
                for out, want, tangent in zip(turn(a, b), (wq, wk), (ta, tb)):
                    if out is None:
                        continue
                    got = forward_ad.unpack_dual(out)
                    assert torch.equal(got.primal, want)
                    if tangent is None:
                        assert got.tangent is None or float(got.tangent.abs().max()) == 0.0
                    else:
                        assert torch.allclose(got.tangent, tangent, atol=1e-6)


# ------------------------------------------------------------------------------------------ extreme scores
@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('plen,rows', [(0, 2), (4000, 2), (4000, 80)])       # own keys, prefix items of few and of many rows
def test_attention_behind_a_sink(dev, dtype, plen, rows):
    """One key takes nearly all of the softmax and has no values; what the rows give comes from thousands of keys
    that are each 2^-26 .. 2^-28 of it."""
    g = torch.Generator().manual_seed(plen + rows)
    own, d, page = 3000 if plen == 0 else 20, 64, 64
    lens = torch.tensor([own] * rows, dtype=torch.int32)
    kc, vc, tables, common = paged(g, [own], page, 1, d, dtype, spare=-(-plen // page))
    tables = tables.expand(rows, -1).contiguous()
    kc.zero_()
    kc[..., 1] = torch.rand(kc.shape[:3], generator=g).to(dtype)             # scores in [-28, -26] times ln 2
    kc[..., 0] = -26.0
    vc.copy_((torch.rand(vc.shape, generator=g) * 20 + 40).to(dtype))
    at = tables[0, 0] if plen == 0 else common[0]
    kc[at, 0, 3], vc[at, 0, 3] = 0.0, 0.0
    q = torch.zeros(rows, 2, d, dtype=dtype)
    q[..., 0], q[..., 1] = 1.0, -2.0
    scale = math.log(2)
    want, lse, size = O.attention(q, kc, vc, tables, lens, common if plen else None, plen, None, scale)
    got, l2 = IF.shared_prefix_attention(q.to(dev), kc.to(dev), vc.to(dev), tables.to(dev), lens.to(dev),
                                         common.to(dev) if plen else None, plen if plen else None, scale=scale, return_lse=True)
    assert float(want.min()) > 5e-4
    # beside the rounding of normal numbers, in fp16 half the smallest step 2^-24 of a probability whose largest is 2^7
    lost = (own + plen) * 2.0 ** -32 * 60 if dtype is HF else 0.0
    near(got._t, want, O.attention_bound(want, size, dtype) + lost)
    near(l2._t, lse, 1e-3)


# ------------------------------------------------------------------------------------------ tables wider than their sequences
def plan(T, B, hq, hkv, d, most, packed, plen, own):
    import ctypes
    from paddle.ops import _native as N
    if N._load() is None:
        pytest.skip(N.load_error)
    out = (ctypes.c_int * 5)()
    N.check(N.lib.pa_prefix_attn_plan(T, B, hq, hkv, d, most, int(packed), plen, own, out), 'prefix_attn_plan')
    return list(out)


@pytest.mark.parametrize('T,B,hq,hkv,d,most', [(8192, 4, 64, 8, 128, 8192), (65536, 64, 64, 8, 128, 2048), (4096, 1, 16, 1, 256, 4096),
                                               (300, 300, 64, 8, 128, 1), (32768, 8, 128, 1, 64, 32768)])
def test_workspace_does_not_follow_the_tables(T, B, hq, hkv, d, most):
    """Tables made for the longest length that is allowed, 2^20 tokens here, beside ones for 8192: at most 1 GiB of
    partial results more."""
    slot = T * hq * (d + 2) * 4
    fits, wide = (plan(T, B, hq, hkv, d, most, most > 1, 5000, own)[4] for own in (8192, 1 << 20))
    assert (wide - fits) * slot <= 1 << 30
    assert wide >= fits


@pytest.mark.gpu
def test_chunks_with_wide_tables():
    """The same chunks with tables that fit and with ones 100 times as wide: answers to the joins' rounding, memory to
    1 GiB."""
    g = torch.Generator().manual_seed(14)
    own, n, hq, hkv, d, page = [2100, 900, 2048], [2048, 900, 1], 32, 2, 128, 64
    kc, vc, tables, common = (t.cuda() for t in paged(g, own, page, hkv, d, BF, spare=2))
    cu, lens = torch.tensor([0] + n).cumsum(0).int().cuda(), torch.tensor(own, dtype=torch.int32).cuda()
    q = torch.randn(sum(n), hq, d, generator=g).to(BF).cuda()
    wide = torch.nn.functional.pad(tables, (0, 100 * tables.shape[1]), value=-1)
    outs, peaks = [], []
    for t in (tables, wide):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        outs.append(IF.shared_prefix_attention(q, kc, vc, t, lens, common, cu_seqlens_q=cu, max_seqlen_q=2048)._t.double())
        peaks.append(torch.cuda.max_memory_allocated() - before)
    assert peaks[1] - peaks[0] <= 1 << 30
    # 8 bits of each probability and of the result, on either side; values of normal size
    assert float((outs[0] - outs[1]).abs().max()) <= 4 * 2.0 ** -8


@pytest.mark.parametrize('dev', DEVICES)
def test_strides_of_one_head(dev):
    """A dimension of size 1 has no stride that matters: caches of one key head (or of pages of one place, or of one
    block) that differ from contiguous ones in nothing else are taken as they are."""
    g = torch.Generator().manual_seed(15)
    for nblk, page, odd in ((5, 16, (16 * 64, 3, 64, 1)), (5, 1, (64, 64, 7, 1)), (1, 16, (5, 64, 64, 1))):
        kc, vc = (torch.randn(nblk, 1, page, 64, generator=g).to(BF).to(dev) for _ in range(2))
        q = torch.randn(1, 4, 64, generator=g).to(BF).to(dev)
        tables, lens = torch.arange(nblk, dtype=torch.int32)[None].to(dev), torch.tensor([nblk * page], dtype=torch.int32).to(dev)
        want = IF.shared_prefix_attention(q, kc, vc, tables, lens)
        got = IF.shared_prefix_attention(q, kc.as_strided(kc.shape, odd), vc.as_strided(vc.shape, odd), tables, lens)
        assert torch.equal(got._t, want._t)


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('dtype', [BF, FF])
def test_interleaved_pairs_at_odd_addresses(dev, dtype):
    """Contiguous views that begin at an odd element: pairs are loaded together, so they are copied first."""
    g = torch.Generator().manual_seed(16)
    f, odd = frequencies(8).to(dev), lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731
    q, k, gq, gk = (torch.randn(1, 3, h, 16, generator=g).to(dtype).to(dev) for h in (3, 2, 3, 2))
    leaves = [t.clone().requires_grad_() for t in (q, k)]

    def both(q, k, gq, gk):
        y = [t._t for t in IF.fused_partial_rotary_embedding(q, k, f, interleaved=True)]
        return [t.detach() for t in y] + list(torch.autograd.grad(y, [q, k], [gq, gk]))
    want = both(*leaves, gq, gk)
    got = both(*(odd(t).detach().requires_grad_() for t in (q, k)), odd(gq), odd(gk))
    assert odd(q).data_ptr() % (2 * q.element_size()) and odd(q).is_contiguous()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    qkv, bias = torch.randn(1, 4 * 16, generator=g).to(dtype).to(dev), torch.randn(64, generator=g).to(dtype).to(dev)
    table, lens = torch.tensor([[1, 0]], dtype=torch.int32).to(dev), torch.tensor([5], dtype=torch.int32).to(dev)
    outs = []
    for x, b in ((qkv, bias), (odd(qkv), bias), (qkv, odd(bias)), (odd(qkv), odd(bias))):
        kc, vc = (torch.zeros(2, 1, 4, 16, dtype=dtype, device=dev) for _ in range(2))
        outs.append((IF.paged_rotary_append(x, kc, vc, table, lens, None, f, True, qkv_bias=b)[0]._t, kc, vc))
        assert all(torch.equal(a, c) for a, c in zip(outs[-1], outs[0]))


# ------------------------------------------------------------------------------------------ scaled frequencies
@pytest.mark.parametrize('rot,base,span,factor', [(64, 10000.0, 4096, 8.0), (128, 500000.0, 8192, 32.0), (32, 100.0, 64, 3.0)])
@pytest.mark.parametrize('bounds', [None, (2.0, 16.0)])
def test_scaled_frequencies_pair_by_pair(rot, base, span, factor, bounds):
    """Every pair by its own formula, the blended ones between the kept and the divided ones among them."""
    plain = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    lo, hi = bounds or (1.0, 4.0)
    want, blended = [], 0
    for f in plain:
        wavelength = 2 * math.pi / f
        if wavelength < span / hi:
            want.append(f)
        elif wavelength > span / lo:
            want.append(f / factor)
        else:
            part = (span / wavelength - lo) / (hi - lo)
            want.append((1 - part) * f / factor + part * f)
            blended += 1
    more = {} if bounds is None else dict(low_freq_factor=lo, high_freq_factor=hi)
    got, s = IF.rotary_inv_freq(rot, base, dict(type='wavelength', factor=factor, original_max_position=span, **more))
    assert blended > 0 and s == 1.0
    assert all(math.isclose(a, b, rel_tol=1e-12) for a, b in zip(got._t.tolist(), want, strict=True))
    # the pair that makes `turns` turns over the span: base ** (-2 i / rot) * span = 2 pi turns, solved for i
    slow, fast = bounds or (1.0, 32.0)
    at = lambda turns: rot * math.log(span / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
    first, last = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
    want = []
    for i, f in enumerate(plain):
        part = min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0)
        want.append(f * (1 - part) + f / factor * part)
    more = {} if bounds is None else dict(beta_slow=slow, beta_fast=fast)
    got, s = IF.rotary_inv_freq(rot, base, dict(type='yarn', factor=factor, original_max_position=span, **more))
    assert any(1 < a / b < factor for a, b in zip(plain, want))
    assert all(math.isclose(a, b, rel_tol=1e-12) for a, b in zip(got._t.tolist(), want, strict=True))
    assert math.isclose(s, 0.1 * math.log(factor) + 1, rel_tol=1e-12)
    assert IF.rotary_inv_freq(rot, base, dict(type='yarn', factor=factor, original_max_position=span, attention_factor=0.75))[1] == 0.75


def test_plan_refuses_calls_without_heads():
    """An error code, not a division by zero."""
    with pytest.raises(RuntimeError):
        plan(4, 4, 0, 2, 64, 1, False, 0, 64)
