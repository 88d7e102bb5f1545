"""Measured cases of the operators of one serving step over a paged KV cache.

Rotary positions (part of the head, scaled for long contexts; forward and backward), the append of
a step's keys and values to the pages with the rotation applied on the way, attention of a batch
that shares a long prefix, and sampling from filtered logits with given random numbers.

``run`` computes the plain form (elementary torch operations in 32 bits, 64 where the value of an
angle or of a sum next to a border decides) unless ``own`` is set, in which case it calls the
framework.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

_DT = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
_SIZE = {'bf16': 2, 'fp16': 2, 'fp32': 4}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one training micro-batch of the Llama-2 13B attention: both directions, whole heads
        dict(name='rope_train_13b', op='rope', batch=2, seq=4096, hq=40, hkv=40, d=128, rot=128, dtype='bf16',
             interleaved=False, factor=1.0, first=0),
        # long-context fine-tuning of a grouped-query model: a quarter of the head rotated, positions past
        # a million, frequencies stretched, an odd length
        dict(name='rope_far_partial', op='rope', batch=1, seq=2777, hq=32, hkv=8, d=128, rot=32, dtype='fp32',
             interleaved=True, factor=32.0, first=1000003),
        # the queries and keys of one decode step
        dict(name='rope_decode', op='rope', batch=16, seq=1, hq=32, hkv=8, d=128, rot=128, dtype='bf16',
             interleaved=False, factor=8.0, first=5000),
        # one decode step of 16 sequences: latency
        dict(name='append_decode', op='append', batch=16, most=1, hq=32, hkv=8, d=128, rot=128, dtype='bf16',
             interleaved=False, page=64, past=4000),
        # a mixed step: chunks of prompts of up to 600 tokens beside decodes, half of a 64-wide head rotated
        dict(name='append_mixed', op='append', batch=37, most=600, hq=16, hkv=16, d=64, rot=32, dtype='fp16',
             interleaved=True, page=16, past=1500),
        # a few users of one system prompt: latency
        dict(name='prefix_few', op='prefix', batch=4, most=1, hq=32, hkv=8, d=128, prefix=1000, tail=150, page=16,
             dtype='bf16'),
        # an ordinary serving batch of grouped-query heads (the 8B configuration) behind a long system prompt
        dict(name='prefix_batch', op='prefix', batch=64, most=1, hq=32, hkv=8, d=128, prefix=8192, tail=1000, page=64,
             dtype='bf16'),
        # many samples of one long document
        dict(name='prefix_many', op='prefix', batch=256, most=1, hq=64, hkv=8, d=128, prefix=32768, tail=1500, page=64,
             dtype='bf16'),
        # ragged chunks of new tokens (prompts after the shared part), 64-wide heads that share nothing
        dict(name='prefix_chunks', op='prefix', batch=9, most=67, hq=12, hkv=12, d=64, prefix=2051, tail=700, page=32,
             dtype='fp16'),
        # one sequence of a chat: all filters on
        dict(name='sample_one', op='sample', rows=1, vocab=50304, dtype='fp32', kind='all'),
        # a batch at the largest vocabulary of the repository's models, nucleus alone
        dict(name='sample_nucleus', op='sample', rows=64, vocab=128256, dtype='bf16', kind='nucleus'),
        # a large batch in which every request brings its own settings
        dict(name='sample_many', op='sample', rows=512, vocab=32000, dtype='fp32', kind='mixed'),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['rope', 'append', 'prefix', 'sample'])
    if op == 'rope':
        d = rng.choice([64, 80, 96, 128, 256])
        hkv = rng.choice([1, 2, 5, 8])
        hq = hkv * rng.choice([1, 3, 4, 8])
        tokens = _log(rng, 1, 2 * 4096 * 80 * 128 // ((hq + hkv) * d))
        batch = rng.randint(1, min(8, tokens))
        return dict(op=op, batch=batch, seq=max(1, min(tokens // batch, 16384)), hq=hq, hkv=hkv, d=d,
                    rot=rng.choice([d, d // 2, d // 4 // 2 * 2]), dtype=rng.choice(['bf16', 'fp16', 'fp32']),
                    interleaved=rng.random() < 0.5, factor=rng.choice([1.0, 4.0, 32.0]), first=_log(rng, 1, 1 << 20))
    if op == 'append':
        most = rng.choice([1, 1, 4, _log(rng, 8, 700)])
        return dict(op=op, batch=_log(rng, 1, 256 if most < 8 else 32), most=most, hq=(h := rng.choice([1, 4, 8, 16])) *
                    rng.choice([1, 3, 4]), hkv=h, d=(d := rng.choice([64, 80, 128])), rot=rng.choice([d, d // 2]),
                    dtype=rng.choice(['bf16', 'fp16']), interleaved=rng.random() < 0.5,
                    page=rng.choice([8, 16, 32, 64, 128]), past=_log(rng, 10, 4000))
    if op == 'prefix':
        most = rng.choice([1, 1, 3, _log(rng, 5, 100)])
        hkv = rng.choice([1, 2, 4, 8])
        return dict(op=op, batch=_log(rng, 1, 128 if most < 8 else 12), most=most, hq=hkv * rng.choice([1, 4, 5, 7, 8]),
                    hkv=hkv, d=rng.choice([64, 128, 256]), prefix=_log(rng, 1, 20000), tail=_log(rng, max(1, most), 1500),
                    page=rng.choice([8, 16, 32, 64, 128]), dtype=rng.choice(['bf16', 'fp16']))
    return dict(op=op, rows=_log(rng, 1, 300), vocab=_log(rng, 1000, 130000), dtype=rng.choice(['bf16', 'fp16', 'fp32']),
                kind=rng.choice(['all', 'nucleus', 'top_k', 'mixed', 'plain']))


# ----------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(int(seed) * 7919 + 17)


def _rand(g, *shape, dtype='fp32', scale=1.0):
    """Normal values; large arrays straight in their own type, with no copy in 32 bits."""
    return torch.randn(*shape, generator=g, device='cuda', dtype=_DT[dtype]).mul_(scale)


def _frequencies(rot, factor, base=500000.0, span=8192):
    """Angles per position of the rot / 2 pairs, the slow ones stretched by `factor` (each pair by how
    many turns it makes over the `span` positions trained on: over 32 kept, under 1 divided)."""
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    turns = span * f / (2 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return (f * keep + f / factor * (1.0 - keep)).cuda()


def _lengths(batch, lo, hi, step):
    """`batch` lengths spread over [lo, hi], the first the longest: the same for every seed, so that what
    comes out has one shape."""
    i = torch.arange(batch, device='cuda')
    return (hi - (i * step) % (hi - lo + 1)).to(torch.int32)


def _new_tokens(batch, most):
    """How many new tokens each sequence brings: one each, or some one and some up to `most`."""
    n = _lengths(batch, 1, most, 37)
    return torch.where(torch.arange(batch, device='cuda') % 3 == 1, torch.ones_like(n), n)


def _cumulative(n):
    return torch.cat([torch.zeros(1, dtype=torch.int32, device='cuda'), n.cumsum(0).to(torch.int32)])


def _pages(g, lens, page, spare):
    """A block table for these lengths: the pages of all sequences in random order, -1 past a sequence's own."""
    need = (lens + page - 1) // page
    first = need.cumsum(0) - need
    total = int(need.sum()) + spare
    order = torch.randperm(total, generator=g, device='cuda').to(torch.int32)
    col = torch.arange(int(need.max()), device='cuda', dtype=torch.int32)
    at = (first[:, None] + col[None, :]).clamp(max=total - 1).long()
    table = torch.where(col[None, :] < need[:, None], order[at], torch.full_like(order[at], -1))
    return table.contiguous(), order[total - spare:].contiguous(), total


def prepare(case, seed):
    g, c = _gen(seed), dict(case)
    op, dt = c['op'], c['dtype']
    if op == 'rope':
        b, s, d = c['batch'], c['seq'], c['d']
        # what a fused projection gives: queries, keys and values of a token side by side
        qkv = _rand(g, b, s, c['hq'] + 2 * c['hkv'], d, dtype=dt)
        start = torch.randint(0, 64, (b, 1), generator=g, device='cuda') + c['first']
        f = _frequencies(c['rot'], c['factor'])
        return dict(c, q=qkv[:, :, :c['hq']].detach().requires_grad_(), gq=_rand(g, b, s, c['hq'], d, dtype=dt),
                    k=qkv[:, :, c['hq']:c['hq'] + c['hkv']].detach().requires_grad_(),
                    gk=_rand(g, b, s, c['hkv'], d, dtype=dt), inv_freq=f,
                    pos=start + torch.arange(s, device='cuda')[None, :],
                    scale=1.0 if c['factor'] == 1.0 else 0.1 * math.log(c['factor']) + 1.0)
    if op == 'append':
        mixed = torch.randperm(c['batch'], generator=g, device='cuda')
        n = _new_tokens(c['batch'], c['most'])[mixed]
        past = _lengths(c['batch'], c['past'] // 2, c['past'], 211)[mixed]
        table, _, total = _pages(g, past + n, c['page'], 0)
        cu = _cumulative(n)
        shape = (total, c['hkv'], c['page'], c['d'])
        return dict(c, qkv=_rand(g, int(cu[-1]), (c['hq'] + 2 * c['hkv']) * c['d'], dtype=dt), table=table, past=past,
                    cu=cu if c['most'] > 1 else None, kc=_rand(g, *shape, dtype=dt), vc=_rand(g, *shape, dtype=dt),
                    inv_freq=_frequencies(c['rot'], 4.0), scale=0.1 * math.log(4.0) + 1.0)
    if op == 'prefix':
        mixed = torch.randperm(c['batch'], generator=g, device='cuda')
        n = _new_tokens(c['batch'], c['most'])[mixed]
        tail = torch.maximum(_lengths(c['batch'], (c['tail'] + 2) // 3, c['tail'], 211)[mixed], n)
        blocks = -(-c['prefix'] // c['page'])
        table, common, total = _pages(g, tail, c['page'], blocks)
        cu = _cumulative(n)
        shape = (total, c['hkv'], c['page'], c['d'])
        return dict(c, q=_rand(g, int(cu[-1]), c['hq'], c['d'], dtype=dt, scale=1.5), table=table, common=common,
                    lens=tail, cu=cu if c['most'] > 1 else None, kc=_rand(g, *shape, dtype=dt),
                    vc=_rand(g, *shape, dtype=dt))
    # logits of a language model: a broad bulk, and a few tokens that stand out of it
    rows, vocab = c['rows'], c['vocab']
    x = _rand(g, rows, vocab, scale=2.5)
    x += torch.rand(rows, vocab, generator=g, device='cuda').sub_(0.999).clamp_(min=0.0).mul_(9000.0)
    if c['kind'] == 'mixed':  # a grammar that forbids some tokens
        x.masked_fill_(torch.rand(rows, vocab, generator=g, device='cuda') < 0.1, float('-inf'))
    u = lambda: torch.rand(rows, generator=g, device='cuda')  # noqa: E731
    whole = lambda v, t=torch.float32: torch.full((rows,), v, device='cuda', dtype=t)  # noqa: E731
    kind = c['kind']
    some = torch.arange(rows, device='cuda')
    t, k, p, m = whole(1.0), whole(0, torch.int32), whole(1.0), whole(0.0)
    if kind == 'all':
        t, k, p, m = whole(0.8), whole(50, torch.int32), whole(0.95), whole(0.02)
    elif kind == 'nucleus':
        t, p = whole(0.7), whole(0.9)
    elif kind == 'top_k':
        k = torch.randint(1, 400, (rows,), generator=g, device='cuda', dtype=torch.int32)
    elif kind == 'mixed':
        t = torch.where(some % 7 == 3, torch.zeros_like(t), 0.5 + u())
        k = torch.where(some % 3 == 0, torch.randint(1, 200, (rows,), generator=g, device='cuda', dtype=torch.int32), k)
        p = torch.where(some % 2 == 0, 0.5 + 0.5 * u(), p)
        m = torch.where(some % 5 == 1, 0.1 * u(), m)
    return dict(c, x=x.to(_DT[dt]), u=u(), t=t, k=k, p=p, m=m)


# ------------------------------------------------------------------------------------- plain forms
def _angles(pos, inv_freq, scale):
    """Cosine and sine of each position's angles, in 64 bits (a far position times a frequency)."""
    a = pos.double()[..., None] * inv_freq.double()
    return (a.cos() * scale), (a.sin() * scale)


def _turn(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] values of each head of x [..., heads, d] turned by the angles [..., pairs]."""
    h = cos.shape[-1]
    cos, sin = cos[..., None, :].to(x.dtype), sin[..., None, :].to(x.dtype)
    if interleaved:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:2 * h]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r, x[..., 2 * h:]], -1)


def _rope_plain(s):
    cos, sin = _angles(s['pos'], s['inv_freq'], s['scale'])
    with torch.no_grad():
        return dict(q=_turn(s['q'].float(), cos, sin, s['interleaved']).to(s['q'].dtype),
                    k=_turn(s['k'].float(), cos, sin, s['interleaved']).to(s['k'].dtype),
                    dq=_turn(s['gq'].float(), cos, -sin, s['interleaved']).to(s['q'].dtype),
                    dk=_turn(s['gk'].float(), cos, -sin, s['interleaved']).to(s['k'].dtype))


def _token_places(s):
    """Sequence of each token and its place in it, counted from the sequence's first cached token."""
    t = s['qkv'].shape[0]
    if s['cu'] is None:
        seq = torch.arange(t, device='cuda')
        return seq, s['past'].long()
    at = torch.arange(t, device='cuda', dtype=torch.int32)
    seq = torch.searchsorted(s['cu'], at, right=True) - 1
    return seq, s['past'].long()[seq] + (at - s['cu'][seq]).long()


def _append_plain(s):
    hq, hkv, d = s['hq'], s['hkv'], s['d']
    x = s['qkv'].view(-1, hq + 2 * hkv, d)
    seq, place = _token_places(s)
    cos, sin = _angles(place, s['inv_freq'], s['scale'])
    q = _turn(x[:, :hq].float(), cos, sin, s['interleaved']).to(x.dtype)
    k = _turn(x[:, hq:hq + hkv].float(), cos, sin, s['interleaved']).to(x.dtype)
    page = s['table'][seq, place // s['page']].long()
    s['kc'][page, :, place % s['page']] = k
    s['vc'][page, :, place % s['page']] = x[:, hq + hkv:]
    return dict(q=q, k_cache=s['kc'], v_cache=s['vc'])


def _part(q, k, v, seen):
    """Softmax pieces of q [b, m, d] over k, v [b, l, d] where `seen` [b, m, l] (None: everywhere): the
    maximum, the sum and the weighted values."""
    a = torch.bmm(q, k.transpose(1, 2))
    if seen is not None:
        a = a.masked_fill(~seen, float('-inf'))
    top = a.amax(-1, keepdim=True).clamp(min=-3.0e38)
    e = torch.exp(a - top)
    return top, e.sum(-1, keepdim=True), torch.bmm(e, v)


def _prefix_plain(s):
    q, page, hkv, d = s['q'], s['page'], s['hkv'], s['d']
    t, hq, _ = q.shape
    group, b = hq // hkv, s['batch']
    qs = (q.float() / math.sqrt(d)).view(t, hkv, group, d)
    # the shared part: every query of a key head against one copy of its keys
    n = s['prefix']
    kp = s['kc'][s['common'].long()].transpose(0, 1).reshape(hkv, -1, d)[:, :n].float()
    vp = s['vc'][s['common'].long()].transpose(0, 1).reshape(hkv, -1, d)[:, :n].float()
    m1, l1, o1 = (x.view(hkv, t, group, -1).transpose(0, 1) for x in
                  _part(qs.transpose(0, 1).reshape(hkv, t * group, d), kp, vp, None))
    # the sequences' own parts, padded to the longest
    cu = s['cu'] if s['cu'] is not None else torch.arange(t + 1, device='cuda', dtype=torch.int32)
    count = (cu[1:] - cu[:-1]).long()
    seq = torch.searchsorted(cu, torch.arange(t, device='cuda', dtype=torch.int32), right=True) - 1
    place = torch.arange(t, device='cuda') - cu[seq].long()
    most, longest = s['most'], s['table'].shape[1] * page
    padded = torch.zeros(b, most, hkv, group, d, device='cuda')
    padded[seq, place] = qs
    own_pages = s['table'].clamp(min=0).long()
    ks = s['kc'][own_pages].permute(0, 2, 1, 3, 4).reshape(b * hkv, longest, d).float()
    vs = s['vc'][own_pages].permute(0, 2, 1, 3, 4).reshape(b * hkv, longest, d).float()
    last = s['lens'].long()[:, None] - count[:, None] + torch.arange(most, device='cuda')[None, :]
    seen = torch.arange(longest, device='cuda')[None, None, :] <= last[:, :, None]
    seen = seen[:, None, :, None, :].expand(b, hkv, most, group, longest).reshape(b * hkv, most * group, longest)
    parts = _part(padded.permute(0, 2, 1, 3, 4).reshape(b * hkv, most * group, d), ks, vs, seen)
    m2, l2, o2 = (x.view(b, hkv, most, group, -1).permute(0, 2, 1, 3, 4)[seq, place] for x in parts)
    top = torch.maximum(m1, m2)
    w1, w2 = torch.exp(m1 - top), torch.exp(m2 - top)
    return dict(out=((o1 * w1 + o2 * w2) / (l1 * w1 + l2 * w2)).reshape(t, hq, d).to(q.dtype))


def _sample_plain(s):
    x = s['x'].double()
    rows, vocab = x.shape
    greedy = s['t'] <= 0
    temp = torch.where(greedy, torch.ones_like(s['t']), s['t']).double()[:, None]
    w, at = torch.sort(x, dim=-1, descending=True, stable=True)  # ties: the lowest index first
    w = torch.exp((w - w[:, :1]) / temp)
    col = torch.arange(vocab, device='cuda')[None, :]
    k = torch.where(s['k'] > 0, s['k'], torch.full_like(s['k'], vocab)).long()[:, None]
    w = torch.where(col < torch.where(greedy[:, None], torch.ones_like(k), k), w, torch.zeros_like(w))
    p = s['p'].double()[:, None]
    before = w.cumsum(-1) - w
    kept = (before < p * w.sum(-1, keepdim=True)) | (p >= 1.0) | (col == 0)
    kept &= w >= s['m'].double()[:, None]
    w = torch.zeros_like(w).scatter_(1, at, torch.where(kept, w, torch.zeros_like(w)))  # back in the vocabulary's order
    total = w.sum(-1, keepdim=True)
    ids = (w.cumsum(-1) > s['u'].double()[:, None] * total).int().argmax(-1, keepdim=True)
    return dict(probs=(w.gather(1, ids) / total).float(), ids=ids)


def run(state):
    s = state
    if not own:
        return {'rope': _rope_plain, 'append': _append_plain, 'prefix': _prefix_plain, 'sample': _sample_plain}[s['op']](s)
    import paddle
    import paddle.incubate.nn.functional as IF
    if s['op'] == 'rope':
        q, k = IF.fused_partial_rotary_embedding(s['q'], s['k'], s['inv_freq'], s['pos'], interleaved=s['interleaved'],
                                                 attention_scale=s['scale'])
        dq, dk = torch.autograd.grad([q._t, k._t], [s['q'], s['k']], [s['gq'], s['gk']])
        return dict(q=q._t.detach(), k=k._t.detach(), dq=dq, dk=dk)
    if s['op'] == 'append':
        q, kc, vc = IF.paged_rotary_append(s['qkv'], s['kc'], s['vc'], s['table'], s['past'], cu_seqlens_q=s['cu'],
                                           inv_freq=s['inv_freq'], interleaved=s['interleaved'],
                                           attention_scale=s['scale'])
        return dict(q=q._t, k_cache=kc._t, v_cache=vc._t)
    if s['op'] == 'prefix':
        o = IF.shared_prefix_attention(s['q'], s['kc'], s['vc'], s['table'], s['lens'], prefix_blocks=s['common'],
                                       prefix_len=s['prefix'], cu_seqlens_q=s['cu'], max_seqlen_q=s['most'])
        return dict(out=o._t)
    probs, ids = paddle.filtered_sampling(s['x'], s['u'], temperature=s['t'], top_k=s['k'], top_p=s['p'], min_p=s['m'])
    return dict(probs=probs._t, ids=ids._t)


# ---------------------------------------------------------------------------------- what it takes
def work(case):
    c = case
    z = _SIZE[c['dtype']]
    if c['op'] == 'rope':
        n = c['batch'] * c['seq'] * (c['hq'] + c['hkv']) * c['d']
        return {'bytes': 4 * n * z + 2 * 8 * c['batch'] * c['seq'], 'flops': 6 * n * c['rot'] / c['d']}
    # new tokens and cached ones on average: what prepare() draws
    if c['op'] in ('append', 'prefix'):
        tokens = c['batch'] * (1 + (c['most'] - 1) * 0.5 * 2 / 3)
    if c['op'] == 'append':
        n = tokens * (c['hq'] + 2 * c['hkv']) * c['d']
        return {'bytes': 2 * n * z, 'flops': 3 * tokens * (c['hq'] + c['hkv']) * c['rot']}
    if c['op'] == 'prefix':
        cached = c['prefix'] + c['batch'] * c['tail'] * 2 / 3
        keys = c['prefix'] + c['tail'] * 2 / 3
        return {'bytes': z * (2 * cached * c['hkv'] * c['d'] + 2 * tokens * c['hq'] * c['d']),
                'flops': 4 * tokens * c['hq'] * c['d'] * keys}
    return {'bytes': c['rows'] * (c['vocab'] * z + 32), 'flops': 4 * c['rows'] * c['vocab']}


# ------------------------------------------------------------------------------------ definitions
def _rotation(pos, inv_freq, scale, d, interleaved):
    """The d x d matrices that turn a head at these positions, as their two diagonals and a partner index:
    y = x * c + x[partner] * n."""
    h = inv_freq.numel()
    a = pos.double().unsqueeze(-1) * inv_freq.double()
    c = torch.ones(*pos.shape, d, dtype=torch.float64, device='cuda')
    n = torch.zeros_like(c)
    i = torch.arange(h, device='cuda')
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
    partner = torch.arange(d, device='cuda')
    partner[lo], partner[hi] = hi, lo
    c[..., lo] = c[..., hi] = torch.cos(a) * scale
    n[..., lo], n[..., hi] = -torch.sin(a) * scale, torch.sin(a) * scale
    return c.unsqueeze(-2), n.unsqueeze(-2), partner


def _exact_rope(s):
    c, n, partner = _rotation(s['pos'], s['inv_freq'], s['scale'], s['d'], s['interleaved'])
    ahead = lambda x: x.detach().double() * c + x.detach().double()[..., partner] * n  # noqa: E731
    back = lambda y: y.double() * c + (y.double() * n)[..., partner]  # noqa: E731  # the transposed matrix
    return dict(q=ahead(s['q']), k=ahead(s['k']), dq=back(s['gq']), dk=back(s['gk']))


def _exact_append(s):
    hq, hkv, d, page = s['hq'], s['hkv'], s['d'], s['page']
    kc, vc = s['kc'].double(), s['vc'].double()
    x = s['qkv'].double().view(-1, hq + 2 * hkv, d)
    cu = list(range(s['batch'] + 1)) if s['cu'] is None else s['cu'].tolist()
    q = torch.empty(x.shape[0], hq, d, dtype=torch.float64, device='cuda')
    past, table = s['past'].tolist(), s['table'].long()
    for b in range(s['batch']):
        rows = slice(cu[b], cu[b + 1])
        place = past[b] + torch.arange(cu[b + 1] - cu[b], device='cuda')
        c, n, partner = _rotation(place, s['inv_freq'], s['scale'], d, s['interleaved'])
        y = x[rows, :hq + hkv] * c + x[rows, :hq + hkv][..., partner] * n
        q[rows] = y[:, :hq]
        kc[table[b, place // page], :, place % page] = y[:, hq:]
        vc[table[b, place // page], :, place % page] = x[rows, hq + hkv:]
    return dict(q=q, k_cache=kc, v_cache=vc)


def _exact_prefix(s):
    hkv, d, page, n = s['hkv'], s['d'], s['page'], s['prefix']
    group = s['hq'] // hkv
    out = torch.empty(s['q'].shape, dtype=torch.float64, device='cuda')
    cu = list(range(s['batch'] + 1)) if s['cu'] is None else s['cu'].tolist()
    lens = s['lens'].tolist()
    j = torch.arange(max(n, 1), device='cuda')
    kp, vp = (x[s['common'].long()[j // page], :, j % page][:n].double().permute(1, 0, 2).contiguous()
              for x in (s['kc'], s['vc']))
    for b in range(s['batch']):
        i = torch.arange(lens[b], device='cuda')
        ks, vs = (x[s['table'].long()[b, i // page], :, i % page].double().permute(1, 0, 2) for x in (s['kc'], s['vc']))
        new = cu[b + 1] - cu[b]
        q = s['q'][cu[b]:cu[b + 1]].double().view(new, hkv, group, d).permute(1, 0, 2, 3).reshape(hkv, new * group, d)
        a1 = torch.bmm(q, kp.transpose(1, 2).contiguous()) / math.sqrt(d)
        a2 = torch.bmm(q, ks.transpose(1, 2).contiguous()) / math.sqrt(d)
        later = i[None, :] > (lens[b] - new + torch.arange(new, device='cuda'))[:, None]
        a2 = a2.masked_fill(later.repeat_interleave(group, 0)[None], float('-inf'))
        w = torch.softmax(torch.cat([a1, a2], -1), -1)
        o = torch.bmm(w[..., :n].contiguous(), vp) + torch.bmm(w[..., n:].contiguous(), vs.contiguous())
        out[cu[b]:cu[b + 1]] = o.view(hkv, new, group, d).permute(1, 0, 2, 3).reshape(new, hkv * group, d)
    return dict(out=out)


def _exact_sample(s):
    probs = torch.empty(s['rows'], 1, dtype=torch.float64, device='cuda')
    ids = torch.empty(s['rows'], 1, dtype=torch.int64, device='cuda')
    for r in range(s['rows']):
        x = s['x'][r].double()
        t, k, p, m = float(s['t'][r]), int(s['k'][r]), float(s['p'][r]), float(s['m'][r])
        if t <= 0:
            ids[r, 0] = (x == x.max()).nonzero()[0, 0]
            probs[r, 0] = 1.0
            continue
        w = torch.softmax(x / t, 0)
        by_weight = torch.argsort(x, descending=True, stable=True)
        if k > 0:
            by_weight = by_weight[:k]
        if p < 1.0:
            c = w[by_weight].cumsum(0)
            # as many as it takes to reach the share p, at least one
            by_weight = by_weight[:1 + int((c[:-1] < p * c[-1]).sum())]
        by_weight = by_weight[w[by_weight] >= m * w.max()]
        chosen = by_weight.sort().values
        c = w[chosen].cumsum(0)
        at = min(int((c <= float(s['u'][r]) * c[-1]).sum()), chosen.numel() - 1)
        ids[r, 0] = chosen[at]
        probs[r, 0] = w[chosen[at]] / c[-1]
    return dict(probs=probs, ids=ids)


def exact(case, seed):
    s = prepare(case, seed)
    return {'rope': _exact_rope, 'append': _exact_append, 'prefix': _exact_prefix, 'sample': _exact_sample}[s['op']](s)
