"""The serving operators of the temporal head, as they are measured: what each case stands for, its inputs, a plain form in elementary torch
operations, the calls a user makes of the framework (``own = True``), the bytes and operations a pass cannot do without, and the definition in 64 bits.

Four operators serve many live clips ("streams") of different lengths from one key / value cache that is cut into pages:
  plan   the cache's block tables and the slots of the new tokens, from the streams' lengths
  write  the new tokens' keys and values into their slots
  attn   causal attention of each stream's new tokens over its pages
  w4     a linear layer of few rows on 4-bit weights with group scales
"""
import math

import torch

own = False

BF16 = torch.bfloat16
I32 = torch.int32


# ---- cases -------------------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # three clips roll one frame further: the smallest step of the head, all latency
        {'name': 'plan_roll_3', 'op': 'plan', 'streams': 3, 'new_max': 1, 'past_max': 14, 'page': 16},
        # a full server takes a burst of chunks of every length
        {'name': 'plan_burst_2000', 'op': 'plan', 'streams': 2000, 'new_max': 64, 'past_max': 4000, 'page': 32},
        # one new frame of 64 streams, keys and values inside the head's fused projection (4 heads of 512)
        {'name': 'write_64x4x512', 'op': 'write', 'tokens': 64, 'kv_heads': 4, 'hd': 512, 'page': 16},
        # a burst of chunks with shared key heads
        {'name': 'write_8191x8x128', 'op': 'write', 'tokens': 8191, 'kv_heads': 8, 'hd': 128, 'page': 32},
        # the head's roll-out at three clips of 10 to 15 frames
        {'name': 'attn_roll_3', 'op': 'attn', 'streams': 3, 'new_max': 1, 'past_max': 14, 'heads': 4, 'kv_heads': 4, 'hd': 512, 'page': 16},
        # 64 streams up to the head's 1024 positions, one frame each
        {'name': 'attn_decode_64x4x512', 'op': 'attn', 'streams': 64, 'new_max': 1, 'past_max': 1023, 'heads': 4, 'kv_heads': 4, 'hd': 512, 'page': 16},
        # long streams, shared key heads, one token each: the cache's bytes are the work
        {'name': 'attn_decode_long', 'op': 'attn', 'streams': 60, 'new_max': 1, 'past_max': 9000, 'heads': 32, 'kv_heads': 8, 'hd': 128, 'page': 32},
        # clips enter: chunks of up to 192 frames on top of what is cached
        {'name': 'attn_chunk_16x4x512', 'op': 'attn', 'streams': 16, 'new_max': 192, 'past_max': 800, 'heads': 4, 'kv_heads': 4, 'hd': 512, 'page': 16},
        # two long chunks behind a long past: matrix-bound
        {'name': 'attn_chunk_long', 'op': 'attn', 'streams': 2, 'new_max': 4099, 'past_max': 4200, 'heads': 16, 'kv_heads': 4, 'hd': 128, 'page': 64},
        # the head's output projection for one token
        {'name': 'w4_1x2048x2048', 'op': 'w4', 'm': 1, 'n': 2048, 'k': 2048, 'group': 128, 'bias': True, 'gelu': False, 'res': True},
        # the head's second feed-forward product for three clips
        {'name': 'w4_3x2048x8192', 'op': 'w4', 'm': 3, 'n': 2048, 'k': 8192, 'group': 64, 'bias': True, 'gelu': False, 'res': True},
        # a wide layer for a batch of streams
        {'name': 'w4_33x16384x8192', 'op': 'w4', 'm': 33, 'n': 16384, 'k': 8192, 'group': 128, 'bias': True, 'gelu': True, 'res': False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['plan', 'write', 'attn', 'attn', 'attn', 'attn', 'w4', 'w4'])
    if op == 'plan':
        s = _log(rng, 1, 2000)
        return {'op': op, 'streams': s, 'new_max': _log(rng, 1, max(1, min(512, 120000 // s))), 'past_max': _log(rng, 1, 4000), 'page': rng.choice([16, 32, 64, 128])}
    if op == 'write':
        hd, kvh = rng.choice([64, 128, 256, 512]), rng.choice([1, 2, 4, 8])
        return {'op': op, 'tokens': _log(rng, 1, 8 * 1024 * 1024 // (hd * kvh)), 'kv_heads': kvh, 'hd': hd, 'page': rng.choice([16, 32, 64, 128])}
    if op == 'w4':
        g = rng.choice([32, 64, 128])
        return {'op': op, 'm': _log(rng, 1, 64), 'n': _log(rng, 100, 16000), 'k': g * _log(rng, 2, 8192 // g), 'group': g, 'bias': rng.random() < 0.7,
                'gelu': rng.random() < 0.3, 'res': rng.random() < 0.3}
    hd = rng.choice([64, 64, 128, 128, 256, 512])
    kvh = rng.choice([1, 2, 4, 8])
    heads = kvh * rng.choice([1, 1, 2, 4, 8])
    new = 1 if rng.random() < 0.4 else _log(rng, 2, 2000)
    past = _log(rng, 8, 8000)
    # keep the cache under 0.6 GB and the scores' work under the largest listed case's
    most = min(0.6e9 / (4.0 * kvh * hd * (new + past)), 5e10 / (1.0 * heads * hd * new * (new + past)), 30000.0 / new, 200.0)
    return {'op': op, 'streams': _log(rng, 1, max(1, int(most))), 'new_max': new, 'past_max': past, 'heads': heads, 'kv_heads': kvh, 'hd': hd,
            'page': rng.choice([16, 32, 64, 128])}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """(new, past) of every stream as host lists: ragged, the first one at the case's largest.  The same for every seed, so that a case is the same work."""
    g = torch.Generator().manual_seed(1000003 * case['streams'] + 101 * case['new_max'] + case['past_max'])
    s = case['streams']
    new = torch.randint(max(1, (case['new_max'] + 1) // 2), case['new_max'] + 1, (s,), generator=g)
    past = torch.randint(max(0, case['past_max'] // 4), case['past_max'] + 1, (s,), generator=g)
    new[0], past[0] = case['new_max'], case['past_max']
    return new.tolist(), past.tolist()


def _pages(n, page):
    return (n + page - 1) // page


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device='cuda', dtype=torch.float32)


def _bf16_randn(g, *shape):
    """Normal values in bf16, made in slices so that a large cache does not pass through a float copy of its size."""
    out = torch.empty(shape, device='cuda', dtype=BF16)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 26):
        n = min(1 << 26, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device='cuda', dtype=torch.float32)
    return out


def _table(lists, width, pages, g):
    """Every stream's pages drawn from a shuffled pool, as a table of `width` columns (unused entries 0)."""
    perm = torch.randperm(pages, generator=g, device='cuda').to(I32)
    flat, at = torch.zeros((len(lists), width), device='cuda', dtype=I32), 0
    col = torch.arange(width, device='cuda')[None, :]
    owned = torch.tensor(lists, device='cuda')[:, None]
    mask = col < owned
    n = int(sum(lists))
    flat[mask] = perm[at:at + n]
    return flat, perm[n:]


def prepare(case, seed):
    g = _gen(seed)
    st = {'case': case}
    if case['op'] == 'plan':
        new, past = _lengths(case)
        page, width = case['page'], _pages(case['past_max'] + case['new_max'], case['page'])
        have = [_pages(p, page) for p in past]
        need = sum(_pages(p + n, page) - h for p, n, h in zip(past, new, have))
        st['table'], free = _table(have, width, sum(have) + need + 7, g)
        st.update(lens=torch.tensor(past, device='cuda', dtype=I32), new=torch.tensor(new, device='cuda', dtype=I32), owned=torch.tensor(have, device='cuda', dtype=I32),
                  free=free, n_free=torch.tensor([free.numel()], device='cuda', dtype=I32), tokens=sum(new))
    elif case['op'] == 'write':
        t, w = case['tokens'], case['kv_heads'] * case['hd']
        qkv = _bf16_randn(g, t, 3 * w)                              # the fused projection's rows: q | k | v
        pages = _pages(t, case['page']) * 2
        st['k'], st['v'] = (qkv[:, i * w:(i + 1) * w].view(t, case['kv_heads'], case['hd']) for i in (1, 2))
        st['kc'], st['vc'] = (_bf16_randn(g, pages, case['page'], case['kv_heads'], case['hd']) for _ in range(2))
        st['slots'] = torch.randperm(pages * case['page'], generator=g, device='cuda')[:t].to(I32)
    elif case['op'] == 'attn':
        new, past = _lengths(case)
        page, kv = case['page'], [n + p for n, p in zip(new, past)]
        have = [_pages(x, page) for x in kv]
        pages = sum(have) + 3
        st['table'], _ = _table(have, max(have), pages, g)
        st['kc'], st['vc'] = (_bf16_randn(g, pages, page, case['kv_heads'], case['hd']) for _ in range(2))
        st['q'] = _bf16_randn(g, sum(new), case['heads'], case['hd'])
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        st.update(new=new, kv=kv, host_cu=cu, cu=torch.tensor(cu, device='cuda', dtype=I32), kv_lens=torch.tensor(kv, device='cuda', dtype=I32))
    else:
        m, n, k, grp = case['m'], case['n'], case['k'], case['group']
        st['x'] = _bf16_randn(g, m, k)
        st['q'] = torch.randint(0, 256, (n, k // 2), generator=g, device='cuda', dtype=torch.uint8)
        st['s'] = ((0.5 + torch.rand((n, k // grp), generator=g, device='cuda')) * (0.2 / math.sqrt(k))).to(BF16)
        st['bias'] = _randn(g, n) if case['bias'] else None
        st['res'] = _bf16_randn(g, m, n) if case['res'] else None
    return st


# ---- one pass ----------------------------------------------------------------------------------------------------------------------------------
def run(st):
    return {'plan': _plan, 'write': _write, 'attn': _attn, 'w4': _w4}[st['case']['op']](st)


def _plan(st):
    page = st['case']['page']
    if own:
        from avt_amd import ops
        p = ops.paged_plan(st['lens'], st['new'], st['owned'], st['table'], st['free'], st['n_free'], page, st['tokens'])
        return [p.cu, p.kv_lens, p.owned, p.n_free, p.slots, p.positions, p.streams, st['table']]
    lens, new, owned, table, free = st['lens'].long(), st['new'].long(), st['owned'].long(), st['table'], st['free']
    width = table.size(1)
    cu = torch.cat([torch.zeros(1, device='cuda', dtype=torch.long), new.cumsum(0)])
    total = lens + new
    pages = (total + page - 1) // page
    fits = pages <= width
    need = torch.where(fits, (pages - owned).clamp(min=0), 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= st['n_free']))
    kv = torch.where(granted, total, 0)
    owned_out = torch.where(granted, torch.maximum(owned, pages), owned)
    n_free = st['n_free'] - torch.where(granted, need, 0).sum()
    col = torch.arange(width, device='cuda')[None, :]
    j = col - owned[:, None]
    fresh = granted[:, None] & (j >= 0) & (j < need[:, None])
    at = (st['n_free'] - 1 - (upto - need)[:, None] - j).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[at], table))
    t = torch.arange(st['tokens'], device='cuda')
    stream = torch.searchsorted(cu, t, right=True) - 1
    pos = lens[stream] + t - cu[stream]
    slot = table[stream, (pos // page).clamp(max=width - 1)] * page + pos % page
    slot = torch.where(granted[stream], slot, -1)
    return [cu.to(I32), kv.to(I32), owned_out.to(I32), n_free.to(I32), slot.to(I32), pos.to(I32), stream.to(I32), table]


def _write(st):
    kc, vc = st['kc'], st['vc']
    if own:
        from avt_amd import ops
        ops.paged_kv_write(st['k'], st['v'], kc, vc, st['slots'])
    else:
        at = st['slots'].long()
        kc.view(-1, *kc.shape[2:])[at] = st['k']
        vc.view(-1, *vc.shape[2:])[at] = st['v']
    return [kc, vc]


def _attn(st):
    c = st['case']
    if own:
        from avt_amd import ops
        return ops.paged_attn(st['q'], st['kc'], st['vc'], st['table'], st['cu'], st['kv_lens'], max_new=max(st['new']), max_kv=max(st['kv']))
    return _attn_in(st, torch.float32, c['heads']).to(BF16)


def _attn_in(st, dtype, heads_at_once):
    """softmax(scale q k^T) v of every stream, causal, in `dtype`; some heads at a time."""
    c = st['case']
    grp, hd, page = c['heads'] // c['kv_heads'], c['hd'], c['page']
    out = torch.zeros(st['q'].size(0), c['heads'], hd, device='cuda', dtype=dtype)
    kvs = max(1, min(c['kv_heads'], heads_at_once // grp))
    for r, (n, kv) in enumerate(zip(st['new'], st['kv'])):
        lo = st['host_cu'][r]
        ids = st['table'][r, :_pages(kv, page)].long()
        hidden = torch.arange(kv, device='cuda')[None, :] > torch.arange(kv - n, kv, device='cuda')[:, None]
        for h in range(0, c['kv_heads'], kvs):
            k, v = (x[ids, :, h:h + kvs].reshape(-1, kvs, hd)[:kv].to(dtype).transpose(0, 1).contiguous() for x in (st['kc'], st['vc']))      # [kvs, kv, hd]
            q = st['q'][lo:lo + n, h * grp:(h + kvs) * grp].to(dtype).view(n, kvs, grp, hd).permute(1, 2, 0, 3).reshape(kvs, grp * n, hd)
            s = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(hd ** -0.5).view(kvs, grp, n, kv)
            s.masked_fill_(hidden, -math.inf)
            p = s.sub_(s.amax(-1, keepdim=True)).exp_()
            den = p.sum(-1, keepdim=True)
            o = torch.matmul(p.view(kvs, grp * n, kv), v).view(kvs, grp, n, hd) / den
            out[lo:lo + n, h * grp:(h + kvs) * grp] = o.permute(2, 0, 1, 3).reshape(n, kvs * grp, hd)
    return out.view(st['q'].size(0), c['heads'] * hd)


def _w4(st):
    c = st['case']
    if own:
        from avt_amd import ops
        return ops.w4_linear(st['x'], ops.W4Weight(st['q'], st['s']), bias=st['bias'], act=ops.ACT_GELU_TANH if c['gelu'] else ops.ACT_NONE, res=st['res'])
    n, k = c['n'], c['k']
    u = torch.stack([st['q'] & 15, st['q'] >> 4], dim=-1).view(n, k)
    w = ((u.float() - 8.0).view(n, -1, c['group']) * st['s'].float()[:, :, None]).view(n, k)
    y = torch.matmul(st['x'].float(), w.t())
    if c['bias']:
        y = y + st['bias']
    if c['gelu']:
        y = 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    if c['res']:
        y = y + st['res'].float()
    return y.to(BF16)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------------------
def work(case):
    if case['op'] == 'plan':
        new, past = _lengths(case)
        grown = sum(_pages(p + n, case['page']) - _pages(p, case['page']) for p, n in zip(past, new))
        return {'bytes': 4.0 * (3 * len(new) + grown + len(new)) + 4.0 * (3 * len(new) + 3 * sum(new) + grown), 'flops': 0.0}
    if case['op'] == 'write':
        return {'bytes': 2.0 * 4 * case['tokens'] * case['kv_heads'] * case['hd'] + 4.0 * case['tokens'], 'flops': 0.0}
    if case['op'] == 'attn':
        new, past = _lengths(case)
        seen = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
        rows = 2.0 * 2 * sum(new) * case['heads'] * case['hd']
        return {'bytes': rows + 2.0 * 2 * sum(n + p for n, p in zip(new, past)) * case['kv_heads'] * case['hd'], 'flops': 4.0 * case['hd'] * case['heads'] * seen}
    m, n, k = case['m'], case['n'], case['k']
    return {'bytes': n * k / 2.0 + 2.0 * n * k / case['group'] + 2.0 * m * k + 2.0 * m * n * (2 if case['res'] else 1) + (4.0 * n if case['bias'] else 0.0), 'flops': 2.0 * m * n * k}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case['op'] == 'plan':
        return None                                                 # whole numbers
    st = prepare(case, seed)
    f = torch.float64
    if case['op'] == 'write':
        at, both = st['slots'].long(), []
        for new, old in ((st['k'], st['kc']), (st['v'], st['vc'])):
            cache = old.to(f).flatten(0, 1)
            cache.index_copy_(0, at, new.to(f))
            both.append(cache.view(old.shape))
        return both
    if case['op'] == 'w4':
        out = torch.empty(case['m'], case['n'], device='cuda', dtype=f)
        x = st['x'].to(f)
        for lo in range(0, case['n'], 2048):
            b = st['q'][lo:lo + 2048].long()
            w = torch.empty(b.size(0), case['k'], device='cuda', dtype=f)
            w[:, 0::2], w[:, 1::2] = (b % 16 - 8).to(f), (b // 16 - 8).to(f)
            w *= st['s'][lo:lo + 2048].to(f).repeat_interleave(case['group'], dim=1)
            out[:, lo:lo + 2048] = x @ w.T
        if case['bias']:
            out += st['bias'].to(f)
        if case['gelu']:
            out = out * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (out + 0.044715 * out ** 3)))
        if case['res']:
            out += st['res'].to(f)
        return out
    grp, hd, page = case['heads'] // case['kv_heads'], case['hd'], case['page']
    out = torch.zeros(st['q'].size(0), case['heads'], hd, device='cuda', dtype=f)
    for r, (n, kv) in enumerate(zip(st['new'], st['kv'])):
        lo, tok = st['host_cu'][r], torch.arange(kv, device='cuda')
        page_of, row = st['table'][r].long()[tok // page], tok % page
        for h in range(case['kv_heads']):
            k, v = st['kc'][page_of, row, h].to(f), st['vc'][page_of, row, h].to(f)
            for i in range(0, n, 1024):
                m = min(1024, n - i)
                q = st['q'][lo + i:lo + i + m, h * grp:(h + 1) * grp].to(f).reshape(m * grp, hd)
                w = ((q @ k.T) / math.sqrt(hd)).view(m, grp, kv)
                last = kv - n + i + torch.arange(m, device='cuda')
                w = torch.where(tok[None, None, :] <= last[:, None, None], w, torch.full((), -math.inf, device='cuda', dtype=f))
                out[lo + i:lo + i + m, h * grp:(h + 1) * grp] = (torch.softmax(w, dim=-1).view(m * grp, kv) @ v).view(m, grp, hd)
    return out.view(st['q'].size(0), case['heads'] * hd)
