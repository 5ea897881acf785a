"""The paged key/value cache operators as a user's program calls them: `kv_append` (write new frames' keys and values,
quantising them), `kv_read` (gather them back) and `paged_attention` (new tokens over everything cached).

Where the sizes come from: the relation head's temporal encoder has 4 heads of 128 over up to 100 (subject, object) pairs and
a positional table of 5000 frames, crops videos to 900 frames, and the object encoders and the mask decoder have 8 heads of
32; clips come in 1 to 32 frames.  The grouped-head and 65536-long cases are generic.

A case says: `op`; `seqs` sequences, the last `idle` of them empty; `new` tokens of each; `longest` cached positions
(`ragged`: lengths spread from one up to it); heads, head size and page size; the types of the pool (`cache`) and of the
queries / new rows / result (`rows`); `padded`: a key padding mask that blocks 3 frames in 10, and all frames of one sequence.
"""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16, 'e4m3': torch.float8_e4m3fn, 'i8': torch.int8}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2, 'e4m3': 1, 'i8': 1}
CODES = {'e4m3': 448.0, 'i8': 127.0}
TINY = 2.0 ** -126


def _case(op, name=None, seqs=1, new=1, q_heads=4, kv_heads=4, dim=128, page=16, longest=64, ragged=False, idle=0, cache='f32',
          rows='f32', padded=False, causal=True):
    c = dict(op=op, seqs=seqs, new=new, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, longest=longest, ragged=ragged,
             idle=idle, cache=cache, rows=rows, padded=padded, causal=causal)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one tracked pair, one new frame, two seconds of history: what a live relation query waits for
        _case('attend', 'attend-pair-60-f32', longest=60),
        # all 100 pairs of a video, one new frame, histories up to the 900-frame crop, tubes absent in some frames
        _case('attend', 'attend-pairs-900-f32-padded', seqs=100, longest=900, ragged=True, padded=True),
        # a 32-frame clip appended to histories as long as the positional table, 8-bit pool
        _case('attend', 'attend-pairs-5000-clip32-e4m3', seqs=100, new=32, longest=5000, ragged=True, cache='e4m3', rows='bf16'),
        # heads of 32, a 4-frame clip whose frames see each other (bidirectional encoder), f32 rows over a bf16 pool
        _case('attend', 'attend-objects-301-clip4-bf16', seqs=25, new=4, q_heads=8, kv_heads=8, dim=32, page=8, longest=301,
              ragged=True, cache='bf16', rows='f32', causal=False),
        # shared key heads, few sequences, a very long cache: nothing but the split over its length fills the card
        _case('attend', 'attend-long-65536-gqa4-bf16', seqs=8, q_heads=32, kv_heads=8, page=64, longest=65536, cache='bf16', rows='bf16'),
        # many sequences of shared heads over an integer pool, one slot of the batch idle
        _case('attend', 'attend-gqa8-4095-i8', seqs=33, q_heads=16, kv_heads=2, dim=64, page=32, longest=4095, ragged=True, idle=1,
              cache='i8', rows='f16'),
        # one new frame of 100 pairs written to a 16-bit pool: the latency of the write
        _case('append', 'append-pairs-1-bf16', seqs=100, longest=900, ragged=True, cache='bf16'),
        # a 32-frame clip of 100 pairs, quantised
        _case('append', 'append-pairs-clip32-e4m3', seqs=100, new=32, longest=901, ragged=True, cache='e4m3'),
        # whole histories entering an integer pool
        _case('append', 'append-prompt-4096-i8', seqs=16, new=4096, q_heads=8, kv_heads=8, page=64, longest=4096, cache='i8', rows='bf16'),
        # a short history back from an 8-bit pool
        _case('read', 'read-129-e4m3', seqs=3, longest=129, ragged=True, cache='e4m3', rows='bf16'),
        # the whole video's keys and values back in f32, for the bidirectional pass at its end
        _case('read', 'read-pairs-900-bf16', seqs=100, longest=900, ragged=True, cache='bf16'),
        # the loop of a live video: a frame is appended, then attended from
        _case('step', 'step-pairs-900-e4m3', seqs=100, longest=900, ragged=True, cache='e4m3'),
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    op = rng.choice(('attend', 'attend', 'attend', 'append', 'read', 'step'))
    cache, rows = rng.choice((('f32', 'f32'), ('bf16', 'f32'), ('f16', 'f32'), ('e4m3', 'f32'), ('i8', 'f32'), ('bf16', 'bf16'),
                              ('e4m3', 'bf16'), ('i8', 'bf16'), ('f16', 'f16'), ('e4m3', 'f16'), ('i8', 'f16')))
    kv_heads = rng.choice((1, 2, 4, 8))
    c = _case(op, seqs=_log(rng, 1, 128), new=1 if rng.random() < 0.5 else _log(rng, 2, 32), kv_heads=kv_heads,
              q_heads=kv_heads * rng.choice((1, 1, 2, 3, 4, 8)), dim=rng.choice((32, 64, 80, 96, 128, 128, 256)),
              page=rng.choice((8, 16, 32, 64, 256)), longest=_log(rng, 1, 16384), ragged=rng.random() < 0.7, cache=cache, rows=rows,
              padded=rng.random() < 0.3, causal=rng.random() < 0.8)
    while c['seqs'] * c['kv_heads'] * c['dim'] * c['longest'] * BYTES[cache] > 5e8 or c['seqs'] * c['q_heads'] * c['new'] * c['longest'] > 1e8:
        c['longest'] = c['longest'] // 2 + 1
        c['seqs'] = max(1, c['seqs'] * 3 // 4)
    c['idle'] = rng.randint(0, 2) if c['seqs'] > 4 else 0
    return c


def _lengths(c):
    """cached positions of each sequence, this call's new ones among them: of the case alone, the seed shuffles them"""
    live = c['seqs'] - c['idle']
    golden = 0.6180339887498949
    n = [c['longest'] if b == 0 or not c['ragged'] else 1 + int((c['longest'] - 1) * (b * golden % 1.0)) for b in range(live)]
    return n + [0] * c['idle']


def _new(c, n):
    return min(c['new'], n)


def prepare(case, seed):
    c = case
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)
    S, H, D, B, T = c['page'], c['kv_heads'], c['dim'], c['seqs'], c['new']
    lens = torch.tensor(_lengths(c), dtype=torch.int32)
    order = torch.randperm(B - c['idle'], generator=torch.Generator().manual_seed(seed))
    lens[:B - c['idle']] = lens[order]
    lens = lens.to(dev)
    width = -(-c['longest'] // S)
    pool = B * width + 3
    pages = torch.randperm(pool, generator=g, device=dev)
    table = pages[:B * width].view(B, width).to(torch.int32)
    shape = (pool, H, S, D)

    def filled():
        """a pool as it stands in the middle of a run: every slot has been written before"""
        if c['cache'] == 'i8':
            return torch.randint(-127, 128, shape, generator=g, device=dev, dtype=torch.int8)
        x = torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16 if c['cache'] == 'e4m3' else TYPES[c['cache']])
        return (x * 100.0).clamp_(-448, 448).to(TYPES['e4m3']) if c['cache'] == 'e4m3' else x

    s = dict(case=c, table=table, spare=pages[-1], lens=lens, new_lens=lens.clamp(max=T), k=filled(), v=filled(), k_scale=None, v_scale=None)
    if c['cache'] in CODES:
        unit = 1.0 / 100.0 if c['cache'] == 'e4m3' else 1.0 / 73.0
        for n in ('k_scale', 'v_scale'):
            s[n] = (0.5 + torch.rand(shape[:3], generator=g, device=dev)) * unit
    rows = TYPES[c['rows']]
    if c['op'] in ('attend', 'step'):
        s['q'] = torch.randn((B, T, c['q_heads'], D), generator=g, device=dev).to(rows)
        s['padding'] = None
        if c['padded']:
            s['padding'] = torch.rand((B, c['longest']), generator=g, device=dev) < 0.3
            s['padding'][B // 2] = True
    if c['op'] in ('append', 'step'):
        # the new keys and values are column blocks of one projection's output, as the encoder layer makes them
        kv = torch.randn((B, T, 2, H, D), generator=g, device=dev).to(rows)
        s['new_k'], s['new_v'] = kv[:, :, 0], kv[:, :, 1]
    if own:
        from openpvsg_amd import ops
        s['pages'] = ops.KVPages(s['k'], s['v'], s['k_scale'], s['v_scale'])
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------
def _plain_store(codes, scales, x, live, page, slot, spare, cache):
    """rows x (B, T, H, D) to their slots; where there is no row to write, slot 0 of a page that nobody has keeps what it holds"""
    x = x.float()
    if cache in CODES:
        scale = (x.abs().amax(-1) * (1.0 / CODES[cache])).clamp_min(TINY)
        scales[page, :, slot] = torch.where(live[..., None], scale, scales[spare, :, 0])
        x = x / scale[..., None]
        if cache == 'i8':
            x = x.round()
    x = x.to(codes.dtype)
    if cache == 'e4m3':
        codes, x = codes.view(torch.uint8), x.view(torch.uint8)
    codes[page, :, slot] = torch.where(live[..., None, None], x, codes[spare, :, 0])


def _plain_append(s):
    c = s['case']
    t = torch.arange(c['new'], device=s['lens'].device)
    live = t[None, :] < s['new_lens'][:, None]
    at = ((s['lens'] - s['new_lens'])[:, None] + t[None, :]).clamp(max=s['table'].shape[1] * c['page'] - 1)
    page = torch.where(live, s['table'].long().gather(1, at // c['page']), s['spare'])
    slot = torch.where(live, at % c['page'], 0)
    _plain_store(s['k'], s['k_scale'], s['new_k'], live, page, slot, s['spare'], c['cache'])
    _plain_store(s['v'], s['v_scale'], s['new_v'], live, page, slot, s['spare'], c['cache'])


def _plain_gather(codes, scales, table):
    """(B, H, positions, D) in f32"""
    B, W = table.shape
    x = codes[table.long()].float() if codes.dtype != torch.float8_e4m3fn else codes.view(torch.uint8)[table.long()].view(codes.dtype).float()
    if scales is not None:
        x = x * scales[table.long()][..., None]
    return x.transpose(1, 2).reshape(B, x.shape[2], -1, x.shape[-1])


def _plain_read(s):
    c = s['case']
    there = torch.arange(c['longest'], device=s['lens'].device)[None, :] < s['lens'][:, None]
    out = []
    for codes, scales in ((s['k'], s['k_scale']), (s['v'], s['v_scale'])):
        x = _plain_gather(codes, scales, s['table'])[:, :, :c['longest']].transpose(1, 2)
        out.append(torch.where(there[:, :, None, None], x, 0.0).to(TYPES[c['rows']]))
    return out


def _plain_attend(s):
    c = s['case']
    B, T, HQ, D = s['q'].shape
    H, L = c['kv_heads'], c['longest']
    G = HQ // H
    k = _plain_gather(s['k'], s['k_scale'], s['table'])[:, :, :L]
    v = _plain_gather(s['v'], s['v_scale'], s['table'])[:, :, :L]
    p = torch.arange(L, device=k.device)
    t = torch.arange(T, device=k.device)
    there = p[None, :] < s['lens'][:, None]
    if s['padding'] is not None:
        there = there & ~s['padding']
    seen = there[:, None, :] & (t[None, :, None] < s['new_lens'][:, None, None])
    if c['causal']:
        seen = seen & (p[None, None, :] <= (s['lens'] - s['new_lens'])[:, None, None] + t[None, :, None])
    k = torch.where(there[:, None, :, None], k, 0.0)
    v = torch.where(there[:, None, :, None], v, 0.0)
    q = s['q'].float().view(B, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, D)
    z = (q @ k.transpose(2, 3).contiguous()).view(B, H, T, G, L) * (1.0 / math.sqrt(D))
    z = torch.where(seen[:, None, :, None, :], z, -math.inf)
    m = z.amax(-1, keepdim=True)
    w = torch.exp(z - torch.where(m == -math.inf, 0.0, m))
    total = w.sum(-1, keepdim=True)
    o = (w.view(B, H, T * G, L) @ v).view(B, H, T, G, D)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 2, 1, 3, 4).reshape(B, T, HQ, D).to(s['q'].dtype)


def _plain(s):
    op = s['case']['op']
    if op == 'attend':
        return _plain_attend(s)
    if op == 'read':
        return _plain_read(s)
    _plain_append(s)
    return _written(s) if op == 'append' else [_plain_attend(s)] + _written(s)


# ---- the framework's ----------------------------------------------------------------------------------------------------------
def _written(s):
    return [x for x in (s['k'], s['v'], s['k_scale'], s['v_scale']) if x is not None]


def _own(s):
    from openpvsg_amd import ops
    c, op = s['case'], s['case']['op']
    if op == 'read':
        return list(ops.kv_read(s['pages'], s['table'], s['lens'], c['longest'], dtype=TYPES[c['rows']]))
    if op in ('append', 'step'):
        ops.kv_append(s['pages'], s['new_k'], s['new_v'], s['table'], s['lens'], new_lens=s['new_lens'])
        if op == 'append':
            return _written(s)
    o = ops.paged_attention(s['q'], s['pages'], s['table'], s['lens'], new_lens=s['new_lens'], key_padding_mask=s['padding'], causal=c['causal'])
    return o if op == 'attend' else [o] + _written(s)


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------
def work(case):
    c = case
    n = _lengths(c)
    row = c['kv_heads'] * (c['dim'] * BYTES[c['cache']] + (4 if c['cache'] in CODES else 0)) * 2
    plain_row = c['kv_heads'] * c['dim'] * BYTES[c['rows']] * 2
    fresh = sum(_new(c, x) for x in n)
    byte = flop = 0
    if c['op'] in ('append', 'step'):
        byte += fresh * (row + plain_row)
        flop += fresh * c['kv_heads'] * c['dim'] * 2 * 3
    if c['op'] == 'read':
        byte += sum(n) * row + c['seqs'] * c['longest'] * plain_row
        flop += sum(n) * c['kv_heads'] * c['dim'] * 2
    if c['op'] in ('attend', 'step'):
        byte += sum(n) * row + 2 * c['seqs'] * c['new'] * c['q_heads'] * c['dim'] * BYTES[c['rows']]
        byte += c['seqs'] * c['longest'] if c['padded'] else 0
        pairs = 0
        for x in n:
            t = _new(c, x)
            pairs += t * x - (t * (t - 1) // 2 if c['causal'] else 0)
        flop += 4 * pairs * c['q_heads'] * c['dim']
    return {'bytes': byte, 'flops': flop}


# ---- 64 bits, a sequence at a time ----------------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    lens, fresh, table = s['lens'].tolist(), s['new_lens'].tolist(), s['table'].long()
    full = {}
    for n in ('k', 'v'):
        x = s[n].double()
        full[n] = x * s[n + '_scale'].double()[..., None] if s[n + '_scale'] is not None else x
    kept = {n: (s[n].double() if c['cache'] != 'i8' else None) for n in ('k', 'v')}
    scales = {n: (s[n + '_scale'].double() if s[n + '_scale'] is not None else None) for n in ('k', 'v')}
    if c['op'] in ('append', 'step'):
        for b in range(c['seqs']):
            if not fresh[b]:
                continue
            p = torch.arange(lens[b] - fresh[b], lens[b], device=table.device)
            page, slot = table[b, torch.div(p, c['page'], rounding_mode='floor')], p % c['page']
            for n in ('k', 'v'):
                x = s['new_' + n][b, :fresh[b]].double()
                unit = None
                if scales[n] is not None:
                    unit = torch.clamp(x.abs().max(dim=-1).values / CODES[c['cache']], min=TINY)
                    scales[n][page, :, slot] = unit
                code = x if unit is None else x / unit[..., None]
                if kept[n] is not None:
                    kept[n][page, :, slot] = code
                if unit is None:
                    full[n][page, :, slot] = code.to(TYPES[c['cache']]).double()
    state = [kept['k'], kept['v']] + ([scales['k'], scales['v']] if scales['k'] is not None else [])
    if c['op'] == 'append':
        return state
    if c['op'] == 'read':
        out = []
        for n in ('k', 'v'):
            y = torch.zeros((c['seqs'], c['longest'], c['kv_heads'], c['dim']), dtype=torch.float64, device=table.device)
            for b in range(c['seqs']):
                p = torch.arange(lens[b], device=table.device)
                y[b, :lens[b]] = full[n][table[b, torch.div(p, c['page'], rounding_mode='floor')], :, p % c['page']]
            out.append(y)
        return out
    if c['op'] == 'step' and c['cache'] in CODES:
        # what is attended to is the new rows' codes; where x / s falls next to a border between two codes, 32 and 64 bits
        # pick different ones, so the result has no one value in 64 bits
        return [None] + state
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device=table.device)
    group = c['q_heads'] // c['kv_heads']
    for b in range(c['seqs']):
        n = lens[b]
        if not n:
            continue
        p = torch.arange(n, device=table.device)
        hide = s['padding'][b, :n] if s['padding'] is not None else torch.zeros(n, dtype=torch.bool, device=table.device)
        pages = table[b, : -(-n // c['page'])]
        for h in range(c['kv_heads']):
            kb = full['k'][pages, h].reshape(-1, c['dim'])[:n]
            vb = full['v'][pages, h].reshape(-1, c['dim'])[:n]
            q = s['q'][b, :fresh[b], h * group:(h + 1) * group].double()
            z = torch.matmul(q.reshape(-1, c['dim']), kb.t()).view(fresh[b], group, n) / math.sqrt(c['dim'])
            block = hide[None, :].expand(fresh[b], n)
            if c['causal']:
                block = block | (p[None, :] > n - fresh[b] + torch.arange(fresh[b], device=table.device)[:, None])
            z = z.masked_fill(block[:, None, :], -math.inf)
            w = torch.softmax(z, dim=-1).masked_fill(block.all(-1)[:, None, None], 0.0)
            out[b, :fresh[b], h * group:(h + 1) * group] = torch.matmul(w.reshape(-1, n), vb).view(fresh[b], group, -1)
    return out if c['op'] == 'attend' else [out] + state
