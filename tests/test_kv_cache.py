"""The paged key/value cache: kv_append, kv_read, paged_attention (csrc/kv_cache.hip, csrc/paged_attention.h) against plain
statements in 64 bits.  Pools are filled with NaN wherever no row has been written, so whatever reads past a sequence shows."""
import ctypes
import math

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu

SCALED = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
ROWS = (torch.float32, torch.bfloat16, torch.float16)
POOLS = ROWS + tuple(SCALED)
PAIRS = [(r, c) for r in ROWS for c in POOLS if r == torch.float32 or r == c or c in SCALED]
NAN = float('nan')


def short(t):
    return str(t).replace('torch.', '').replace('float8_', '')


# ---- plain statements (CPU) -------------------------------------------------------------------------------------------------
def quantise(x, dtype):
    """rows (..., D) -> (stored values in `dtype`, scale or None), bit for bit what a pool holds"""
    x = x.float()
    if dtype not in SCALED:
        return x.to(dtype), None
    s = (x.abs().amax(-1) * torch.tensor(1.0 / SCALED[dtype], dtype=torch.float32)).clamp_min(2.0 ** -126)
    y = x / s[..., None]
    return (y.round().nan_to_num(0.0).to(torch.int8) if dtype == torch.int8 else y.to(dtype)), s


def wide(code, scale):
    x = code.float().double()
    return x if scale is None else x * scale.double()[..., None]


def reference(q, k, v, lens, fresh, hide, causal, scale):
    """q (B,T,HQ,D); k, v: lists of (len_b, H, D) in 64 bits -> out in 64 bits and how far off it may be, per element"""
    B, T, HQ, D = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    eps = torch.finfo(q.dtype).eps / 2
    for b in range(B):
        n = int(lens[b])
        H = k[b].shape[1]
        for t in range(int(fresh[b])):
            see = torch.ones(n, dtype=torch.bool)
            if hide is not None:
                see[:hide.shape[1]] &= ~hide[b, :n]
                see[hide.shape[1]:] = False
            if causal:
                see[n - int(fresh[b]) + t + 1:] = False
            if not bool(see.any()):
                continue
            for j in range(HQ):
                h = j // (HQ // H)
                kk, vv, qq = k[b][see, h], v[b][see, h], q[b, t, j].double()
                z = kk @ qq * scale
                w = torch.exp(z - z.max())
                o = (w / w.sum()) @ vv
                out[b, t, j] = o
                # f32 sums of D products (each rounding 2^-24 of the terms' magnitudes), the product with the scale(s) and the
                # subtraction of the maximum: the error of z, which is a relative error of every weight -- twice, for the sum too;
                # exp2 and the sums over the keys: 2^-23 + keys * 2^-24; the split weights: 2^-17; one rounding of the result
                dz = (D + 6) * 2.0 ** -24 * float((kk.abs() @ qq.abs()).max()) * abs(scale)     # |scale * e| = |scale| |e|
                rel = 2 * dz + (int(see.sum()) + 16) * 2.0 ** -24 + (0 if q.dtype == torch.float32 else 2.0 ** -17)
                tol[b, t, j] = rel * vv.abs().amax(0) * 2 + eps * o.abs() + torch.finfo(q.dtype).smallest_normal * eps
    return out, tol


class Cache:
    """a pool on the device, its mirror as lists of rows, and a table that uses pages in a shuffled order"""

    def __init__(self, ops, lens, heads, dim, page, dtype, seed, extra=0, nhd=False, slack=0, poison=True):
        g = torch.Generator().manual_seed(seed)
        self.g, self.lens, self.page, self.dtype = g, torch.tensor(lens, dtype=torch.int32), page, dtype
        B, W = len(lens), max(1, -(-max(lens + [1]) // page)) + extra
        pool = B * W + 2
        self.table = torch.randperm(pool, generator=g)[:B * W].view(B, W).to(torch.int32)
        shape = (pool, heads, page, dim + slack)
        fill = {torch.int8: 77, torch.float8_e4m3fn: 0x7f}.get(dtype)
        self.host = []
        for _ in range(2):
            if fill is not None:
                code = torch.full(shape, fill, dtype=torch.uint8).view(dtype)
                scale = torch.full(shape[:3], NAN if poison else 1.0)
            else:
                code, scale = torch.full(shape, NAN if poison else 1.0).to(dtype), None
            self.host.append([code, scale])
        self.rows = []
        for code, scale in self.host:
            per = []
            for b, n in enumerate(lens):
                x = torch.randn((n, heads, dim), generator=g) * (0.5 + torch.rand((n, heads, 1), generator=g))
                c, s = quantise(x, dtype)
                p = torch.arange(n)
                at = self.table[b, p // page].long()
                code.view(torch.uint8 if dtype in SCALED else dtype)[at, :, p % page, :dim] = c.view(torch.uint8 if dtype in SCALED else dtype)
                if s is not None:
                    scale[at, :, p % page] = s
                per.append(wide(c, s))
            self.rows.append(per)

        def up(code):
            if nhd:
                return code.view(torch.uint8 if dtype in SCALED else dtype).transpose(1, 2).contiguous().cuda().view(dtype).transpose(1, 2)[..., :dim]
            return code.view(torch.uint8 if dtype in SCALED else dtype).cuda().view(dtype)[..., :dim]
        self.pages = ops.KVPages(*(up(c) for c, _ in self.host), *(s.cuda() if s is not None else None for _, s in self.host))
        self.dev_table, self.dev_lens = self.table.cuda(), self.lens.cuda()


def bits(t):
    return t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]).cpu()


def check(ops, c, q, new_lens=None, hide=None, causal=True, scale=None, **kw):
    got = ops.paged_attention(q.cuda(), c.pages, c.dev_table, c.dev_lens, new_lens=None if new_lens is None else new_lens.cuda(),
                              key_padding_mask=None if hide is None else hide.cuda(), causal=causal, scale=scale, **kw)
    assert got.dtype == q.dtype and got.shape == q.shape
    fresh = torch.minimum(c.lens, torch.full_like(c.lens, q.shape[1]) if new_lens is None else new_lens.clamp(0, q.shape[1]))
    want, tol = reference(q, c.rows[0], c.rows[1], c.lens, fresh, hide, causal, q.shape[3] ** -0.5 if scale is None else scale)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), 'worst %.3g of its tolerance' % float((err / tol.clamp_min(1e-300)).max())
    return got


def queries(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---- without a GPU: what the entry points refuse -----------------------------------------------------------------------------
def pages_struct(**kw):
    from openpvsg_amd import _lib
    d = dict(k=4096, v=8192, k_scale=None, v_scale=None, page_stride=4 * 16 * 64, head_stride=16 * 64, slot_stride=64, scale_page_stride=64,
             scale_head_stride=16, num_pages=8, heads=4, page_size=16, dim=64, type=0, faults=None)
    d.update(kw)
    return _lib.KvPages(*(d[n] for n, _ in _lib.KvPages._fields_))


BAD_POOLS = [dict(k=None), dict(v=8200), dict(page_size=24), dict(page_size=4), dict(dim=40), dict(dim=272), dict(dim=0), dict(type=7), dict(type=3),
             dict(num_pages=0), dict(heads=0), dict(slot_stride=66), dict(slot_stride=32), dict(type=4, k_scale=1024, v_scale=1030),
             dict(type=4, k_scale=1024, v_scale=2048, scale_page_stride=62)]


@pytest.mark.parametrize('bad', BAD_POOLS, ids=str)
def test_bad_pools_are_refused(hip_lib, bad):
    p, one = pages_struct(**bad), ctypes.c_void_p(4096)
    assert hip_lib.pvsg_kv_append(p, one, one, 0, 64, 64, 64, one, 2, 2, one, None, 1, 1, None) == 1
    assert hip_lib.pvsg_kv_read(p, one, one, 0, one, 2, 2, one, 1, 0, 4, None) == 1
    assert hip_lib.pvsg_paged_attention(p, one, 64, 64, 64, one, 0, one, 2, 2, one, None, None, 0, 0, 1, 1, 4, 1.0, 1, 0, None, None, None) == 1
    assert len(hip_lib.pvsg_last_error()) > 10


def test_bad_calls_are_refused(hip_lib):
    p, one = pages_struct(), ctypes.c_void_p(4096)

    def append(k=one, row=0, st=(64, 64, 64), table=one, width=2, lens=one, B=1, T=1):
        return hip_lib.pvsg_kv_append(p, k, one, row, *st, table, width, width, lens, None, B, T, None)

    def read(out=one, kind=0, B=1, start=0, length=4):
        return hip_lib.pvsg_kv_read(p, out, one, kind, one, 2, 2, one, B, start, length, None)

    def attend(pool=p, q=one, out=one, row=0, T=1, HQ=4, width=2, work=None, count=None, st=(64, 64, 64), B=1):
        return hip_lib.pvsg_paged_attention(pool, q, *st, out, row, one, width, width, one, None, None, 0, 0, B, T, HQ, 1.0, 1, 0, work, count, None)

    for rc in (append(k=None), append(row=3), append(st=(64, 64, 66)), append(table=None), append(width=0), append(width=1 << 27), append(lens=None),
               append(B=-1), append(B=70000), append(T=-1), append(k=ctypes.c_void_p(4100)),
               read(out=None), read(kind=4), read(B=-2), read(start=-1), read(length=-1), read(out=ctypes.c_void_p(4104)),
               attend(q=None), attend(out=None), attend(row=5), attend(T=33), attend(HQ=6), attend(HQ=0),
               attend(width=5000), attend(width=5000, work=one), attend(width=5000, work=ctypes.c_void_p(4100), count=one),
               attend(width=5000, work=one, count=ctypes.c_void_p(4098)), attend(st=(64, 66, 64)), attend(row=1),
               attend(pool=pages_struct(type=2), row=1), attend(pool=pages_struct(type=1), row=2)):
        assert rc == 1, hip_lib.pvsg_last_error()
    # nothing to do is no error and launches nothing
    assert append(B=0) == 0 and append(T=0) == 0 and read(length=0) == 0 and read(B=0) == 0 and attend(B=0) == 0 and attend(T=0) == 0


def test_calls_past_one_launch_are_refused(hip_lib):
    """a launch holds fewer than 2^32 threads: 2^24 workgroups of 256"""
    p, one = pages_struct(dim=256, heads=1, page_stride=16 * 256, head_stride=16 * 256, slot_stride=256), ctypes.c_void_p(4096)
    big = (1 << 27) + 8                                              # rows of 32 lanes
    assert hip_lib.pvsg_kv_append(p, one, one, 0, 256, 256, 256, one, 2, 2, one, None, 1, big, None) == 1
    assert hip_lib.pvsg_kv_read(p, one, one, 0, one, 2, 2, one, 1, 0, big, None) == 1
    p = pages_struct(heads=1024)
    assert hip_lib.pvsg_paged_attention(p, one, 64, 64, 64, one, 0, one, 2, 2, one, None, None, 0, 0, 65535, 1, 1024, 1.0, 1, 0, None, None, None) == 1


def test_workspace_is_bounded_by_the_card(hip_lib):
    """none where every cache is a few tiles, and two parts for each of at most 1024 workgroups however long the caches are"""
    def f(B=1, T=1, HQ=4, row=0, width=1, longest=0, **kw):
        return hip_lib.pvsg_paged_attention_workspace_bytes(pages_struct(**kw), B, T, HQ, row, width, longest)
    assert f() == 0 and f(width=1000, longest=1) == 0 and f(B=0, width=1000) == 0
    last = 0
    for width in (64, 1000, 4096, 1 << 20):
        n = f(width=width)
        assert last <= n <= 2 * 1024 * 32 * (64 + 2) * 4
        last = n
    assert f(B=60000, T=32, HQ=64, width=1 << 20) <= 2 * 1024 * 32 * (64 + 2) * 4


def test_cpu_tensors_are_refused(hip_lib):
    from openpvsg_amd import ops
    with pytest.raises(RuntimeError, match='no CPU path'):
        ops.KVPages(torch.zeros(2, 2, 8, 16), torch.zeros(2, 2, 8, 16))


def test_quantise_statement_round_trips():
    """the plain statement the GPU tests compare with: half a step of each type at most"""
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(3))
    for dtype, steps in ((torch.float8_e4m3fn, 2.0 ** -4), (torch.int8, None)):
        c, s = quantise(x, dtype)
        err = (wide(c, s) - x.double()).abs()
        half = x.double().abs() * steps + s.double()[:, None] * 2.0 ** -10 if steps else s.double()[:, None] * 0.5
        assert bool((err <= half * (1 + 2.0 ** -20)).all())


# ---- append ----------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize('pool', POOLS, ids=short)
@pytest.mark.parametrize('row', ROWS, ids=short)
def test_append_is_bit_exact_and_touches_nothing_else(hip_lib, row, pool):
    from openpvsg_amd import ops
    for seed, (B, T, H, D, page, new) in enumerate(((1, 1, 1, 16, 8, None), (5, 7, 3, 80, 8, [7, 0, 3, 9, -2]), (3, 33, 4, 128, 16, None), (2, 5, 2, 256, 32, [5, 4]))):
        lens = [T + 9 * b for b in range(B)]
        lens[-1] = T // 2                                          # fewer positions than rows: the first ones are taken
        c = Cache(ops, lens, H, D, page, pool, seed)
        kv = torch.randn((B, T, 2, H, D), generator=c.g) * torch.exp(2 * torch.randn((B, T, 1, H, 1), generator=c.g)).clamp(max=8000.0)
        kv[0, 0, 0, 0] = 0.0                                         # a row of zeros
        kv = kv.to(row)
        dev = kv.cuda()
        want = [[x.clone() if x is not None else None for x in pair] for pair in c.host]
        for b in range(B):
            n = max(0, min(T, lens[b], T if new is None else new[b]))
            p = torch.arange(lens[b] - n, lens[b])
            at = c.table[b, p // page].long()
            for which in range(2):
                code, s = quantise(kv[b, :n, which], pool)
                if pool == torch.float16:
                    code = kv[b, :n, which].float().to(pool)
                view = torch.uint8 if pool in SCALED else pool
                want[which][0].view(view)[at, :, p % page] = code.view(view)
                if s is not None:
                    want[which][1][at, :, p % page] = s
        r = ops.kv_append(c.pages, dev[:, :, 0], dev[:, :, 1], c.dev_table, c.dev_lens, None if new is None else torch.tensor(new, dtype=torch.int32).cuda())
        assert r is c.pages
        for which, (code, s) in enumerate(((c.pages.k, c.pages.k_scale), (c.pages.v, c.pages.v_scale))):
            assert torch.equal(bits(code), bits(want[which][0])), (B, T, H, D, which)
            if s is not None:
                assert torch.equal(bits(s), bits(want[which][1]))
        ops.page_fault_check()


@gpu
def test_append_of_rows_that_are_not_finite_or_tiny(hip_lib):
    from openpvsg_amd import ops
    for pool in SCALED:
        c = Cache(ops, [4], 2, 32, 8, pool, 1)
        x = torch.randn(1, 4, 2, 32)
        x[0, 0, 0, 5], x[0, 1, 1, 31], x[0, 2] = NAN, float('inf'), 1e-42
        ops.kv_append(c.pages, x.cuda(), x.cuda(), c.dev_table, c.dev_lens)
        for y in ops.kv_read(c.pages, c.dev_table, c.dev_lens, 4):
            y = y.cpu()[0]
            assert bool(y[0, 0].isnan().all()) and bool(y[1, 1].isnan().all())
            assert bool((y[2].abs() <= 1e-37).all())
            for t, h in ((0, 1), (1, 0), (3, 0), (3, 1)):
                s = x[0, t, h].abs().max() / SCALED[pool]
                assert bool(((y[t, h] - x[0, t, h]).abs() <= (s * 0.5 if pool == torch.int8 else x[0, t, h].abs() * 2.0 ** -4 + s * 2.0 ** -10) * 1.001).all())


# ---- read ------------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize('pool', POOLS, ids=short)
@pytest.mark.parametrize('row', ROWS, ids=short)
def test_read_gives_the_rows_and_zeros_behind_them(hip_lib, row, pool):
    from openpvsg_amd import ops
    for lens, H, D, page, start, length in (([1], 1, 16, 8, 0, 1), ([0, 13, 40, 8], 3, 96, 8, 0, 41), ([37, 5], 2, 256, 16, 7, 45), ([20], 4, 128, 32, 20, 3)):
        c = Cache(ops, lens, H, D, page, pool, 5)
        for got, rows in zip(ops.kv_read(c.pages, c.dev_table, c.dev_lens, length, start=start, dtype=row), c.rows):
            want = torch.zeros(len(lens), length, H, D, dtype=torch.float64)
            for b, x in enumerate(rows):
                x = x[start:start + length]
                want[b, :x.shape[0]] = x
            # code * scale is rounded to f32, and that to the output's type: a value next to a border may take the other side, so
            # half a step and a half of f32's
            tol = want.abs() * (torch.finfo(row).eps / 2 + 2.0 ** -24) + torch.finfo(row).smallest_normal * torch.finfo(row).eps
            assert got.dtype == row and bool(((got.cpu().double() - want).abs() <= tol).all())
    ops.page_fault_check()


# ---- attention -------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize('row,pool', PAIRS, ids=lambda t: short(t))
def test_attention_types_and_head_sizes(hip_lib, row, pool):
    from openpvsg_amd import ops
    for seed, (lens, H, G, D, page, T) in enumerate((([1], 1, 1, 16, 8, 1), ([33, 0, 7, 64], 4, 1, 32, 8, 1), ([100, 31], 2, 4, 64, 16, 2),
                                                     ([257, 129], 2, 2, 80, 32, 3), ([70, 300], 1, 3, 128, 16, 1), ([45], 2, 5, 128, 64, 4), ([19, 66], 1, 2, 256, 8, 1),
                                                     ([50], 1, 8, 208, 16, 5))):
        c = Cache(ops, lens, H, D, page, pool, seed)
        check(ops, c, queries((len(lens), T, H * G, D), row, seed))
    ops.page_fault_check()


@gpu
@pytest.mark.parametrize('causal', (True, False))
@pytest.mark.parametrize('T', (1, 2, 16, 17, 32))
def test_attention_new_tokens(hip_lib, T, causal):
    """one to 32 new tokens, some sequences with fewer (or none): rows past them are zero, also over what was there"""
    from openpvsg_amd import ops
    for row, pool, H, G, D in ((torch.float32, torch.float32, 2, 1, 32), (torch.bfloat16, torch.float8_e4m3fn, 1, 3, 64), (torch.float16, torch.float16, 2, 2, 128)):
        lens = [T, 130, 5, 0, 301]
        c = Cache(ops, lens, H, D, 8, pool, T)
        new = torch.tensor([T, max(1, T // 2), T, T, 0], dtype=torch.int32)
        q = queries((5, T, H * G, D), row, T)
        got = check(ops, c, q, new_lens=new, causal=causal)
        out = torch.full_like(got, 7.0)
        assert ops.paged_attention(q.cuda(), c.pages, c.dev_table, c.dev_lens, new_lens=new.cuda(), causal=causal, out=out) is out
        assert torch.equal(bits(out), bits(got))


@gpu
@pytest.mark.parametrize('row,pool', ((torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.int8)), ids=short)
def test_attention_padding(hip_lib, row, pool):
    """masks of every kind: random, all of a sequence, all that a causal row sees, shorter than the cache, wider than it"""
    from openpvsg_amd import ops
    lens = [200, 77, 9, 150]
    for T, M in ((1, 200), (3, 201), (3, 77), (2, 1)):
        c = Cache(ops, lens, 2, 64, 16, pool, M)
        hide = torch.rand((4, M), generator=c.g) < 0.4
        hide[1] = True
        hide[2, :9 - T + 1] = True
        check(ops, c, queries((4, T, 4, 64), row, M), hide=hide)
        wider = torch.zeros(4, M + 5, dtype=torch.bool)
        wider[:, :M] = hide
        check(ops, c, queries((4, T, 4, 64), row, M), hide=wider[:, :M])                # a view with rows M + 5 apart
    c = Cache(ops, lens, 2, 64, 16, pool, 1)
    got = ops.paged_attention(queries((4, 1, 4, 64), row, 1).cuda(), c.pages, c.dev_table, c.dev_lens, key_padding_mask=torch.zeros(4, 0, dtype=torch.bool, device='cuda'))
    assert not bool(got.any())


@gpu
@pytest.mark.parametrize('bad', (NAN, float('inf'), -float('inf')))
@pytest.mark.parametrize('row,pool', ((torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                      (torch.bfloat16, torch.float8_e4m3fn)), ids=short)
def test_what_is_masked_never_reaches_a_result(hip_lib, row, pool, bad):
    from openpvsg_amd import ops
    T, n, D = 4, 90, 64
    hide = torch.zeros(1, n, dtype=torch.bool)
    hide[0, [3, 40, 41]] = True
    q = queries((1, T, 4, D), row, 9)
    c = Cache(ops, [n], 2, D, 16, pool, 2)
    clean = check(ops, c, q, hide=hide).cpu()
    for at in (3, 40, 87, 88, 89):                                   # masked, masked, and the later tokens of the clip
        slot = (int(c.table[0, at // 16]), slice(None), at % 16)
        if pool == torch.float8_e4m3fn:
            c.pages.k_scale[slot], c.pages.v_scale[slot] = bad, bad
            c.pages.k.view(torch.uint8)[slot], c.pages.v.view(torch.uint8)[slot] = 0x7f, 0x7f
        else:
            c.pages.k[slot], c.pages.v[slot] = bad, bad
    got = ops.paged_attention(q.cuda(), c.pages, c.dev_table, c.dev_lens, key_padding_mask=hide.cuda()).cpu()
    # the first token sees nothing of it: within both calls' tolerances of the clean result (and no NaN)
    want, tol = reference(q, c.rows[0], c.rows[1], c.lens, torch.tensor([T]), hide, True, D ** -0.5)
    assert bool(((got.double() - want).abs() <= tol)[0, 0].all()) and bool(clean.isfinite().all())
    assert not bool(got[0, 1:].isfinite().all())                     # the later ones do see it


@gpu
@pytest.mark.parametrize('row,pool', ((torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)), ids=short)
def test_a_visible_infinity_comes_out_as_one(hip_lib, row, pool):
    from openpvsg_amd import ops
    c = Cache(ops, [300, 40], 2, 32, 8, pool, 4)
    c.pages.v[int(c.table[0, 20]), 1, 3, 7] = float('inf')          # position 163 of sequence 0, key head 1
    c.pages.v[int(c.table[0, 2]), 0, 0, 9] = NAN
    q = queries((2, 1, 4, 32), row, 4)
    got = ops.paged_attention(q.cuda(), c.pages, c.dev_table, c.dev_lens).cpu()
    want, tol = reference(q, c.rows[0], c.rows[1], c.lens, torch.tensor([1, 1]), None, True, 32 ** -0.5)
    assert bool((got[0, 0, 2:, 7] == float('inf')).all()) and bool(got[0, 0, :2, 9].isnan().all())
    ok = (got.double() - want).abs() <= tol
    ok[0, 0, 2:, 7] = ok[0, 0, :2, 9] = True
    assert bool(ok.all())


@gpu
@pytest.mark.parametrize('row,pool,D', ((torch.float32, torch.float32, 128), (torch.bfloat16, torch.bfloat16, 64), (torch.bfloat16, torch.int8, 256)), ids=str)
def test_attention_split_over_a_long_cache(hip_lib, row, pool, D):
    """one sequence over many workgroups, joined: any plan gives the result, and the same plan the same bits"""
    from openpvsg_amd import ops
    c = Cache(ops, [9001, 1, 4097], 1, D, 16, pool, 6)
    q = queries((3, 1, 2, D), row, 6)
    a = check(ops, c, q)
    assert torch.equal(bits(a), bits(check(ops, c, q)))
    for hint in (1, 100, 5000, 10 ** 9):
        check(ops, c, q, max_len=hint)
    check(ops, c, queries((3, 1, 40, D), row, 7))                    # 40 rows a key head: several row groups


@gpu
@pytest.mark.parametrize('B', (63, 64, 65, 129, 256, 257, 300, 1500, 4200))
def test_attention_batches_of_every_size(hip_lib, B):
    """the shares of a long batch: most sequences short, some long, some empty (each workgroup finds its share by a scan over the lengths)"""
    from openpvsg_amd import ops
    g = torch.Generator().manual_seed(B)
    lens = (1 + 60 * torch.rand(B, generator=g) ** 3).int()
    lens[torch.randint(0, B, (max(2, B // 50),), generator=g)] = 0
    lens[torch.randint(0, B, (3,), generator=g)] = torch.tensor([1500, 2500, 1100], dtype=torch.int32)
    lens[B - 1] = 1300
    c = Cache(ops, lens.tolist(), 1, 16, 16, torch.float32, B)
    check(ops, c, queries((B, 1, 2, 16), torch.float32, B))


@gpu
def test_attention_scale_and_large_logits(hip_lib):
    from openpvsg_amd import ops
    c = Cache(ops, [130, 64], 2, 64, 16, torch.float32, 3)
    for scale in (0.0, 1.0, 3.0, -0.5):
        check(ops, c, queries((2, 2, 2, 64), torch.float32, 3), scale=scale)


@gpu
@pytest.mark.parametrize('pool', POOLS, ids=short)
def test_layouts(hip_lib, pool):
    """pools with slots before heads, pools with room behind each row, tables and queries that are parts of wider tensors"""
    from openpvsg_amd import ops
    for nhd, slack in ((True, 0), (False, 16), (True, 48)):
        c = Cache(ops, [50, 7, 121], 3, 48, 16, pool, 8, extra=2, nhd=nhd, slack=slack)
        wide_q = queries((3, 2, 9, 48), torch.float32, 8)
        check(ops, c, wide_q)
        want = ops.paged_attention(wide_q.cuda()[:, :, :6].contiguous(), c.pages, c.dev_table, c.dev_lens)
        table = torch.zeros(3, c.table.shape[1] + 3, dtype=torch.int32, device='cuda')
        table[:, 1:-2] = c.dev_table
        got = ops.paged_attention(wide_q.cuda()[:, :, :6], c.pages, table[:, 1:-2], c.dev_lens)
        assert torch.equal(bits(got), bits(want))
        flat = torch.zeros(wide_q.numel() + 1, device='cuda')          # rows that start 4 bytes off
        flat[1:] = wide_q.cuda().flatten()
        assert torch.equal(bits(ops.paged_attention(flat[1:].view(wide_q.shape)[:, :, :6], c.pages, table[:, 1:-2], c.dev_lens)), bits(want))
        x = queries((3, 4, 3, 48), torch.float32, 9).cuda()
        ops.kv_append(c.pages, x, x.transpose(1, 2).contiguous().transpose(1, 2), table[:, 1:-2], c.dev_lens)
        for got, rows in zip(ops.kv_read(c.pages, table[:, 1:-2], c.dev_lens, 121), (x, x)):
            code, s = quantise(rows[0].cpu(), pool)
            assert float((got[0, 46:50].cpu().double() - wide(code, s)).abs().max()) <= 2.0 ** -24 * 8


@gpu
def test_bad_page_ids_and_lengths_are_skipped_and_reported(hip_lib):
    from openpvsg_amd import ops
    ops.page_fault_check()
    c = Cache(ops, [64, 64], 2, 32, 16, torch.float32, 1)
    bad = c.dev_table.clone()
    bad[0, 1], bad[0, 3], bad[1, 0] = -1, c.pages.num_pages, 1 << 30
    hide = torch.zeros(2, 64, dtype=torch.bool)
    hide[0, 16:32] = hide[0, 48:] = hide[1, :16] = True
    q = queries((2, 1, 2, 32), torch.float32, 2)
    want = ops.paged_attention(q.cuda(), c.pages, c.dev_table, c.dev_lens, key_padding_mask=hide.cuda(), causal=False)
    ops.page_fault_check()
    got = ops.paged_attention(q.cuda(), c.pages, bad, c.dev_lens, causal=False)
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-6)
    with pytest.raises(RuntimeError, match='paged_attention met page ids'):
        ops.page_fault_check()
    ops.page_fault_check()                                           # reported once
    k, _ = ops.kv_read(c.pages, bad, c.dev_lens, 64)
    full, _ = ops.kv_read(c.pages, c.dev_table, c.dev_lens, 64)
    assert torch.equal(k, torch.where(hide.cuda()[:, :, None, None], torch.zeros_like(full), full))
    with pytest.raises(RuntimeError, match='kv_read met'):
        ops.page_fault_check()
    before = bits(c.pages.k)
    x = torch.ones(2, 16, 2, 32, device='cuda')
    ops.kv_append(c.pages, x[:1], x[:1], bad[:1], c.dev_lens[:1])    # the last 16 positions of sequence 0: its page is bad
    assert torch.equal(bits(c.pages.k), before)
    with pytest.raises(RuntimeError, match='kv_append met'):
        ops.page_fault_check()
    # a length past the table: what the table holds is used, the rows behind it are dropped
    longer = torch.tensor([70, 64], dtype=torch.int32, device='cuda')
    ops.kv_append(c.pages, x[:, :8], x[:, :8], c.dev_table, longer)
    with pytest.raises(RuntimeError, match='kv_append met'):
        ops.page_fault_check()
    k, _ = ops.kv_read(c.pages, c.dev_table, longer, 72)
    assert bool((k[0, 62:64] == 1).all()) and not bool(k[0, 64:].any()) and torch.equal(k[0, :62], full[0, :62]) and bool((k[1, 56:64] == 1).all())
    with pytest.raises(RuntimeError, match='kv_read met'):
        ops.page_fault_check()
    negative = torch.tensor([-5, 64], dtype=torch.int32, device='cuda')
    assert not bool(ops.paged_attention(q.cuda(), c.pages, c.dev_table, negative)[0].any())
    ops.page_fault_check()


@gpu
def test_idle_sequences_need_no_pages(hip_lib):
    """a batch padded with sequences of length 0, whose table rows hold anything"""
    from openpvsg_amd import ops
    ops.page_fault_check()
    for T, longest in ((1, 40), (3, 3000)):
        c = Cache(ops, [0, longest, 0, 17, 0], 2, 64, 16, torch.bfloat16, T)
        c.dev_table[0], c.dev_table[2], c.dev_table[4] = -1, 1 << 30, -(1 << 31)
        got = check(ops, c, queries((5, T, 4, 64), torch.bfloat16, T))
        assert not bool(got[::2].any())
        x = torch.ones(5, T, 2, 64, dtype=torch.bfloat16, device='cuda')
        ops.kv_append(c.pages, x, x, c.dev_table, c.dev_lens)
        k, _ = ops.kv_read(c.pages, c.dev_table, c.dev_lens, longest)
        assert not bool(k[::2].any()) and bool((k[1, longest - T:] == 1).all())
        ops.page_fault_check()


@gpu
@pytest.mark.parametrize('row,pool', ((torch.float32, torch.float32), (torch.bfloat16, torch.float8_e4m3fn)), ids=short)
def test_captured_and_eager_joins_give_the_same_bits(hip_lib, row, pool):
    """split rows joined by whoever comes last, with a stream's own counters and with a graph's: many ragged sequences, rows of one and
    of two tiles"""
    from openpvsg_amd import ops
    lens = [1 + (7919 * i) % 2500 for i in range(70)] + [6000, 0]
    for H, G, T, D in ((2, 1, 1, 64), (1, 5, 4, 128), (1, 2, 32, 32)):
        c = Cache(ops, lens, H, D, 32, pool, 1)
        q = queries((len(lens), T, H * G, D), row, 2).cuda()
        out = torch.full_like(q, 3.0)
        eager = [ops.paged_attention(q, c.pages, c.dev_table, c.dev_lens) for _ in range(3)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention(q, c.pages, c.dev_table, c.dev_lens, out=out)
        for i in range(3):
            out.fill_(3.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(bits(out), bits(eager[i]))
        some = [0, 7, 70, 71]
        fresh = torch.minimum(c.lens, torch.full_like(c.lens, T))
        want, tol = reference(q.cpu()[some], [c.rows[0][b] for b in some], [c.rows[1][b] for b in some], c.lens[some], fresh[some], None, True, D ** -0.5)
        assert bool(((out.cpu()[some].double() - want).abs() <= tol).all())


@gpu
def test_shared_memory_is_refused(hip_lib):
    """scales that K and V share are not written, and the result does not go where the queries are read from"""
    from openpvsg_amd import ops
    f = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device='cuda')  # noqa: E731
    table, lens, x, scales = f(3, 2, dtype=torch.int32), f(3, dtype=torch.int32), f(3, 1, 2, 32), f(4, 2, 8)
    with pytest.raises(RuntimeError, match='same memory'):
        ops.kv_append(ops.KVPages(f(4, 2, 8, 32, dtype=torch.int8), f(4, 2, 8, 32, dtype=torch.int8), scales, scales), x, x, table, lens)
    p, both = ops.KVPages.empty(4, 2, 8, 32), f(6, 1, 4, 32)
    for q, out in ((both[:3], both[:3]), (both[:3], both[2:5]), (both[2:5], both[:3]), (both[:, :, :2][:3], both.view(-1)[64:256].view(3, 1, 2, 32))):
        with pytest.raises(RuntimeError, match='overlaps'):
            ops.paged_attention(q, p, table, lens, out=out)
    out = both[3:]
    assert ops.paged_attention(both[:3], p, table, lens, out=out) is out


@gpu
def test_refusals_on_the_device(hip_lib):
    from openpvsg_amd import ops
    f = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device='cuda')  # noqa: E731
    for k, v, ks, vs in ((f(2, 2, 8, 20), f(2, 2, 8, 20), None, None), (f(2, 2, 12, 16), f(2, 2, 12, 16), None, None), (f(2, 2, 8, 272), f(2, 2, 8, 272), None, None),
                         (f(2, 2, 8, 16), f(2, 2, 8, 32), None, None), (f(2, 2, 8, 16), f(2, 2, 8, 16, dtype=torch.bfloat16), None, None),
                         (f(2, 2, 8, 16, dtype=torch.float64), f(2, 2, 8, 16, dtype=torch.float64), None, None), (f(2, 8, 16), f(2, 8, 16), None, None),
                         (f(2, 2, 8, 16, dtype=torch.int8), f(2, 2, 8, 16, dtype=torch.int8), None, None), (f(2, 2, 8, 16), f(2, 2, 8, 16), f(2, 2, 8), f(2, 2, 8)),
                         (f(2, 2, 8, 16, dtype=torch.int8), f(2, 2, 8, 16, dtype=torch.int8), f(2, 8, 2).transpose(1, 2), f(2, 2, 8)),
                         (f(2, 2, 16, 8).transpose(2, 3), f(2, 2, 16, 8).transpose(2, 3), None, None), (f(2, 2, 8, 17)[..., 1:], f(2, 2, 8, 17)[..., 1:], None, None),
                         (f(2, 2, 1, 16).expand(2, 2, 8, 16), f(2, 2, 1, 16).expand(2, 2, 8, 16), None, None),
                         (f(2, 1, 8, 16).expand(2, 2, 8, 16), f(2, 1, 8, 16).expand(2, 2, 8, 16), None, None),
                         (f(1, 2, 8, 16).expand(2, 2, 8, 16), f(1, 2, 8, 16).expand(2, 2, 8, 16), None, None)):
        with pytest.raises(RuntimeError):
            ops.KVPages(k, v, ks, vs)
    p = ops.KVPages.empty(4, 2, 8, 32)
    h = ops.KVPages.empty(4, 2, 8, 32, dtype=torch.float16)
    table, lens = f(3, 2, dtype=torch.int32), f(3, dtype=torch.int32)
    x, q = f(3, 1, 2, 32), f(3, 1, 4, 32)
    one = f(4, 2, 8, 32)
    bad = [lambda: ops.kv_append(ops.KVPages(one, one), x, x, table, lens), lambda: ops.kv_append(p, x, x, table.long(), lens), lambda: ops.kv_append(p, x, x, table[:2], lens), lambda: ops.kv_append(p, x, x, table, lens[:2]),
           lambda: ops.kv_append(p, x, x.half(), table, lens), lambda: ops.kv_append(p, q, q, table, lens), lambda: ops.kv_append(p, x[0], x[0], table, lens),
           lambda: ops.kv_append(p, x.cpu(), x.cpu(), table, lens), lambda: ops.kv_append(p, x.double(), x.double(), table, lens),
           lambda: ops.kv_append(p, x, x, table.cpu(), lens), lambda: ops.kv_append(p, x, x, table, lens, new_lens=lens.long()),
           lambda: ops.kv_append(p, x.clone().requires_grad_(), x, table, lens), lambda: ops.kv_append(p, x, f(3, 2, 2, 32), table, lens),
           lambda: ops.kv_read(p, table, lens, -1), lambda: ops.kv_read(p, table, lens, 1, start=-1), lambda: ops.kv_read(p, table, lens, 4, dtype=torch.int8),
           lambda: ops.kv_read(p, table[:, :0], lens, 4), lambda: ops.kv_read(p, table, lens[:1], 4),
           lambda: ops.paged_attention(f(3, 33, 4, 32), p, table, lens), lambda: ops.paged_attention(f(3, 1, 3, 32), p, table, lens),
           lambda: ops.paged_attention(f(3, 1, 4, 16), p, table, lens), lambda: ops.paged_attention(q.half(), p, table, lens),
           lambda: ops.paged_attention(q.bfloat16(), h, table, lens), lambda: ops.paged_attention(q, p, table, lens, key_padding_mask=f(3, 16)),
           lambda: ops.paged_attention(q, p, table, lens, key_padding_mask=f(2, 16, dtype=torch.bool)), lambda: ops.paged_attention(q.clone().requires_grad_(), p, table, lens),
           lambda: ops.paged_attention(q, p, table, lens, out=q.half()), lambda: ops.paged_attention(q, p, table, lens, out=f(3, 1, 32, 4).transpose(2, 3)),
           lambda: ops.paged_attention(q, p, f(3, (1 << 27) + 1, dtype=torch.int32), lens)]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            print('call %d was not refused' % i)
    with torch.no_grad():
        assert ops.paged_attention(q.clone().requires_grad_(), p, table, lens).shape == q.shape
    assert ops.paged_attention(q[:0], p, table[:0], lens[:0]).shape == (0, 1, 4, 32) and ops.paged_attention(q[:, :0], p, table, lens).shape == (3, 0, 4, 32)
    assert ops.kv_read(p, table, lens, 0)[0].shape == (3, 0, 2, 32) and ops.kv_append(p, x[:, :0], x[:, :0], table, lens) is p


@gpu
def test_offsets_past_32_bits(hip_lib):
    """pages whose elements start past 2^32: the first and the last pages of a pool of 4.6e9 codes a side"""
    from openpvsg_amd import ops
    P, H, S, D = 70400, 8, 64, 128
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip('needs 24 GiB of free device memory')
    pages = ops.KVPages(*(torch.empty((P, H, S, D), dtype=torch.int8, device='cuda') for _ in range(2)), *(torch.empty((P, H, S), device='cuda') for _ in range(2)))
    assert pages.k.numel() > 1 << 32
    table = torch.tensor([[P - 1, 0, P - 3]], dtype=torch.int32, device='cuda')
    x = queries((1, 140, 2, H, D), torch.float32, 1)
    lens = torch.tensor([140], dtype=torch.int32, device='cuda')
    ops.kv_append(pages, x[:, :, 0].cuda(), x[:, :, 1].cuda(), table, lens)
    rows = [wide(*quantise(x[0, :, i], torch.int8)) for i in range(2)]
    for got, want in zip(ops.kv_read(pages, table, lens, 140), rows):
        assert float((got[0].cpu().double() - want).abs().max()) <= 2.0 ** -24 * 8
    q = queries((1, 1, H, D), torch.float32, 2)
    want, tol = reference(q, [rows[0]], [rows[1]], [140], [1], None, True, D ** -0.5)
    got = ops.paged_attention(q.cuda(), pages, table, lens).cpu().double()
    assert bool(((got - want).abs() <= tol).all())


# ---- together ----------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize('row,pool', ((torch.float32, torch.float32), (torch.float32, torch.float8_e4m3fn), (torch.bfloat16, torch.bfloat16)), ids=short)
def test_a_live_run(hip_lib, row, pool):
    """clips of 1..32 frames appended and attended from, sequence by sequence at its own pace; the result of each step is that of
    the rows that were given, rounded as the pool rounds them"""
    from openpvsg_amd import ops
    B, H, G, D, S, W = 3, 2, 2, 32, 8, 12
    g = torch.Generator().manual_seed(11)
    pages = ops.KVPages.empty(B * W, H, S, D, dtype=pool)
    table = torch.randperm(B * W, generator=g).view(B, W).to(torch.int32).cuda()
    lens = torch.zeros(B, dtype=torch.int32)
    past = [[torch.zeros(0, H, D, dtype=torch.float64) for _ in range(B)] for _ in range(2)]
    for step, T in enumerate((5, 1, 32, 1, 1, 17, 8)):
        new = torch.tensor([T, max(0, T - step), 1], dtype=torch.int32)
        lens = lens + new
        kv = torch.randn((B, T, 2, H, D), generator=g).to(row)
        q = torch.randn((B, T, H * G, D), generator=g).to(row)
        dev = kv.cuda()
        ops.kv_append(pages, dev[:, :, 0], dev[:, :, 1], table, lens.cuda(), new.cuda())
        got = ops.paged_attention(q.cuda(), pages, table, lens.cuda(), new.cuda())
        for i in range(2):
            for b in range(B):
                past[i][b] = torch.cat([past[i][b], wide(*quantise(kv[b, :int(new[b]), i], pool))])
        want, tol = reference(q, past[0], past[1], lens, new, None, True, D ** -0.5)
        assert bool(((got.cpu().double() - want).abs() <= tol).all()), step
    back = ops.kv_read(pages, table, lens.cuda(), int(lens.max()))
    for i in range(2):
        for b in range(B):
            assert float((back[i][b, :int(lens[b])].cpu().double() - past[i][b]).abs().max()) <= 2.0 ** -24 * 8
    ops.page_fault_check()


@gpu
def test_temporal_encoder_frame_by_frame(hip_lib):
    """The relation head's temporal encoder over a growing video: the newest frames' attention from the cache equals the module's own
    attention over all frames so far (its self-attention is not causal: every new frame sees every frame)."""
    from openpvsg_amd import ops
    from openpvsg_amd.relation import TemporalTransformer
    torch.manual_seed(5)
    attn = TemporalTransformer(512, 57).eval().transformer_encoder.layers[0].self_attn
    P, H, D = 4, attn.num_heads, attn.head_dim
    x = torch.randn(P, 41, 512)
    pages = ops.KVPages.empty(P * 6, H, 8, D)
    table = torch.arange(P * 6, dtype=torch.int32, device='cuda').view(P, 6)
    lens = torch.zeros(P, dtype=torch.int32, device='cuda')
    w, b = attn.in_proj_weight.detach().cuda(), attn.in_proj_bias.detach().cuda()
    wo, bo = attn.out_proj.weight.detach().cuda(), attn.out_proj.bias.detach().cuda()
    t = 0
    for n in (4, 32, 1, 1, 3):
        lens += n
        qkv = (x[:, t:t + n].cuda() @ w.t() + b).view(P, n, 3, H, D)
        ops.kv_append(pages, qkv[:, :, 1], qkv[:, :, 2], table, lens)
        got = ops.paged_attention(qkv[:, :, 0], pages, table, lens, causal=False).reshape(P, n, 512) @ wo.t() + bo
        t += n
        with torch.no_grad():
            seq = x[:, :t].double()
            mod = attn.double()
            want = mod(seq, seq, seq, need_weights=False)[0][:, t - n:] if mod.batch_first else mod(*(seq.transpose(0, 1),) * 3, need_weights=False)[0].transpose(0, 1)[:, t - n:]
        # three f32 contractions of 512 terms in a row, magnitudes about one
        assert float((got.cpu().double() - want).abs().max()) <= 3 * 512 * 2.0 ** -24 * 4


@gpu
def test_steps_replay_from_graphs(hip_lib):
    """append + attention captured once and replayed as the video grows; two graphs, eager calls between the replays"""
    from openpvsg_amd import ops
    B, H, D, S, W = 2, 2, 64, 16, 40
    pages = ops.KVPages.empty(2 * B * W, H, S, D, dtype=torch.float8_e4m3fn)
    tables = torch.arange(2 * B * W, dtype=torch.int32, device='cuda').view(2, B, W)
    g = torch.Generator().manual_seed(2)
    lens = torch.zeros(2, B, dtype=torch.int32, device='cuda')
    x = torch.zeros(B, 1, 3, H, D, device='cuda')

    def step(i):
        lens[i] += 1
        ops.kv_append(pages, x[:, :, 0], x[:, :, 1], tables[i], lens[i])
        return ops.paged_attention(x[:, :, 2], pages, tables[i], lens[i])

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step(0), step(1)
    torch.cuda.synchronize()
    lens.zero_()
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(i))
        graphs.append(graph)
    eager = ops.KVPages.empty(2 * B * W, H, S, D, dtype=torch.float8_e4m3fn)
    for n in range(40):
        for i in range(2):
            x.copy_(torch.randn(x.shape, generator=g))
            graphs[i].replay()
            got = outs[i].clone()
            ops.kv_append(eager, x[:, :, 0], x[:, :, 1], tables[i], lens[i])
            want = ops.paged_attention(x[:, :, 2], eager, tables[i], lens[i])
            torch.cuda.synchronize()
            assert int(lens[i, 0]) == n + 1 and torch.equal(bits(got), bits(want)), (n, i)


@gpu
def test_a_first_pool_made_in_inference_mode(hip_lib, monkeypatch):
    """the fault word that it makes is one that a check outside that mode can clear"""
    from openpvsg_amd import ops
    monkeypatch.setattr(ops, '_page_faults', {})
    monkeypatch.setattr(ops, '_captured_counters', {})
    with torch.inference_mode():
        pages = ops.KVPages.empty(2, 1, 8, 16)
        table, lens = torch.full((1, 1), 2, dtype=torch.int32, device='cuda'), torch.ones(1, dtype=torch.int32, device='cuda')
        ops.kv_append(pages, torch.ones(1, 1, 1, 16, device='cuda'), torch.ones(1, 1, 1, 16, device='cuda'), table, lens)
    with pytest.raises(RuntimeError, match='kv_append met page ids'):
        ops.page_fault_check()
    ops.page_fault_check()
    torch.cuda.synchronize()


@gpu
def test_captured_calls_beyond_the_cleared_counters(hip_lib, monkeypatch):
    """the last set that was cleared beforehand, then sets that the graph clears; replays between eager calls"""
    from openpvsg_amd import ops
    c = Cache(ops, [3000, 700, 1900], 2, 64, 16, torch.float32, 5)
    q = queries((3, 2, 4, 64), torch.float32, 5).cuda()
    eager = ops.paged_attention(q, c.pages, c.dev_table, c.dev_lens)
    spare, _ = ops._captured_counters[q.get_device()]
    last = torch.zeros(1024, dtype=torch.int32).cuda()               # (lives as long as the graph)
    monkeypatch.setitem(ops._captured_counters, q.get_device(), (spare, iter([last])))
    torch.cuda.synchronize()
    graph, outs = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        for _ in range(3):
            outs.append(ops.paged_attention(q, c.pages, c.dev_table, c.dev_lens))
    for _ in range(4):
        for o in outs:
            o.fill_(7.0)
        again = ops.paged_attention(q, c.pages, c.dev_table, c.dev_lens)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(bits(o), bits(eager)) for o in outs + [again])


@gpu
def test_another_stream(hip_lib):
    from openpvsg_amd import ops
    c = Cache(ops, [500, 3], 2, 64, 16, torch.bfloat16, 3)
    q = queries((2, 1, 4, 64), torch.bfloat16, 3).cuda()
    x = queries((2, 2, 2, 64), torch.bfloat16, 4).cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.kv_append(c.pages, x, x, c.dev_table, c.dev_lens)
        got = ops.paged_attention(q, c.pages, c.dev_table, c.dev_lens)
        k, _ = ops.kv_read(c.pages, c.dev_table, c.dev_lens, 500, dtype=torch.bfloat16)
    side.synchronize()
    assert torch.equal(bits(k[0, 498:500]), bits(x[0]))
    assert torch.equal(bits(got), bits(ops.paged_attention(q, c.pages, c.dev_table, c.dev_lens)))
    torch.cuda.synchronize()
