"""The weights of paged_attention (csrc/paged_attention.h) where their bits show: a dominant key whose value is zero, so that the
result is made of small weights alone."""
import pytest
import torch

from .test_kv_cache import Cache

gpu = pytest.mark.gpu


def by_weight(q, k, v, scale):
    """one row q (D,) over its keys k, v (n, D), all in 64 bits -> the result, sum w |v| / sum w, sum |v| / sum w, and how far the f32
    statistics may be off, relative to the second (D products and their sums, twice; exp2; the sums over the keys)"""
    z = (k @ q) * scale
    w = torch.exp(z - z.max())
    dz = (q.shape[0] + 6) * 2.0 ** -24 * float((k.abs() @ q.abs()).max()) * scale
    return (w / w.sum()) @ v, w @ v.abs() / w.sum(), v.abs().sum(0) / w.sum(), 2 * dz + (z.shape[0] + 16) * 2.0 ** -24 + 2.0 ** -22


@gpu
@pytest.mark.parametrize('above', (13.0, 16.0, 17.0, 20.0))
@pytest.mark.parametrize('D', (64, 128))
def test_small_f16_weights_behind_a_dominant_key(hip_lib, D, above):
    """f16 rows over a f16 pool, caches that are split and that are not, two query heads a key head, two new tokens; the dominant key at
    the start, in the middle and near the end, `above` the others' logits"""
    from openpvsg_amd import ops
    lens, H, G, T = [900, 6000, 2300, 40], 2, 2, 2
    c = Cache(ops, lens, H, D, 16, torch.float16, int(above))
    g = torch.Generator().manual_seed(D)
    q = torch.randn((len(lens), 1, H, 1, D), generator=g) * torch.tensor([1.0, 0.875]).view(1, 1, 1, 2, 1)
    q = q.expand(-1, T, -1, -1, -1).reshape(len(lens), T, H * G, D).half()
    rows = []
    for b, n in enumerate(lens):
        k = 0.02 * torch.randn((n, H, D), generator=g)
        v = 50.0 * (1.0 + torch.rand((n, H, D), generator=g)) * torch.where(torch.rand((1, H, D), generator=g) < 0.5, -1.0, 1.0)
        at = (0, n // 2, n - 3, 5)[b]
        first = q[b, 0, ::G].float()
        k[at] = first * (above * D ** 0.5 / first.square().sum(-1, keepdim=True))
        v[at] = 0.0
        k, v = k.half(), v.half()
        p = torch.arange(n)
        page = c.table[b, p // 16].long()
        c.pages.k[page.cuda(), :, (p % 16).cuda()], c.pages.v[page.cuda(), :, (p % 16).cuda()] = k.cuda(), v.cuda()
        rows.append((k.double(), v.double()))
    got = ops.paged_attention(q.cuda(), c.pages, c.dev_table, c.dev_lens).cpu().double()
    for b, n in enumerate(lens):
        for t in range(T):
            for j in range(H * G):
                k, v = rows[b][0][:n - T + 1 + t, j // G], rows[b][1][:n - T + 1 + t, j // G]
                want, size, every, rel = by_weight(q[b, t, j].double(), k, v, D ** -0.5)
                # a weight in two f16 parts of 2^15 times it: 2^-22 of itself, 2^-40 of the largest below 2^-29; one rounding of the result
                tol = (rel + 2.0 ** -22) * size + 2.0 ** -40 * every + torch.finfo(torch.float16).eps / 2 * want.abs() + 2.0 ** -25
                err = (got[b, t, j] - want).abs()
                assert bool((err <= tol).all()), (b, t, j, 'worst %.3g of its tolerance' % float((err / tol).max()))


def cancelling(n, H, D, pool, g):
    """n keys whose weights are known to a few units of f32 (one column of k, the rest zero; exact logits in [-1, 0]) and values that
    cancel under them: the last keys' take back what the ones before leave, so what is left of a result is the weights' own error"""
    z = -(torch.randint(0, 17, (n, H), generator=g) / 16.0)
    z[0] = 0.0
    w = torch.exp(z.double())
    v = torch.where(torch.rand((n, H, D), generator=g) < 0.5, -1.0, 1.0) * (1.0 + torch.randint(0, 8, (n, H, D), generator=g) / 8.0)
    scaled = pool == torch.float8_e4m3fn
    scale = torch.ones(n, H)
    for i in range(n - (6 if scaled else 3), n):
        left = -(w[:i, :, None] * v[:i].double() * scale[:i, :, None]).sum(0) / w[i, :, None]
        if scaled:
            scale[i] = 2.0 ** torch.ceil(torch.log2(left.abs().amax(-1))).float() / 256.0
        v[i] = (left / scale[i, :, None]).float().to(pool).float()
    k = torch.zeros(n, H, D)
    k[..., 0] = z
    return k, v, scale, w


@gpu
@pytest.mark.parametrize('row,pool', ((torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float8_e4m3fn), (torch.float16, torch.float8_e4m3fn),
                                      (torch.float16, torch.float16), (torch.float32, torch.bfloat16)), ids=lambda t: str(t)[6:])
def test_weights_hold_the_bits_of_f32(hip_lib, row, pool):
    from openpvsg_amd import ops
    B, n, H, D = 60, 12, 4, 16
    c = Cache(ops, [n] * B, H, D, 16, pool, 1)
    g = torch.Generator().manual_seed(3)
    per = [cancelling(n, H, D, pool, g) for _ in range(B)]
    at = c.table[:, 0].long().cuda()

    def put(codes, x):
        x = x.transpose(1, 2).to(pool)
        if pool == torch.float8_e4m3fn:
            codes, x = codes.view(torch.uint8), x.view(torch.uint8)
        codes[at, :, :n] = x.cuda()
    put(c.pages.k, torch.stack([p[0] for p in per]))
    put(c.pages.v, torch.stack([p[1] for p in per]))
    if pool == torch.float8_e4m3fn:
        c.pages.k_scale[at, :, :n] = 1.0
        c.pages.v_scale[at, :, :n] = torch.stack([p[2] for p in per]).transpose(1, 2).cuda()
    q = torch.zeros(B, 1, H, D, dtype=row)
    q[..., 0] = 1.0
    got = ops.paged_attention(q.cuda(), c.pages, c.dev_table, c.dev_lens, scale=1.0).cpu().double()[:, 0]
    for b, (k, v, scale, w) in enumerate(per):
        x = v.double() * scale.double()[..., None]
        want = (w[..., None] * x).sum(0) / w.sum(0)[:, None]
        # what f32 gives: z * log2(e) and its rounding, |z| <= 1: 3 * 2^-24; exp2 2^-23; three parts or two of f16 2^-22; the product with a scale
        # 2^-24; the sums over at most 16 keys, three parts each, and over the four waves: 16 * 2^-24.  One rounding of the result.
        tol = 26 * 2.0 ** -24 * (w[..., None] * x.abs()).sum(0) / w.sum(0)[:, None] + torch.finfo(row).eps / 2 * want.abs() + (2.0 ** -25 if row == torch.float16 else 0.0)
        err = (got[b] - want).abs()
        assert bool((err <= tol).all()), (b, 'worst %.3g of its tolerance' % float((err / tol).max()))


@gpu
@pytest.mark.parametrize('row,pool', ((torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                      (torch.bfloat16, torch.float8_e4m3fn)), ids=lambda t: str(t)[6:])
@pytest.mark.parametrize('D', (16, 64))
def test_logits_of_minus_infinity(hip_lib, row, pool, D):
    """a row that sees only those is zero, split or not; beside finite ones they have no weight; one of +infinity makes the row NaN"""
    from openpvsg_amd import ops
    inf = float('inf')
    for n in (1, 70, 5000):
        c = Cache(ops, [n] * 4, 1, D, 16, pool, n)
        q = torch.ones(4, 1, 1, D, dtype=row)
        p = torch.arange(n)

        def put(b, where, x):
            page, slot = c.table[b, where // 16].long().cuda(), (where % 16).cuda()
            if pool == torch.float8_e4m3fn:
                c.pages.k.view(torch.uint8)[page, :, slot] = torch.full((1, D), 1.0).to(pool).view(torch.uint8).cuda()
                c.pages.k_scale[page, :, slot] = x
            else:
                c.pages.k[page, :, slot] = x
        put(0, p, -inf)
        put(1, p[:n // 2], -inf)
        put(2, p, -inf)
        put(2, p[n // 3:n // 3 + 1], inf)
        got = ops.paged_attention(q.cuda(), c.pages, c.dev_table, c.dev_lens).cpu().double()
        assert not bool(got[0].any())
        assert bool(got[2].isnan().all())
        for b, first in ((1, n // 2), (3, 0)):
            want, size, every, rel = by_weight(q[b, 0, 0].double(), c.rows[0][b][first:, 0], c.rows[1][b][first:, 0], D ** -0.5)
            tol = (rel + 2.0 ** -22) * size + 2.0 ** -40 * every + torch.finfo(row).eps / 2 * want.abs() + (2.0 ** -25 if row == torch.float16 else 0.0)
            assert bool(((got[b, 0, 0] - want).abs() <= tol).all()), (n, b)


@gpu
@pytest.mark.parametrize('row,pool', ((torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)), ids=lambda t: str(t)[6:])
def test_logits_past_what_f32_counts_by_ones(hip_lib, row, pool):
    """logits of some 10^7, far apart: the largest key alone, also where f32 cannot hold the maximum less a small number"""
    from openpvsg_amd import ops
    D = 64
    for n in (5, 300, 3000):
        c = Cache(ops, [n], 1, D, 16, pool, n)
        p = torch.arange(n)
        page, slot = c.table[0, p // 16].long().cuda(), (p % 16).cuda()
        size = torch.full((n,), 1000.0)
        best = torch.randint(0, n, (1,), generator=c.g)
        size[best] = 2048.0
        c.pages.k[page, :, slot] = (size[:, None, None] * torch.ones(n, 1, D)).to(pool).cuda()
        q = torch.full((1, 2, 1, D), 2048.0, dtype=row)
        got = ops.paged_attention(q.cuda(), c.pages, c.dev_table, c.dev_lens, causal=False).cpu()
        # every other weight is exp(-1e7) = 0, the largest 1: the value itself
        assert torch.equal(got.double(), c.rows[1][0][best].expand(2, 1, D)[None].reshape(1, 2, 1, D)), n
