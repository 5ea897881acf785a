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
