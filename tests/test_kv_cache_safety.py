"""Paged cache: calls that must be reported or refused, or whose memory must stay what it was."""
import itertools
import random

import pytest
import torch

gpu = pytest.mark.gpu


def test_overlap_of_strided_rows_is_exact():
    """both statements against the rows written out, over random nested axes with and without gaps"""
    from openpvsg_amd import ops
    r = random.Random(1)
    met = touched = 0
    for _ in range(3000):
        size, axes, extent = r.choice((1, 2, 5)), [], 0
        extent = size
        for _ in range(r.randint(0, 3)):
            stride, n = extent + r.choice((0, 0, 1, 3, 9)), r.randint(2, 4)
            axes.insert(0, (stride, n))
            extent += stride * (n - 1)
        rows = [sum(i * s for i, (s, _) in zip(at, axes)) for at in itertools.product(*(range(n) for _, n in axes))]
        mine = {x + d for x in rows for d in range(size)}
        delta = r.randint(-extent - 3, extent + 3)
        want = bool(mine & {x + delta for x in mine})
        assert ops._rows_meet(delta, tuple(axes), size) == want, (delta, axes, size)
        lo = r.randint(-3, extent + 3)
        hi = lo + r.randint(1, 6)
        want_touch = bool({x + 100 for x in mine} & set(range(100 + lo, 100 + hi)))
        assert ops._rows_touch(100, tuple(axes), size, 100 + lo, 100 + hi) == want_touch, (lo, hi, axes, size)
        met, touched = met + want, touched + want_touch
    assert 300 < met < 2700 and 300 < touched < 2700


def test_a_pools_tensors_are_fixed():
    """a replaced tensor would be freed while the kernels go on writing to its address"""
    from openpvsg_amd import _lib, ops
    pages = ops.KVPages.__new__(ops.KVPages)
    pages.k = pages.v = torch.zeros(2, 1, 8, 16)                    # as in the making
    pages._struct = _lib.KvPages()
    for name in ('k', 'v', 'k_scale', 'num_pages', '_struct'):
        with pytest.raises(AttributeError, match='fixed'):
            setattr(pages, name, torch.ones(4, 1, 8, 16))
    with pytest.raises(AttributeError, match='fixed'):
        del pages.k
    assert pages.k.shape == (2, 1, 8, 16)


def test_a_subclass_keeps_attributes_of_its_own():
    from openpvsg_amd import _lib, ops

    class Video(ops.KVPages):
        pass
    pages = Video.__new__(Video)
    pages._struct = _lib.KvPages()
    pages.name = 'a'
    pages.name = 'b'
    assert pages.name == 'b'
    del pages.name
    with pytest.raises(AttributeError, match='fixed'):
        pages.k = None


def test_a_tangent_is_seen():
    from torch.autograd import forward_ad

    from openpvsg_amd import ops
    x = torch.randn(3)
    ops._refuse_tangent(x, 'x')
    with forward_ad.dual_level():
        ops._refuse_tangent(x, 'x')
        with pytest.raises(RuntimeError, match='x carries a forward-mode tangent'):
            ops._refuse_tangent(forward_ad.make_dual(x, torch.ones(3)), 'x')


@gpu
def test_a_fault_on_another_stream_is_reported(hip_lib):
    """the check runs on the default stream while the faulting call still waits in another one's queue"""
    from openpvsg_amd import ops
    pages = ops.KVPages.empty(4, 1, 8, 16)
    table, lens = torch.full((1, 1), 99, dtype=torch.int32, device='cuda'), torch.ones(1, dtype=torch.int32, device='cuda')
    x = torch.ones(1, 1, 1, 16, device='cuda')
    ops.page_fault_check()
    side = torch.cuda.Stream()
    busy = torch.ones(1 << 26, device='cuda')
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(50):
            busy.mul_(1.0)                                          # 50 passes over 256 MB: some milliseconds
        ops.kv_append(pages, x, x, table, lens)
    with pytest.raises(RuntimeError, match='kv_append met'):
        ops.page_fault_check()
    ops.page_fault_check()                                          # reported once
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize('dtype', (torch.float32, torch.int8), ids=str)
def test_pools_that_share_memory(hip_lib, dtype):
    """k and v a page, a slot or half a row apart are not appended to; interleaved ones, which share none, are"""
    from openpvsg_amd import ops
    P, H, S, D = 6, 2, 8, 32
    table, lens, x = torch.arange(4, dtype=torch.int32, device='cuda').view(1, 4), torch.tensor([9], dtype=torch.int32, device='cuda'), torch.randn(1, 9, H, D, device='cuda')
    scales = [torch.zeros(P, H, S, device='cuda') for _ in range(2)] if dtype == torch.int8 else []
    flat = torch.zeros(4 * P * H * S * D, dtype=dtype, device='cuda')
    for apart in (0, 16, D, S * D, H * S * D, (P - 1) * H * S * D):
        k, v = (flat[at:at + P * H * S * D].view(P, H, S, D) for at in (0, apart))
        with pytest.raises(RuntimeError, match='same memory'):
            ops.kv_append(ops.KVPages(k, v, *scales), x, x, table, lens)
    if scales:
        both = torch.zeros(P * H * S + 16, device='cuda')
        a, b = both[:P * H * S].view(P, H, S), both[16:].view(P, H, S)
        with pytest.raises(RuntimeError, match='same memory'):
            ops.kv_append(ops.KVPages(flat[:P * H * S * D].view(P, H, S, D), flat[P * H * S * D:2 * P * H * S * D].view(P, H, S, D), a, b), x, x, table, lens)
        with pytest.raises(RuntimeError, match='same memory'):       # a scale inside the codes
            ops.kv_append(ops.KVPages(flat[:P * H * S * D].view(P, H, S, D), flat[P * H * S * D:2 * P * H * S * D].view(P, H, S, D),
                                      flat[:P * H * S * 4].view(torch.float32).view(P, H, S), scales[1]), x, x, table, lens)
    for split in (flat[:2 * P * H * S * D].view(P, 2, H, S, D).unbind(1), flat[:2 * P * H * S * D].view(P, H, S, 2, D).unbind(3),
                  flat[:2 * P * H * S * D].view(P, H, S, 2 * D).chunk(2, 3)):
        pages = ops.KVPages(*split, *scales)
        ops.kv_append(pages, x, 2 * x, table, lens)
        k, v = ops.kv_read(pages, table, lens, 9)
        assert float((v - 2 * k).abs().max()) <= 1e-6 and float((k - x).abs().max()) <= (0.0 if dtype == torch.float32 else 0.03)
    torch.cuda.synchronize()


@gpu
def test_rows_that_lie_in_the_pool_count_as_they_were(hip_lib):
    """a sequence's rows moved by one slot, within its own pages: each of them is read before any is written"""
    from openpvsg_amd import ops
    P, H, S, D = 8, 2, 16, 64
    for dtype in (torch.float32, torch.bfloat16):
        pages = ops.KVPages.empty(P, H, S, D, dtype=dtype)
        table = torch.arange(P, dtype=torch.int32, device='cuda').view(P, 1)
        pages.k.copy_(torch.randn(P, H, S, D, device='cuda')), pages.v.copy_(torch.randn(P, H, S, D, device='cuda'))
        k, v = pages.k.clone(), pages.v.clone()
        lens = torch.full((P,), S, dtype=torch.int32, device='cuda')
        ops.kv_append(pages, pages.k.transpose(1, 2)[:, :-1], pages.v.transpose(1, 2)[:, :-1], table, lens)
        for now, was in ((pages.k, k), (pages.v, v)):
            assert torch.equal(now[:, :, 1:], was[:, :, :-1]) and torch.equal(now[:, :, 0], was[:, :, 0])
        # both tensors from the same one's pages
        ops.kv_append(pages, pages.v.transpose(1, 2)[:, :4], pages.v.transpose(1, 2)[:, :4], table, lens)
        assert torch.equal(pages.k[:, :, -4:], pages.v[:, :, -4:]) and torch.equal(pages.k[:, :, 1:12], k[:, :, :11])
    torch.cuda.synchronize()


@gpu
def test_out_may_not_lie_in_an_input(hip_lib):
    from openpvsg_amd import ops
    P, H, S, D = 6, 2, 8, 32
    arena = torch.zeros(P, 3, H, S, D, device='cuda')
    pages = ops.KVPages(arena[:, 0], arena[:, 1])
    ints = torch.zeros(4 * 2 * H * D, dtype=torch.int32, device='cuda')
    lens, q = torch.full((4,), 8, dtype=torch.int32, device='cuda'), torch.randn(4, 1, 2 * H, D, device='cuda')
    table = torch.arange(4, dtype=torch.int32, device='cuda').view(4, 1)
    mask = torch.zeros(4, 8, dtype=torch.bool, device='cuda')
    n = q.numel()
    want = ops.paged_attention(q, pages, table, lens, key_padding_mask=mask)
    for out in (arena.view(-1)[:n], arena[3, 1].reshape(-1)[:n], arena.view(-1)[H * S * D * 5 - 16:][:n]):
        with pytest.raises(RuntimeError, match='out overlaps the pool'):
            ops.paged_attention(q, pages, table, lens, out=out.view(q.shape))
    as_float = ints.view(torch.float32)
    for kw in (dict(table=ints[:4].view(4, 1)), dict(lens=ints[-4:]), dict(new_lens=ints[:4]), dict(key_padding_mask=ints.view(torch.bool)[:32].view(4, 8))):
        with pytest.raises(RuntimeError, match='out overlaps the pool'):
            ops.paged_attention(q, pages, kw.pop('table', table), kw.pop('lens', lens), out=as_float[:n].view(q.shape), **kw)
    out = arena[2, 2].reshape(-1)[:n].view(q.shape)                  # between the pool's rows
    assert out.data_ptr() == arena[2, 2].data_ptr()
    assert ops.paged_attention(q, pages, table, lens, key_padding_mask=mask, out=out) is out and torch.equal(out, want)
    torch.cuda.synchronize()


@gpu
def test_derivatives_are_refused(hip_lib):
    """rows, pools and scales whose gradient or tangent would be dropped"""
    from torch.autograd import forward_ad

    from openpvsg_amd import ops
    pages = ops.KVPages.empty(4, 2, 8, 32)
    table, lens = torch.arange(4, dtype=torch.int32, device='cuda').view(2, 2), torch.full((2,), 3, dtype=torch.int32, device='cuda')
    x, q = torch.ones(2, 3, 2, 32, device='cuda'), torch.ones(2, 3, 4, 32, device='cuda')
    code, scale = torch.zeros(4, 2, 8, 32, dtype=torch.int8, device='cuda'), torch.ones(4, 2, 8, device='cuda')
    ops.kv_append(pages, x, x, table, lens)
    with pytest.raises(RuntimeError, match='k_scale requires a gradient'):
        ops.KVPages(code, code.clone(), scale.clone().requires_grad_(), scale)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.kv_append(pages, dual(x), x, table, lens), lambda: ops.kv_append(pages, x, dual(x), table, lens),
                     lambda: ops.paged_attention(dual(q), pages, table, lens), lambda: ops.KVPages(dual(pages.k), pages.v),
                     lambda: ops.KVPages(code, code.clone(), dual(scale), scale)):
            with pytest.raises(RuntimeError, match='forward-mode tangent'):
                call()
        ops.paged_attention(q, pages, table, lens)                   # without one: as ever
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: ops.paged_attention(t, pages, table, lens), (q,), (q,))
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize('dtype', (torch.float32, torch.int8), ids=str)
def test_writes_raise_the_version_counters(hip_lib, dtype):
    """a backward pass that saved a tensor of the pool, or an `out`, stops instead of running on what was written since"""
    from openpvsg_amd import ops
    pages = ops.KVPages.empty(4, 2, 8, 32, dtype=dtype)
    table, lens = torch.arange(4, dtype=torch.int32, device='cuda').view(2, 2), torch.full((2,), 3, dtype=torch.int32, device='cuda')
    x, q = torch.ones(2, 3, 2, 32, device='cuda'), torch.ones(2, 3, 4, 32, device='cuda')
    written = [t for t in (pages.k, pages.v, pages.k_scale, pages.v_scale) if t is not None]
    before = [t._version for t in written]
    ops.kv_append(pages, x, x, table, lens)
    assert all(t._version > n for t, n in zip(written, before))
    before = [t._version for t in written]
    out = torch.empty_like(q)
    n = out._version
    ops.kv_read(pages, table, lens, 3), ops.paged_attention(q, pages, table, lens, out=out)
    assert [t._version for t in written] == before and out._version > n
    w = torch.ones(32, device='cuda', requires_grad=True)
    saved = written[-1] if dtype == torch.int8 else pages.v
    loss = (saved * (w.sum() if dtype == torch.int8 else w)).sum()
    ops.kv_append(pages, x, x, table, lens)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    with torch.inference_mode():                                     # tensors that have no counter
        ops.kv_append(ops.KVPages.empty(4, 2, 8, 32, dtype=dtype), x, x, table, lens)
        ops.paged_attention(q, pages, table, lens, out=torch.empty_like(q))
    torch.cuda.synchronize()
