"""Paged cache: calls that must be reported or refused, or whose memory must stay what it was."""
import pytest
import torch

gpu = pytest.mark.gpu


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
