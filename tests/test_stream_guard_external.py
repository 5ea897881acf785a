"""Streams that torch was handed (ExternalStream) and the one-stream rule of openpvsg_amd/_lib.py: a handle that may be destroyed is
never given to the runtime, and a live one that is busy is still seen."""
import ctypes

import pytest
import torch


def test_a_handle_that_is_not_torchs_is_not_asked_about(monkeypatch):
    """the previous stream of a device, destroyed since: querying it would read freed memory (no GPU needed to see it)"""
    from openpvsg_amd import _lib

    class Runtime:
        asked = []

        def hipStreamQuery(self, handle):
            self.asked.append(handle.value)
            return 600

    monkeypatch.setattr(_lib, '_hip', Runtime())
    monkeypatch.setattr(_lib, '_external', {})
    assert _lib._stream_busy(0xdead0000, dev=0) is False and Runtime.asked == []
    monkeypatch.setattr(_lib, '_torch_owned', {0, 0x1000})
    assert _lib._stream_busy(0x1000, dev=0) is True and Runtime.asked == [0x1000]


@pytest.mark.gpu
def test_a_busy_external_stream_is_seen_and_a_destroyed_one_is_idle(hip_lib):
    from openpvsg_amd import _lib, ops
    g = torch.Generator().manual_seed(1)
    a = torch.randn(200000, 256, generator=g).cuda()
    wp = ops.gemm_bf16x3_pack(torch.randn(1024, 256, generator=g).cuda())
    out = torch.empty(200000, 1024, device='cuda')
    torch.cuda.synchronize()
    hip = ctypes.CDLL('libamdhip64.so')
    stream = ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(stream), 1) == 0          # not a blocking one: the default stream's query waits for those
    with torch.cuda.stream(torch.cuda.ExternalStream(stream.value)):
        for _ in range(20):
            ops.gemm_bf16x3(a, wp, 1024, out=out)
    with pytest.raises(_lib.ConcurrentStreamError):
        ops.gemm_bf16x3(a[:1000], wp, 1024)
    torch.cuda.synchronize()
    want = ops.gemm_bf16x3(a[:1000], wp, 1024)                     # idle: handed over
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(stream.value)):
        ops.gemm_bf16x3(a[:1000], wp, 1024)
    torch.cuda.synchronize()
    assert hip.hipStreamDestroy(stream) == 0
    assert torch.equal(ops.gemm_bf16x3(a[:1000], wp, 1024), want)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_a_busy_pool_stream_is_seen(hip_lib):
    from openpvsg_amd import _lib, ops
    a = torch.randn(200000, 256, device='cuda')
    wp = ops.gemm_bf16x3_pack(torch.randn(1024, 256, device='cuda'))
    out = torch.empty(200000, 1024, device='cuda')
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(20):
            ops.gemm_bf16x3(a, wp, 1024, out=out)
    with pytest.raises(_lib.ConcurrentStreamError):
        ops.gemm_bf16x3(a[:1000], wp, 1024)
    torch.cuda.synchronize()
