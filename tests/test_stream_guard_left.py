"""The one-stream rule of openpvsg_amd/_lib.py after an external stream has been left."""


def test_nothing_is_kept_of_an_external_stream_that_was_left(monkeypatch):
    """back on one of torch's streams no launch of that device looks at events any more; other devices keep theirs"""
    from openpvsg_amd import _lib
    monkeypatch.setattr(_lib, '_torch_owned', {0})
    monkeypatch.setattr(_lib, '_external', {0: [0xdead0000, None], 1: [0xdead1000, None]})
    _lib._stream_taken(0, 0)
    assert _lib._external == {1: [0xdead1000, None]}


def test_leaving_an_external_stream_waits_for_what_others_put_there(monkeypatch):
    """its handle may be dead, so it is not asked; only 16-bit-MFMA kernels on either side make it matter"""
    import torch

    from openpvsg_amd import _lib
    waited = []
    monkeypatch.setattr(torch.cuda, 'synchronize', lambda d=None: waited.append(d))
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    monkeypatch.setattr(_lib, '_cur_dev', lambda: 3)
    monkeypatch.setattr(_lib, '_torch_owned', {0, 0x1000})
    monkeypatch.setattr(_lib, '_external', {})
    monkeypatch.setattr(_lib, '_stream_busy', lambda handle, dev=None: False)
    for name, prev, before, want in (('pvsg_gemm_bf16x3', 0xdead0000, False, [3]), ('pvsg_add_layernorm', 0xdead0000, True, [3]), ('pvsg_add_layernorm', 0xdead0000, False, []),
                                     ('pvsg_gemm_bf16x3', 0x1000, True, []), ('pvsg_gemm_bf16x3', None, False, [])):
        waited.clear()
        ent = [prev, before]
        _lib._stream_changed(name, 0, ent)
        assert waited == want and ent == [0, 'bf16x3' in name], (name, prev)
