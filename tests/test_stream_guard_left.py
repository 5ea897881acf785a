"""The one-stream rule of openpvsg_amd/_lib.py after an external stream has been left."""


def test_nothing_is_kept_of_an_external_stream_that_was_left(monkeypatch):
    """back on one of torch's streams no launch of that device looks at events any more; other devices keep theirs"""
    from openpvsg_amd import _lib
    monkeypatch.setattr(_lib, '_torch_owned', {0})
    monkeypatch.setattr(_lib, '_external', {0: [0xdead0000, None], 1: [0xdead1000, None]})
    _lib._stream_taken(0, 0)
    assert _lib._external == {1: [0xdead1000, None]}
