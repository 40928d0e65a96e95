"""CPU checks of pal_mrope_fill_kv_pages: bad arguments are refused before a
device is touched (null pointers throughout, so a launch could not pass)."""

from __future__ import annotations

import ctypes

import pytest

from proxy_attention_lab import _lib


def call(sections=(12, 10, 10), axes=None, interleaved=0, tokens=4, hkv=2, hd=64, rot=64, style=1, rows=16, src=3, kv=1):
    counts = (ctypes.c_int * len(sections))(*sections) if sections is not None else None
    n = (len(sections) if sections is not None else 3) if axes is None else axes
    return _lib.lib().pal_mrope_fill_kv_pages(None, None, src, None, None, kv, None, None, None, None, None, tokens, hkv,
                                              hd, 16, 8, 1, 1, None, n, counts, interleaved, None, rows, rot, style, None,
                                              None, 0, 1, None)


@pytest.mark.parametrize("bad,word", [
    (dict(sections=(12, 10, 9)), "sum"), (dict(sections=(12, 10, 11)), "sum"), (dict(sections=(40, -4, -4)), "negative"),
    (dict(sections=(8, 8, 8, 4, 4)), "axes"), (dict(axes=0), "axes"), (dict(sections=None), "axes"),
    (dict(sections=(8, 12, 12), interleaved=1), "no room"), (dict(sections=(2 ** 31 - 1, 2 ** 31 - 1, 34)), "sum"),
    (dict(style=0), "rope_style"), (dict(style=3), "rope_style"), (dict(rot=24), "rotary_dim"),
    (dict(rot=128), "rotary_dim"), (dict(hd=60), "multiple"), (dict(hd=264), "head_dim"), (dict(src=2), "source"),
    (dict(kv=3), "pool dtype"), (dict(rows=-1), "table"), (dict(), "table"),
])
def test_refused(bad, word):
    assert call(**bad) == _lib.PAL_ERR_INVALID_ARGUMENT
    assert word in _lib.last_error() and "[mrope_fill_kv_pages]" in _lib.last_error()


def test_no_tokens_is_a_no_op():
    assert call(tokens=0) == 0
    assert call(tokens=0, sections=(12, 10, 10), interleaved=1) == 0
    assert call(tokens=0, sections=(11, 11, 10), interleaved=1) == 0  # every third of 32: 11, 11, 10
