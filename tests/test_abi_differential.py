"""CPU checks of the differential attention entry points: bad arguments are
refused before a device is touched (null pointers throughout), and the lambdas
helper."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import proxy_attention_lab as pal
from proxy_attention_lab import _lib

DEFAULT = dict(kv=1, eps=1e-5, dtype=1, rows=64, seqs=64, hq=32, hkv=8, hd=128, tpp=16, pages=256, width=16, scales=None)


def decode(**kw):
    a = {**DEFAULT, **kw}
    return _lib.lib().pal_paged_differential_attention_decode(
        None, None, None, a["kv"], a["scales"], a["scales"], None, None, None, None, a["eps"], 1.0, None, a["dtype"],
        a["rows"], a["seqs"], a["hq"], a["hkv"], a["hd"], a["tpp"], a["pages"], a["width"], None, 0, None)


def chunk(**kw):
    a = {**DEFAULT, **kw}
    return _lib.lib().pal_paged_differential_attention(
        None, None, None, a["kv"], a["scales"], a["scales"], None, None, None, None, None, None, a["eps"], 1.0, None,
        a["dtype"], a["rows"], a["seqs"], a["hq"], a["hkv"], a["hd"], a["tpp"], a["pages"], a["width"], None, 0, None)


@pytest.mark.parametrize("call", [decode, chunk])
@pytest.mark.parametrize("bad,code,word", [
    (dict(dtype=2), "arg", "dtype"), (dict(kv=0), "arg", "queries' dtype or fp8"), (dict(kv=3), "arg", "fp8"),
    (dict(hq=0), "arg", "dimension"), (dict(pages=-1), "arg", "dimension"), (dict(width=-1), "arg", "dimension"),
    (dict(hq=30), "run", "divisible"), (dict(hq=35, hkv=7), "run", "even"), (dict(hd=80), "run", "head_dim 80"),
    (dict(hd=256), "run", "head_dim 256"), (dict(tpp=64), "run", "tokens_per_page"),
    (dict(kv=2), "arg", "scales"), (dict(kv=2, hd=96), "run", "fp8"), (dict(scales=16), "arg", "scales"),
    (dict(seqs=-1), "arg", "negative"), (dict(eps=-1.0), "arg", "norm_eps"), (dict(eps=float("nan")), "arg", "norm_eps"),
    (dict(width=2 ** 27), "arg", "too large"), (dict(rows=2 ** 31, seqs=2 ** 31), "arg", "too large"), (dict(), "arg", "null"),
])
def test_refused(call, bad, code, word):
    want = _lib.PAL_ERR_INVALID_ARGUMENT if code == "arg" else _lib.PAL_ERR_RUNTIME
    assert call(**bad) == want, _lib.last_error()
    assert word in _lib.last_error()


def test_rows_and_empty_calls():
    assert decode(rows=3) == _lib.PAL_ERR_INVALID_ARGUMENT and "query rows" in _lib.last_error()
    assert decode(seqs=0) == 0 and decode(rows=0, seqs=0) == 0 and chunk(rows=0) == 0


def test_workspace_size_of_bad_arguments():
    size = _lib.lib().pal_paged_differential_attention_workspace_size
    for args in ((2, 2, 64, 32, 8, 128, 16), (1, 0, 64, 32, 8, 128, 16), (1, 1, 0, 32, 8, 128, 16),
                 (1, 1, 64, 30, 8, 128, 16), (1, 1, 64, 35, 7, 128, 16), (1, 1, 64, 32, 8, 80, 16),
                 (1, 2, 64, 32, 8, 96, 16), (1, 1, 64, 32, 8, 128, 64), (1, 1, 2 ** 31, 32, 8, 128, 16)):
        assert size(*args) == 0


def test_operators_need_a_device():
    t = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        pal.paged_differential_attention_decode(t, t, t, i, i, t)
    with pytest.raises(ValueError, match="HIP device"):
        pal.paged_differential_attention(t, t, t, i, i, i, i, t)
    with pytest.raises(TypeError, match="torch.Tensor"):
        pal.paged_differential_attention_decode(None, t, t, i, i, t)


def test_lambda_on_the_host():
    v = [torch.linspace(-0.2, 0.2, 32) * (i + 1) for i in range(4)]
    lam = pal.differential_lambda(*v, 0.2, 4)
    want = np.exp(float(v[0].double() @ v[1].double())) - np.exp(float(v[2].double() @ v[3].double())) + 0.2
    assert lam.shape == (4,) and lam.dtype == torch.float32
    assert float((lam.double() - want).abs().max()) <= 2.0 ** -24 * abs(want)
