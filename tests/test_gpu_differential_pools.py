"""Differential attention and the several-axes RoPE fill over pools of more than
4 GiB, and in the bounds-checked library (libpal_hip_debug.so)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import proxy_attention_lab as pal
from diff_cases import Diff, chunk_case, decode_case
from gpu_util import DEV, announce, dev_index, host_bits
from proxy_attention_lab import _lib
from test_gpu_debug_checks import _flags, dbg  # noqa: F401  (dbg: a fixture)
from test_gpu_fp8_rope import dev_f32, dev_pool, fill_layout, host_pool, src_values
from test_gpu_large_pool import _base, _big, _shifted

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _release_pools():
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("chunk,hd,tpp", [(False, 128, 16), (False, 64, 32), (True, 128, 16), (True, 64, 32)])
def test_pages_past_4_gib(chunk, hd, tpp, fp8):
    lens = [1, 17, 300, 2049, 0, 16]
    d = chunk_case(50, lens[:4], [(0, 70), (130, 64), (900, 129)], 16, 8, hd, tpp, "bf16", fp8=fp8) if chunk else \
        decode_case(50, lens, 16, 8, hd, tpp, "bf16", fp8=fp8)
    base = _base(d.kc if fp8 else d.case.k_pool)
    announce(f"differential attention past 4 GiB, chunk={chunk} hd={hd} fp8={fp8} base page {base}")
    for name in ("k", "v", "ks", "vs") if fp8 else ("k", "v"):
        d.dev[name] = _big(d.dev[name], base)
    d.dev["pt"] = _shifted(d.case.page_table, base)
    out = d.run()
    torch.cuda.synchronize()
    d.check(out, "pages past 4 GiB")


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_mrope_fill_past_4_gib(kv):
    hkv, hd, tpp, sections = 8, 128, 16, [16, 24, 24]
    k, v, pt, pos, q2s, (ks, vs) = fill_layout(51, hkv, hd, tpp, kv)
    rng = np.random.default_rng(51)
    n = len(pos)
    nk, nv, q = (dev_f32(src_values(rng, (n, h, hd), "f32", 2.0), "f32") for h in (hkv, hkv, 16))
    rp = dev_index(rng.integers(0, 300, (3, n)).astype(np.int32))
    table = pal.rope_cos_sin_cache(300, hd, 10000.0, device=DEV)
    base = _base(k)
    small = [dev_pool(k, kv), dev_pool(v, kv)]
    big = [_big(t, base) for t in small]
    scales = [torch.from_numpy(ks).to(DEV), torch.from_numpy(vs).to(DEV)] if kv == "fp8" else []
    got = []
    for pools, sc, table_of in ((small, scales, dev_index(pt, torch.uint32)),
                                (big, [_big(t, base) for t in scales], _shifted(pt, base))):
        announce(f"mrope fill {kv}, {pools[0].shape[0]} pages")
        extra = dict(k_scales=sc[0], v_scales=sc[1]) if sc else {}
        _, _, qo = pal.mrope_fill_kv_pages(nk, nv, *pools, table_of, dev_index(pos), dev_index(q2s, torch.uint32), rp,
                                           table, sections, queries=q, **extra)
        torch.cuda.synchronize()
        first = pools[0].shape[0] - k.shape[0]
        got.append([host_pool(t[first:].contiguous(), kv) for t in pools] + [host_bits(qo.to(torch.bfloat16))])
    for a, b in zip(*got):
        assert np.array_equal(a, b)


def _checked(lib, d: Diff) -> torch.Tensor:
    """One call of the bounds-checked library."""
    x, c = d.dev, d.case
    rows = x["q"].shape[0]
    code = _lib.DTYPE_BFLOAT16 if c.dtype == "bf16" else _lib.DTYPE_FLOAT16
    kv = _lib.DTYPE_FP8_E4M3 if d.fp8 else code
    dims = (c.num_q_heads, c.num_kv_heads, c.head_dim, c.tokens_per_page)
    out = torch.empty((rows, c.num_q_heads // 2, 2 * c.head_dim), dtype=x["q"].dtype, device=DEV)
    nbytes = lib.pal_paged_differential_attention_workspace_size(code, kv, rows, *dims)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    rows_of = () if d.q2s is None else (p(x["q2s"]), p(x["off"]))
    entry = lib.pal_paged_differential_attention_decode if d.q2s is None else lib.pal_paged_differential_attention
    torch.cuda.synchronize()
    st = entry(p(x["q"]), p(x["k"]), p(x["v"]), kv, p(x["ks"]), p(x["vs"]), p(x["pt"]), p(x["lens"]), *rows_of,
               p(x["lam"]), p(x["w"]), d.eps, d.out_scale, p(out), code, rows, c.page_table.shape[0], *dims,
               x["k"].shape[0], c.page_table.shape[1], p(ws), nbytes, torch.cuda.current_stream().cuda_stream)
    assert st == 0, lib.pal_last_error()
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("chunk", [False, True])
def test_checked_library(dbg, chunk, fp8):  # noqa: F811
    """No flag on a sound call, whose results are the release library's; a flag for a bad page id and length."""
    d = chunk_case(52, [40, 600], [(100, 200), (0, 33)], 8, 4, 64, 16, "bf16", fp8=fp8) if chunk else \
        decode_case(52, [40, 600, 17], 8, 4, 64, 16, "bf16", fp8=fp8)
    announce(f"checked differential attention chunk={chunk} fp8={fp8}")
    _flags(dbg)
    got = host_bits(_checked(dbg, d))
    assert _flags(dbg) == 0
    assert np.array_equal(got, host_bits(d.run()))
    pt = d.case.page_table.copy()
    d.case.page_table[0, 1] = d.case.k_pool.shape[0] + 3
    d.dev["pt"] = dev_index(d.case.page_table, torch.uint32)
    _checked(dbg, d)
    assert _flags(dbg) & 1
    d.dev["pt"] = dev_index(pt, torch.uint32)
    d.dev["lens"] = dev_index(d.case.seq_lens + d.case.page_table.shape[1] * 16)
    if chunk:
        d.dev["off"] = dev_index(d.off + d.case.page_table.shape[1] * 16)
    _checked(dbg, d)
    assert _flags(dbg) & 2
