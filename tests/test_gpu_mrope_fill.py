"""GPU tests of mrope_fill_kv_pages: rotary positions of several axes, rotated,
cast and scattered in one pass.

Pools and rotated queries are compared bit for bit with an fp32 restatement
(each product rounded, then one rounding to the pool's type: the arithmetic the
operator documents) scattered by the oracle's fill, and with the formula in 64
bits: two rounded products, one rounded difference and the final cast, i.e.
2^-24 (2 (|x c| + |y s|)) + half a step of the type.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import proxy_attention_lab as pal
from gpu_util import DEV, announce, dev_bits, dev_index, host_bits
from oracle import pal_oracle as orc
from test_gpu_fp8_rope import TD, dev_f32, dev_pool, fill_layout, host_pool, src_values

pytestmark = pytest.mark.gpu


def axis_of(sections, interleaved: bool) -> list[int]:
    """Axis of every frequency, one by one from the definition."""
    out = []
    for f in range(sum(sections)):
        if interleaved:
            a = f % len(sections)
            out.append(a if f < len(sections) * sections[a] else 0)
        else:
            a = 0
            while f >= sum(sections[: a + 1]):
                a += 1
            out.append(a)
    return out


def turn(x, pos, table, sections, interleaved, style, dtype):
    """Rows x [N, H, HD] turned by positions [A, N], in dtype; tokens with a
    position outside the table unturned.  Also the sum of the products' sizes."""
    half = sum(sections)
    axis = axis_of(sections, interleaved)
    rows = table.shape[0]
    ok = ((pos >= 0) & (pos < rows)).all(0)
    p = np.where((pos >= 0) & (pos < rows), pos, 0)
    cos = np.stack([table[p[a], f] for f, a in enumerate(axis)], 1).astype(dtype)[:, None]
    sin = np.stack([table[p[a], half + f] for f, a in enumerate(axis)], 1).astype(dtype)[:, None]
    i = np.arange(half) if style == "neox" else 2 * np.arange(half)
    j = i + half if style == "neox" else i + 1
    x = x.astype(dtype)
    y, size = x.copy(), np.zeros_like(x)
    a, b = x[..., i], x[..., j]
    y[..., i] = a * cos - b * sin
    y[..., j] = b * cos + a * sin
    size[..., i] = np.abs(a * cos) + np.abs(b * sin)
    size[..., j] = np.abs(b * cos) + np.abs(a * sin)
    y[~ok], size[~ok] = x[~ok], 0
    return y, size, ok


def run_case(seed, hkv, hq, hd, tpp, src, kv, sections, interleaved, style, rot, rows=400, outside=False, chunks=None,
             stream=None):
    k, v, pt, pos, q2s, (ks, vs) = fill_layout(seed, hkv, hd, tpp, kv, **({"chunks": chunks} if chunks else {}))
    rng = np.random.default_rng(seed + 1)
    n = len(pos)
    nk, nv, q = (src_values(rng, (n, h, hd), src, 2.0) for h in (hkv, hkv, hq))
    rp = rng.integers(0, rows, size=(len(sections), n)).astype(np.int32)
    if outside:  # some tokens without a row on one axis: past the table, or negative
        rp[rng.integers(0, len(sections), n), np.arange(n)] = rng.choice([rows, rows + 7, -1, 5], n)
    table = pal.rope_cos_sin_cache(rows, rot, 10000.0, device=DEV)
    qdt = "f16" if kv == "f16" else "bf16"
    extra = {}
    if kv == "fp8":
        extra = dict(k_scales=torch.from_numpy(ks).to(DEV), v_scales=torch.from_numpy(vs).to(DEV))
    kd, vd = dev_pool(k, kv), dev_pool(v, kv)
    announce(f"mrope seed={seed} n={n} hd={hd} tpp={tpp} {src}->{kv} {sections} inter={interleaved} {style} rot={rot}")
    _, _, qo = pal.mrope_fill_kv_pages(dev_f32(nk, src), dev_f32(nv, src), kd, vd, dev_index(pt, torch.uint32),
                                       dev_index(pos), dev_index(q2s, torch.uint32), dev_index(rp), table, sections,
                                       stream, interleaved=interleaved, queries=dev_f32(q, src), rotary_dim=rot,
                                       style=style, query_dtype=TD[qdt], **extra)
    torch.cuda.synchronize()
    tab = table.cpu().numpy()
    k32, _, ok = turn(nk, rp, tab, sections, interleaved, style, np.float32)
    q32, _, _ = turn(q, rp, tab, sections, interleaved, style, np.float32)
    # tokens without a row are not written
    ek, ev, _ = orc.fill_kv_pages_ex(k32[ok], nv[ok], k, v, kv, pt, pos[ok], q2s[ok],
                                     k_scales=ks if kv == "fp8" else None, v_scales=vs if kv == "fp8" else None)
    assert np.array_equal(host_pool(kd, kv), ek), "K pool differs"
    assert np.array_equal(host_pool(vd, kv), ev), "V pool differs"
    assert np.array_equal(host_bits(qo), orc.f32_to_bits(q32, qdt)), "rotated queries differ"
    # the formula in 64 bits
    q64, size, _ = turn(q, rp, tab, sections, interleaved, style, np.float64)
    got = qo.double().cpu().numpy()
    step = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}[qdt]
    tiny = {"bf16": 2.0 ** -133, "f16": 2.0 ** -25}[qdt]  # half the smallest subnormal
    exact32 = 2 * 2.0 ** -24 * size
    assert (np.abs(got - q64) <= exact32 + step * (np.abs(q64) + exact32) + tiny).all()


@pytest.mark.parametrize("style", ["neox", "gptj"])
@pytest.mark.parametrize("src,kv", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "fp8"), ("bf16", "fp8"),
                                    ("f32", "f16")])
@pytest.mark.parametrize("sections,interleaved", [((16, 24, 24), False), ((24, 20, 20), True)])
def test_types_and_styles(style, src, kv, sections, interleaved):
    run_case(11, 4, 10 * 4, 128, 16, src, kv, sections, interleaved, style, 128)


@pytest.mark.parametrize("hd,rot,style,sections", [
    (32, 32, "neox", (4, 6, 6)), (32, 16, "neox", (8,)), (64, 32, "neox", (0, 16)), (64, 24, "gptj", (1, 4, 7)),
    (80, 48, "neox", (6, 6, 6, 6)), (96, 96, "gptj", (11, 17, 20)), (128, 64, "neox", (12, 10, 10)),
    (256, 256, "neox", (44, 42, 42)), (256, 64, "gptj", (32, 0, 0)), (200, 128, "gptj", (21, 1, 42)),
])
@pytest.mark.parametrize("src", ["f32", "bf16"])
def test_head_and_rotary_dims(hd, rot, style, sections, src):
    run_case(hd + rot, 2, 6, hd, 16, src, "bf16", sections, False, style, rot)


@pytest.mark.parametrize("sections", [(6, 5, 5), (16,), (8, 8), (4, 4, 4, 4), (16, 0, 0), (6, 4, 4, 2)])
def test_interleaved_sections(sections):
    run_case(sum(s * 7 ** i for i, s in enumerate(sections)), 2, 2, 32, 32, "f32", "bf16", sections, True, "neox", 32)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_positions_without_a_row(kv):
    run_case(5, 2, 4, 64, 16, "f32", kv, (12, 10, 10), True, "neox", 64, rows=40, outside=True)


@pytest.mark.parametrize("hd", [128, 256])
def test_prefill_sized_batch(hd):
    """Windows of 64 tokens (2,048 tokens and more)."""
    run_case(hd, 2, 8, hd, 16, "f32", "bf16", (hd // 8, hd // 8, hd // 4), False, "neox", hd,
             chunks=((0, 1500), (100, 700)))


@pytest.mark.parametrize("hq", [2, 14])
def test_one_token(hq):
    k, v, pt, pos, q2s, _ = fill_layout(1, 2, 64, 16, "bf16", n_decode=1, chunks=())
    assert len(pos) == 1
    run_case(1, 2, hq, 64, 16, "bf16", "bf16", (12, 10, 10), False, "neox", 64, chunks=((0, 1),))


def test_equal_positions_are_rope_fill():
    """The same position on every axis, equal to the write position: the bits of rope_fill_kv_pages."""
    k, v, pt, pos, q2s, _ = fill_layout(9, 4, 128, 16, "bf16")
    rng = np.random.default_rng(9)
    n = len(pos)
    nk, nv, q = (dev_f32(src_values(rng, (n, h, 128), "f32"), "f32") for h in (4, 4, 8))
    table = pal.rope_cos_sin_cache(512, 128, device=DEV)
    idx = (dev_index(pt, torch.uint32), dev_index(pos), dev_index(q2s, torch.uint32))
    a = (dev_bits(k, "bf16"), dev_bits(v, "bf16"))
    b = (dev_bits(k, "bf16"), dev_bits(v, "bf16"))
    announce("mrope with equal positions against rope")
    qa = pal.rope_fill_kv_pages(nk, nv, *a, *idx, table, queries=q)[2]
    # 64-bit positions, as a strided view
    wide = torch.stack([idx[1].long()] * 3).repeat_interleave(2, 1)[:, ::2]
    qb = pal.mrope_fill_kv_pages(nk, nv, *b, *idx, wide, table, (16, 24, 24), queries=q)[2]
    torch.cuda.synchronize()
    for x, y in ((a[0], b[0]), (a[1], b[1]), (qa, qb)):
        assert np.array_equal(host_bits(x), host_bits(y))


def test_no_tokens_and_no_queries():
    k, v, pt, pos, q2s, _ = fill_layout(4, 2, 64, 16, "bf16")
    table = pal.rope_cos_sin_cache(512, 64, device=DEV)
    kd, vd = dev_bits(k, "bf16"), dev_bits(v, "bf16")
    none = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=DEV)
    out = pal.mrope_fill_kv_pages(none, none, kd, vd, dev_index(pt), dev_index(pos[:0]), dev_index(q2s[:0]),
                                  torch.empty((3, 0), dtype=torch.int32, device=DEV), table, (12, 10, 10))
    assert out[0] is kd and out[1] is vd and out[2] is None
    assert np.array_equal(host_bits(kd), k) and np.array_equal(host_bits(vd), v)


def test_on_another_stream():
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    run_case(21, 2, 4, 64, 16, "f32", "bf16", (12, 10, 10), False, "neox", 64, stream=side)


def test_graph_replays():
    k, v, pt, pos, q2s, _ = fill_layout(31, 4, 128, 16, "bf16")
    rng = np.random.default_rng(31)
    n = len(pos)
    t = [dev_f32(src_values(rng, (n, h, 128), "f32"), "f32") for h in (4, 4, 8)]
    rp = dev_index(rng.integers(0, 512, (3, n)).astype(np.int32))
    table = pal.rope_cos_sin_cache(512, 128, device=DEV)
    idx = (dev_index(pt), dev_index(pos), dev_index(q2s))
    kd, vd = dev_bits(k, "bf16"), dev_bits(v, "bf16")

    def step(kp, vp):
        return pal.mrope_fill_kv_pages(t[0], t[1], kp, vp, *idx, rp, table, (16, 24, 24), queries=t[2])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kd, vd)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    announce("graph capture: mrope fill")
    with torch.cuda.graph(g, stream=side):
        out = step(kd, vd)
    for r in range(4):
        for x in t:
            x.copy_(torch.randn(x.shape, device=DEV))
        rp.copy_(torch.randint(0, 512, rp.shape, device=DEV))
        kd.zero_()
        vd.zero_()
        torch.cuda.synchronize()
        announce(f"graph replay {r}: mrope fill")
        g.replay()
        torch.cuda.synchronize()
        ke, ve = torch.zeros_like(kd), torch.zeros_like(vd)
        eager = step(ke, ve)
        torch.cuda.synchronize()
        for x, y in ((kd, ke), (vd, ve), (out[2], eager[2])):
            assert np.array_equal(host_bits(x), host_bits(y)), f"replay {r}"


def test_refusals():
    k, v, pt, pos, q2s, _ = fill_layout(2, 2, 64, 16, "bf16")
    n = len(pos)
    kd, vd = dev_bits(k, "bf16"), dev_bits(v, "bf16")
    new = torch.zeros((n, 2, 64), device=DEV)
    table = pal.rope_cos_sin_cache(512, 64, device=DEV)
    idx = (dev_index(pt), dev_index(pos), dev_index(q2s))

    def call(rp=None, sections=(12, 10, 10), tab=table, **kw):
        rp = torch.zeros((len(sections), n), dtype=torch.int32, device=DEV) if rp is None else rp
        return pal.mrope_fill_kv_pages(new, new, kd, vd, *idx, rp, tab, sections, **kw)

    for sections in ((12, 10, 9), (), (8, 8, 8, 4, 4), (40, -4, -4)):
        with pytest.raises(ValueError, match="sections"):
            call(sections=sections)
    for sections in ((8, 12, 12), (11, 12, 9)):  # every third of 32 frequencies from 1 on: 11
        with pytest.raises(ValueError, match="interleaved"):
            call(sections=sections, interleaved=True)
    with pytest.raises(ValueError, match="rotary_positions must be"):
        call(rp=torch.zeros((2, n), dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="integer"):
        call(rp=torch.zeros((3, n), device=DEV))
    with pytest.raises(ValueError, match="style"):
        call(style="none")
    with pytest.raises(ValueError, match="cos_sin_cache"):
        call(tab=table[:, :32])
    with pytest.raises(ValueError, match="queries"):
        call(queries=torch.zeros((n, 4, 64), dtype=torch.bfloat16, device=DEV))
    torch.cuda.synchronize()
    assert np.array_equal(host_bits(kd), k) and np.array_equal(host_bits(vd), v)
