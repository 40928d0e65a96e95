"""GPU tests of paged_differential_attention_decode and
paged_differential_attention against the definition in 64 bits (diff_cases.py,
which derives the bounds)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import proxy_attention_lab as pal
from diff_cases import Diff, chunk_case, decode_case
from gpu_util import DEV, announce, dev_bits, dev_index, host_bits
from oracle import pal_oracle as orc
from pal_cases import make_paged_case, randn_bits

pytestmark = pytest.mark.gpu

RAGGED = [1, 0, 15, 16, 17, 33, 300, 64, 127, 2]
GROUPS = [(2, 2), (8, 2), (10, 2), (16, 2), (40, 2), (24, 4), (4, 4)]


def run(d: Diff, what: str, norm2=True):
    announce(what)
    out = d.run()
    torch.cuda.synchronize()
    d.check(out, what, norm2)
    return out


# ---------------------------------------------------------------------------
# one row per sequence
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tpp", [16, 32])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_decode_head_dims(hd, tpp, dtype):
    run(decode_case(hd + tpp, RAGGED, 8, 4, hd, tpp, dtype), f"decode hd={hd} tpp={tpp} {dtype}")


@pytest.mark.parametrize("hq,hkv", GROUPS)
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_groups(hq, hkv, fp8):
    run(decode_case(hq * 10 + hkv, RAGGED, hq, hkv, 64, 16, "bf16", fp8=fp8), f"decode {hq}/{hkv} fp8={fp8}")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tpp", [16, 32])
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_fp8(hd, tpp, dtype):
    run(decode_case(hd + tpp + 1, RAGGED, 16, 4, hd, tpp, dtype, fp8=True), f"decode fp8 hd={hd} tpp={tpp} {dtype}")


@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("factor", [2.0 ** -15, 2.0 ** 9])
def test_fp8_value_scales(factor, dtype, chunk):
    """Value scales far from one, on one kv head of the pair or both: neither lost below fp16's range nor past it."""
    d = chunk_case(60, [300], [(40, 100)], 8, 4, 64, 16, dtype, fp8=True, eps=1e-20, out_scale=0.01) if chunk else \
        decode_case(60, [300, 20], 8, 4, 64, 16, dtype, fp8=True, eps=1e-20, out_scale=0.01)
    d.vs *= np.float32(factor)
    d.vs[:, 3] /= np.float32(factor * 1.37)
    d.dev["vs"].copy_(torch.from_numpy(d.vs))
    run(d, f"fp8 value scales x {factor} {dtype} chunk={chunk}")


@pytest.mark.parametrize("norm,out_scale", [(True, 1.0), (False, 0.25), (False, 1.0)])
def test_decode_norm_and_scale(norm, out_scale):
    run(decode_case(3, RAGGED, 8, 4, 64, 16, "f16", norm=norm, out_scale=out_scale), f"decode norm={norm} x {out_scale}")


def test_decode_lambda_zero_is_attention():
    """lambda = 0 without a norm: the first maps' ordinary attention, over either half of the value."""
    lens = [700, 33, 5]
    d = decode_case(4, lens, 4, 4, 64, 16, "bf16", norm=False, out_scale=1.0, lam=np.zeros(2, np.float32))
    out = run(d, "decode lambda 0")
    # one query head per kv head: ordinary head 2i reads kv head 2i, keys K1 and the first half of the value
    ref = pal.paged_attention_decode(d.dev["q"], d.dev["k"], d.dev["v"], d.dev["pt"], d.dev["lens"])
    torch.cuda.synchronize()
    a, b = out[:, :, :64].double().cpu(), ref[:, 0::2].double().cpu()
    # each within three bf16 roundings (probabilities, partial results, result) of averages of |v| <= 5
    far = float((a - b).abs().max())
    assert far <= 2 * 3 * 2.0 ** -8 * 5


@pytest.mark.parametrize("hd,tpp,fp8,lens", [
    (128, 16, False, [20000, 7, 33333]), (64, 32, False, [50001]), (128, 16, True, [30000, 1]), (32, 16, False, [40000] * 2),
])
def test_decode_long(hd, tpp, fp8, lens):
    """Few sequences over many workers: segments of tens of pieces."""
    run(decode_case(len(lens) + hd, lens, 8, 2, hd, tpp, "bf16", fp8=fp8), f"decode long {lens} hd={hd} fp8={fp8}")


@pytest.mark.parametrize("seqs,hi", [(1024, 40), (1025, 40), (2500, 20)])
def test_decode_many_sequences(seqs, hi):
    lens = np.random.default_rng(seqs).integers(0, hi, seqs).tolist()
    run(decode_case(seqs, lens, 4, 2, 32, 16, "f16"), f"decode {seqs} sequences")


def test_decode_all_empty():
    d = decode_case(8, [0, 0, 0], 4, 2, 64, 16, "bf16", width=2)
    out = run(d, "decode, no keys at all")
    assert not out.any()


def test_decode_lengths_past_the_table_and_extra_rows():
    d = decode_case(9, [40, 64, 10], 4, 2, 64, 16, "bf16", extra_rows=2, width=4)
    d.case.seq_lens[:] = [40, 64, -3]
    d.dev["lens"] = dev_index(np.array([40, 1 << 30, -3], np.int32))
    out = run(d, "decode, a length past the page table")
    assert out.shape[0] == 3


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_pages_past_the_pool(fp8, norm):
    d = decode_case(10, [200, 90, 20], 8, 4, 64, 16, "bf16", fp8=fp8, norm=norm)
    d.case.page_table[0, 3] = 2 ** 32 - 1
    d.case.page_table[0, 12] = d.case.k_pool.shape[0]
    d.case.page_table[2, :] = d.case.k_pool.shape[0] + 5  # no valid page at all
    d.dev["pt"] = dev_index(d.case.page_table, torch.uint32)
    out = run(d, "decode, page ids past the pool")
    assert not out[2].any()


def test_decode_index_types_and_strides():
    d = decode_case(11, RAGGED, 8, 4, 64, 16, "bf16")
    want = host_bits(d.run())
    wide = torch.zeros((d.dev["pt"].shape[0], 2 * d.dev["pt"].shape[1]), dtype=torch.int64, device=DEV)
    wide[:, ::2] = d.dev["pt"].to(torch.int64)
    d.dev["pt"] = wide[:, ::2]
    d.dev["lens"] = d.dev["lens"].long()
    d.dev["q"] = d.dev["q"].transpose(0, 1).contiguous().transpose(0, 1)
    d.dev["lam"] = d.dev["lam"].repeat_interleave(2)[::2]
    torch.cuda.synchronize()
    assert np.array_equal(host_bits(d.run()), want)


@pytest.mark.parametrize("chunk", [False, True])
def test_nan_stays_in_its_head(chunk):
    """A NaN query, or a NaN or infinite key or value, reaches only what attends to it."""
    lens = [100, 260, 40]
    d = chunk_case(12, [100], [(60, 200), (0, 40)], 8, 4, 64, 16, "bf16") if chunk else \
        decode_case(12, lens, 8, 4, 64, 16, "bf16")
    clean = d.run().clone()
    torch.cuda.synchronize()
    row = 5 if chunk else 1
    d.dev["q"][row, 3, 7] = float("nan")  # map 2 of output head 1
    out = d.run()
    torch.cuda.synchronize()
    same = torch.ones(out.shape[:2], dtype=torch.bool, device=DEV)
    same[row, 1] = False
    assert out[row, 1].isnan().all() and torch.equal(out[same], clean[same])
    # a key of the last kv pair in one sequence: heads 2, 3 of its rows that see it
    d.dev["q"][row, 3, 7] = 0.5
    clean = d.run().clone()
    s = 1
    page = int(d.case.page_table[s, 2])
    for pool, value in (("k", float("nan")), ("v", float("inf"))):
        block = d.dev[pool][page, 2]  # key 1 of pair 1 / first half of its value
        saved = block.clone()
        if pool == "k":
            block[0, 3, 0] = value  # slot 3: token 35
        else:
            block[0, 3] = value
        out = d.run()
        torch.cuda.synchronize()
        block.copy_(saved)
        sees = torch.tensor([t == s and n > 35 for t, n in d.rows()], device=DEV)
        assert not out[sees][:, 2:].isfinite().all(-1).any()
        assert torch.equal(out[~sees], clean[~sees]) and torch.equal(out[sees][:, :2], clean[sees][:, :2])


@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("both", [False, True])
def test_scores_of_minus_infinity(both, chunk):
    """A map whose visible scores are all -inf contributes nothing; with both maps so, the row is zero."""
    d = chunk_case(13, [70], [(10, 90)], 4, 2, 64, 16, "bf16", norm=False) if chunk else \
        decode_case(13, [70, 100], 4, 2, 64, 16, "bf16", norm=False)
    for head in (0, 1) if both else (1,):
        d.dev["q"][:, head::2, 0] = 1.0
        d.dev["k"][:, head, 0, :, 0] = float("-inf")
    announce(f"scores of -inf, both={both} chunk={chunk}")
    out = d.run()
    torch.cuda.synchronize()
    if both:
        assert not out.any()
        return
    d.q = host_bits(d.dev["q"])
    d.lam = np.zeros_like(d.lam)
    d.check(out, "second map without scores")


def test_decode_large_queries():
    """Scores far past the range of exp: one key takes all of a map."""
    d = decode_case(14, [300, 17, 128], 8, 4, 64, 16, "bf16")
    d.q = orc.f32_to_bits(orc.bits_to_f32(d.q, "bf16") * np.float32(1e18), "bf16")
    d.dev["q"] = dev_bits(d.q, "bf16")
    announce("decode, queries of 1e18")
    out = d.run()
    torch.cuda.synchronize()
    y, _ = d.expected()
    # one-hot maps: x is a difference of two values, no sum is rounded; two roundings of the result's chain
    got = out.double().cpu().numpy()
    assert np.abs(got - y).max() <= 4 * 2.0 ** -8 * np.abs(y).max()


# ---------------------------------------------------------------------------
# chunks and mixed batches
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tpp", [16, 32])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_chunk_head_dims(hd, tpp, dtype):
    run(chunk_case(hd + tpp, [40, 1, 333], [(0, 70), (37, 130), (500, 3), (16, 16)], 8, 4, hd, tpp, dtype),
        f"chunk hd={hd} tpp={tpp} {dtype}")


@pytest.mark.parametrize("hq,hkv", GROUPS)
@pytest.mark.parametrize("fp8", [False, True])
def test_chunk_groups(hq, hkv, fp8):
    run(chunk_case(hq * 10 + hkv, [90, 17], [(0, 150), (77, 40)], hq, hkv, 64, 16, "bf16", fp8=fp8),
        f"chunk {hq}/{hkv} fp8={fp8}")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tpp", [16, 32])
@pytest.mark.parametrize("hd", [64, 128])
def test_chunk_fp8(hd, tpp, dtype):
    run(chunk_case(hd + tpp, [40, 333], [(0, 70), (37, 230)], 16, 4, hd, tpp, dtype, fp8=True),
        f"chunk fp8 hd={hd} tpp={tpp} {dtype}")


@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 127, 128, 129, 257, 640])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2)])
def test_one_chunk_sizes(rows, hq, hkv):
    run(chunk_case(rows, [], [(29, rows)], hq, hkv, 64, 16, "bf16", block=1000), f"one chunk of {rows}, {hq}/{hkv}")


@pytest.mark.parametrize("cached,rows,hd,fp8", [(20000, 40, 64, False), (9000, 300, 128, False), (17000, 33, 128, True),
                                                (8190, 5, 32, False)])
def test_chunk_long_history(cached, rows, hd, fp8):
    """Histories of more than one chunk of page ids."""
    run(chunk_case(rows, [9000], [(cached, rows)], 4, 2, hd, 16, "bf16", fp8=fp8), f"chunk of {rows} on {cached} fp8={fp8}")


@pytest.mark.parametrize("norm", [False, True])
def test_lone_rows_only(norm):
    run(chunk_case(15, [5, 900, 17, 64, 2000, 1, 33], [], 8, 4, 64, 16, "f16", norm=norm), "lone rows only")


def test_many_rows():
    """More rows than one planning pass, lone rows among them."""
    rng = np.random.default_rng(16)
    lens = rng.integers(1, 60, 1500).tolist()
    run(chunk_case(16, lens, [(0, 700), (30, 600)], 4, 2, 32, 16, "bf16"), "1,500 lone rows and two chunks")


@pytest.mark.parametrize("rows,longest", [(900, 4), (5000, 4), (9000, 2), (9000, 300)])
def test_many_runs(rows, longest):
    """Runs of 1 to `longest` rows with keys of any number: more tiles than the card holds at once, and than are put
    in order (4,096), on either side of the 1,024 rows that are planned in the stream kernel."""
    rng = np.random.default_rng(rows + longest)
    seqs = 40
    case = make_paged_case(rows, [0] + rng.integers(1, 400, seqs - 1).tolist(), 4, 4, 32, 16, "bf16")
    q2s = []
    while len(q2s) < rows:
        s = int(rng.integers(0, seqs + 1))
        if not q2s or s != q2s[-1]:
            q2s += [s] * (2 if longest == 2 else int(rng.integers(1, longest + 1)))
    q2s = np.array(q2s[:rows], np.uint32)
    off = rng.integers(0, 450, rows).astype(np.int32)
    q = randn_bits(rng, (rows, 4, 32), "bf16")
    run(Diff(case, q, q2s, off, seed=rows), f"{rows} rows in runs of up to {longest}")


def test_long_page_table():
    """A page table of more steps than the order's buckets hold."""
    case = make_paged_case(45, [70000, 40, 33000], 2, 2, 32, 16, "bf16")
    q2s = np.repeat(np.array([0, 1, 2, 0, 2], np.uint32), [130, 20, 40, 1, 1])
    off = np.concatenate([69000 + np.arange(130), 20 + np.arange(20), np.arange(40) * 800, [70000], [5]]).astype(np.int32)
    q = randn_bits(np.random.default_rng(45), (len(q2s), 2, 32), "bf16")
    run(Diff(case, q, q2s, off, seed=45), "a table of 70,000 keys")


def test_no_sequences():
    """Rows that all name no sequence, with a page table of no rows."""
    d = chunk_case(46, [40], [(0, 10)], 4, 2, 64, 16, "bf16")
    x = d.dev
    n = torch.zeros(0, dtype=torch.int32, device=DEV)
    out = pal.paged_differential_attention(x["q"], x["k"], x["v"], x["pt"][:0], n, x["q2s"], x["off"], x["lam"])
    torch.cuda.synchronize()
    assert tuple(out.shape) == (11, 2, 128) and not out.any()


def test_any_limits_in_a_run():
    """Offsets of a run in any order, past the length, zero and negative; rows naming no sequence."""
    rng = np.random.default_rng(17)
    case = make_paged_case(17, [500, 90, 0], 8, 4, 64, 16, "bf16")
    q2s = np.array([0] * 200 + [7] * 3 + [1] * 90 + [2] * 5 + [9] + [0] * 2 + [2 ** 32 - 1] * 2, np.uint32)
    off = rng.integers(-5, 700, len(q2s)).astype(np.int32)
    off[:40] = 0
    off[130:140] = -(2 ** 31)
    off[140] = 2 ** 31 - 1
    q = randn_bits(rng, (len(q2s), 8, 64), "bf16")
    run(Diff(case, q, q2s, off, seed=17), "limits in any order")


@pytest.mark.parametrize("norm", [True, False])  # (the norm would hide what changes both maps alike)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tpp", [16, 32])
def test_chunk_pages_past_the_pool(fp8, tpp, norm):
    d = chunk_case(18, [200], [(150, 100), (0, 64)], 8, 4, 64, tpp, "bf16", fp8=fp8, norm=norm)
    pages = d.case.k_pool.shape[0]
    d.case.page_table[0, 2] = pages
    d.case.page_table[1, 1] = 2 ** 32 - 1
    d.case.page_table[1, 5] = pages + 3
    d.case.page_table[2, :] = pages + 9
    d.dev["pt"] = dev_index(d.case.page_table, torch.uint32)
    run(d, f"chunk, page ids past the pool fp8={fp8} norm={norm}")


def test_rows_shuffled_in_short_blocks():
    run(chunk_case(19, [40, 77], [(0, 128), (64, 100)], 8, 4, 64, 16, "bf16", block=7), "rows shuffled in blocks of 7")


def test_no_rows():
    d = chunk_case(20, [40], [(0, 10)], 4, 2, 64, 16, "bf16")
    e = torch.empty((0, 4, 64), dtype=torch.bfloat16, device=DEV)
    i = torch.empty(0, dtype=torch.int32, device=DEV)
    out = pal.paged_differential_attention(e, d.dev["k"], d.dev["v"], d.dev["pt"], d.dev["lens"], i, i, d.dev["lam"])
    assert tuple(out.shape) == (0, 2, 128)
    out = pal.paged_differential_attention_decode(e, d.dev["k"], d.dev["v"], d.dev["pt"][:0], i, d.dev["lam"])
    assert tuple(out.shape) == (0, 2, 128)


@pytest.mark.parametrize("chunk", [False, True])
def test_no_pages(chunk):
    lam = torch.ones(2, device=DEV)
    k = torch.empty(pal.get_k_cache_shape(0, 2, 64, 16, torch.bfloat16), dtype=torch.bfloat16, device=DEV)
    v = torch.empty(pal.get_v_cache_shape(0, 2, 64, 16, torch.bfloat16), dtype=torch.bfloat16, device=DEV)
    q = torch.ones((3, 4, 64), dtype=torch.bfloat16, device=DEV)
    pt = torch.zeros((3, 2), dtype=torch.int32, device=DEV)
    n = torch.full((3,), 20, dtype=torch.int32, device=DEV)
    out = pal.paged_differential_attention(q, k, v, pt, n, torch.arange(3, device=DEV), n, lam) if chunk else \
        pal.paged_differential_attention_decode(q, k, v, pt, n, lam)
    torch.cuda.synchronize()
    assert not out.any()


# ---------------------------------------------------------------------------
# streams, graphs, repeatability, refusals
# ---------------------------------------------------------------------------


def _both():
    return (decode_case(30, [3000, 17, 512, 900], 16, 4, 128, 16, "bf16"),
            chunk_case(31, [900, 40], [(100, 300), (0, 77)], 16, 4, 128, 16, "bf16"))


def test_repeats_are_bit_equal():
    for d in _both():
        want = host_bits(d.run())
        for _ in range(3):
            assert np.array_equal(host_bits(d.run()), want)


def test_two_streams_at_once():
    ds = _both()
    want = [host_bits(d.run()) for d in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    announce("two streams at once")
    outs = [[d.run(stream=s) for d, s in zip(ds, streams)] for _ in range(5)]
    torch.cuda.synchronize()
    for pair in outs:
        for o, w in zip(pair, want):
            assert np.array_equal(host_bits(o), w)


def test_graphs_share_nothing():
    """Two graphs captured on one stream, replayed at once on two streams, and after eager calls."""
    ds = _both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for d in ds:
            d.run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for d in ds:
        g = torch.cuda.CUDAGraph()
        announce("graph capture: differential attention")
        with torch.cuda.graph(g, stream=side):
            outs.append(d.run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in ds]
    for r in range(4):
        for d in ds:
            d.dev["q"].copy_(torch.randn(d.dev["q"].shape, device=DEV))
        want = [host_bits(d.run()) for d in ds]
        torch.cuda.synchronize()
        announce(f"graph replay {r}: both at once")
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert np.array_equal(host_bits(o), w), f"replay {r}"


def test_graph_replays_plan_anew():
    """A captured mixed batch whose lengths, limits and rows' sequences change between replays: lone rows, tiles and
    their order are found at every replay, on both sides of the rows that are planned in the stream kernel."""
    rng = np.random.default_rng(34)
    for rows in (700, 1500):
        lens = rng.integers(1, 90, 300).tolist()
        d = chunk_case(34, lens, [(30, rows - 500), (0, 200)], 8, 4, 32, 16, "bf16")
        seqs = len(d.case.seq_lens)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            d.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        announce(f"graph capture: {rows} rows")
        with torch.cuda.graph(g, stream=side):
            out = d.run()
        for r in range(4):
            n = int(d.off.shape[0])
            q2s = np.sort(rng.integers(0, seqs, n)) if r % 2 else np.repeat(rng.permutation(seqs), -(-n // seqs))[:n]
            d.dev["q2s"].copy_(dev_index(q2s.astype(np.uint32), torch.uint32))
            d.dev["off"].copy_(dev_index(rng.integers(-3, 300, n).astype(np.int32)))
            d.dev["lens"].copy_(dev_index((d.case.seq_lens * rng.integers(0, 2, seqs)).astype(np.int32)))
            want = host_bits(d.run())
            torch.cuda.synchronize()
            announce(f"graph replay {r} of {rows} rows")
            g.replay()
            torch.cuda.synchronize()
            assert np.array_equal(host_bits(out), want), f"replay {r} of {rows} rows"


def test_refusals():
    d = decode_case(40, [40, 20], 8, 4, 64, 16, "bf16")
    x = d.dev

    def call(q=x["q"], k=x["k"], v=x["v"], pt=x["pt"], lens=x["lens"], lam=x["lam"], **kw):
        return pal.paged_differential_attention_decode(q, k, v, pt, lens, lam, **kw)

    bad = [
        (dict(lam=x["lam"].half()), "lambdas"), (dict(lam=x["lam"][:3]), "lambdas"), (dict(lam=x["lam"].cpu()), "lambdas"),
        (dict(norm_weight=torch.ones(64, device=DEV)), "norm_weight"),
        (dict(norm_weight=torch.ones(128, device=DEV, dtype=torch.bfloat16)), "norm_weight"),
        (dict(norm_eps=-1.0), "norm_eps"), (dict(norm_eps=float("nan")), "norm_eps"),
        (dict(q=x["q"][:, :7]), "pairs"), (dict(q=x["q"][0]), "queries"), (dict(q=x["q"][:1]), "query rows"),
        (dict(pt=x["pt"][0]), "page_table"), (dict(lens=x["lens"][:1]), "lengths"),
        (dict(k_scales=torch.ones(1, device=DEV)), "fp8"),
    ]
    for kw, word in bad:
        with pytest.raises(ValueError, match=word):
            call(**kw)
    odd_k, odd_v = x["k"][:, :3].contiguous(), x["v"][:, :3].contiguous()
    with pytest.raises(ValueError, match="pairs"):
        call(k=odd_k, v=odd_v, q=x["q"][:, :6].contiguous())
    with pytest.raises(RuntimeError, match="divisible"):
        call(q=x["q"][:, :6].contiguous(), lam=x["lam"][:3].contiguous())
    n = torch.zeros(3, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="one entry per query row"):
        pal.paged_differential_attention(x["q"], x["k"], x["v"], x["pt"], x["lens"], n, n, x["lam"])
    big = [torch.zeros(f(4, 2, 256, 16, torch.bfloat16), dtype=torch.bfloat16, device=DEV)
           for f in (pal.get_k_cache_shape, pal.get_v_cache_shape)]
    with pytest.raises(RuntimeError, match="head_dim 256"):
        call(q=torch.zeros((2, 4, 256), dtype=torch.bfloat16, device=DEV), k=big[0], v=big[1],
             lam=torch.ones(2, device=DEV))


def test_differential_lambda():
    g = torch.Generator().manual_seed(1)
    v = [0.1 * torch.randn(64, generator=g) for _ in range(4)]
    lam = pal.differential_lambda(*(t.to(DEV) for t in v), 0.8, 6)
    want = np.exp(float(v[0].double() @ v[1].double())) - np.exp(float(v[2].double() @ v[3].double())) + 0.8
    assert lam.dtype == torch.float32 and tuple(lam.shape) == (6,) and lam.is_contiguous()
    assert (lam.double().cpu() - want).abs().max() <= 2.0 ** -24 * abs(want)
    per_head = pal.differential_lambda(*(t.expand(6, 64) for t in v), 0.8, 6)
    assert (per_head.double() - want).abs().max() <= 2.0 ** -24 * abs(want)
    with pytest.raises(ValueError, match="vectors"):
        pal.differential_lambda(v[0], v[1], v[2], v[3][:5], 0.8, 6)
    with pytest.raises(ValueError, match="vectors"):
        pal.differential_lambda(*(t.expand(5, 64) for t in v), 0.8, 6)


# ---------------------------------------------------------------------------
# together with the fills
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_prompt_then_decode_steps(kv):
    """As a program runs them: prompts with image tokens filled by mrope_fill_kv_pages and attended in chunks, then
    decode steps; the last step's rows against the definition over the pools as they were filled."""
    rng = np.random.default_rng(50)
    hq, hkv, hd, tpp, pages = 16, 4, 64, 16, 40
    dtype = torch.float8_e4m3fn if kv == "fp8" else torch.bfloat16
    k = torch.zeros(pal.get_k_cache_shape(pages, hkv, hd, tpp, dtype), device=DEV).to(dtype)
    v = torch.zeros(pal.get_v_cache_shape(pages, hkv, hd, tpp, dtype), device=DEV).to(dtype)
    sc = torch.full((pages, hkv), 1 / 64, device=DEV)
    scales = dict(k_scales=sc, v_scales=sc) if kv == "fp8" else {}
    prompt = [70, 33, 150]
    pt = dev_index(rng.permutation(pages)[:36].reshape(3, 12).astype(np.int32))
    table = pal.rope_cos_sin_cache(400, hd, device=DEV)
    lam = pal.differential_lambda(*(0.1 * torch.randn(4, hd, generator=torch.Generator().manual_seed(2))).to(DEV), 0.6, hq // 2)
    weight = torch.ones(2 * hd, device=DEV)

    def fill(n, pos, q2s, rope):
        new = [torch.from_numpy(rng.standard_normal((n, h, hd)).astype(np.float32)).to(DEV) for h in (hkv, hkv, hq)]
        return pal.mrope_fill_kv_pages(new[0], new[1], k, v, pt, dev_index(pos), dev_index(q2s), dev_index(rope), table,
                                       (12, 10, 10), interleaved=True, queries=new[2], **scales)[2]

    q2s = np.repeat(np.arange(3), prompt).astype(np.int32)
    pos = np.concatenate([np.arange(n) for n in prompt]).astype(np.int32)
    q = fill(len(pos), pos, q2s, np.stack([pos, pos // 7, pos % 7]).astype(np.int32))
    lens = np.array(prompt, np.int32)
    kw = dict(norm_weight=weight, out_scale=0.4, **scales)
    announce(f"prompt, then decode steps over {kv} pages")
    first = pal.paged_differential_attention(q, k, v, pt, dev_index(lens), dev_index(q2s), dev_index(pos + 1), lam, **kw)
    state = [(q, q2s, pos + 1, lens.copy(), first, k.clone(), v.clone())]
    for _ in range(3):
        q = fill(3, lens, np.arange(3, dtype=np.int32), np.stack([lens] * 3).astype(np.int32))
        lens = lens + 1
        out = pal.paged_differential_attention_decode(q, k, v, pt, dev_index(lens), lam, **kw)
    state.append((q, None, None, lens.copy(), out, k, v))
    torch.cuda.synchronize()
    for q, seq, off, n, out, kp, vp in state:
        case = make_paged_case(0, [1], hq, hkv, hd, tpp, "bf16")
        case.page_table, case.seq_lens = pt.cpu().numpy().astype(np.uint32), n
        d = Diff.__new__(Diff)
        d.case, d.q, d.q2s, d.off, d.fp8 = case, host_bits(q), None if seq is None else seq.astype(np.uint32), off, kv == "fp8"
        d.lam, d.weight, d.out_scale, d.eps = lam.cpu().numpy(), weight.cpu().numpy(), 0.4, 1e-5
        if kv == "fp8":
            d.kc, d.vc = kp.view(torch.uint8).cpu().numpy(), vp.view(torch.uint8).cpu().numpy()
            d.ks = d.vs = sc.cpu().numpy()
        else:
            case.k_pool, case.v_pool = host_bits(kp), host_bits(vp)
        d.check(out, "prompt" if seq is not None else "third decode step")
