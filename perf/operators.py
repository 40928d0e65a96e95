"""Calls of the differential attention operators and of the several-axes RoPE fill.

Three operators over the paged KV cache:

  decode  paged_differential_attention_decode: one new token per sequence
  chunk   paged_differential_attention: chunks of new tokens, with single
          decode rows ahead of them in a mixed batch
  mrope   mrope_fill_kv_pages: rotate K and Q by positions of several axes,
          cast, and scatter K and V into the cache

Query heads 2i and 2i + 1 are the two maps of output head i; kv heads 2j and
2j + 1 hold the two keys of pair j and the two halves of its value:

  x = (softmax(q1 K1^T / sqrt(hd)) - lambda softmax(q2 K2^T / sqrt(hd))) [V1 V2]
  y = out_scale * weight * x / sqrt(mean(x^2) + eps)     (weight given)
  y = out_scale * x                                       (no weight)

Rotation: frequency f of a token turns by the position of axis a(f).

Keys, values and queries are N(0, 1); pages are randomly permuted in a pool
with about 10 % free pages.  Lengths follow from the case (``lens_seed``),
values and page tables from the seed given to ``prepare``.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda:0"
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_FP8 = torch.float8_e4m3fn
_EPS = 1e-5

# 32 query heads on 8 kv heads of dimension 128 over 16-token pages is the
# shape of most of the benchmark's workloads
_BASE = {"hq": 32, "hkv": 8, "hd": 128, "tpp": 16, "dtype": "bf16", "fp8": False, "lens_seed": 1}


def _case(name: str, kind: str, **values) -> dict:
    return {"name": name, "kind": kind, **_BASE, **values}


def listed() -> list[dict]:
    return [
        # a handful of short requests on a small model: launches and latency
        _case("decode_tiny", "decode", seqs=4, ctx_lo=33, ctx_hi=250, hq=8, hkv=4, hd=64, dtype="f16", norm=True),
        # the serving step of a full batch
        _case("decode_64", "decode", seqs=64, ctx_lo=512, ctx_hi=4096, norm=True),
        # the same batch over an fp8 cache
        _case("decode_fp8_64", "decode", seqs=64, ctx_lo=512, ctx_hi=4096, fp8=True, norm=True),
        # many short contexts (classification, short answers), no sharing of kv heads
        _case("decode_short_1000", "decode", seqs=1000, ctx_lo=1, ctx_hi=256, hq=16, hkv=16, dtype="f16", norm=True),
        # long documents; the head norm left to the caller
        _case("decode_long", "decode", seqs=4, ctx_lo=32768, ctx_hi=131072, hd=64, tpp=32, norm=False),
        # a single short prompt, nothing cached: time to the first token
        _case("chunk_single", "chunk", rows_dec=0, ctx_lo=1, ctx_hi=1, chunks=1, new_lo=333, new_hi=333, cached_lo=0,
              cached_hi=0, hq=16, hkv=8, hd=64, norm=True),
        # chunked prefill of a ragged batch
        _case("chunk_8", "chunk", rows_dec=0, ctx_lo=1, ctx_hi=1, chunks=8, new_lo=512, new_hi=2048, cached_lo=0,
              cached_hi=2048, norm=True),
        # chunked prefill over an fp8 cache
        _case("chunk_fp8", "chunk", rows_dec=0, ctx_lo=1, ctx_hi=1, chunks=4, new_lo=256, new_hi=1024, cached_lo=0,
              cached_hi=4096, fp8=True, dtype="f16", norm=True),
        # decode rows and prefill chunks in one call (continuous batching)
        _case("mixed", "chunk", rows_dec=96, ctx_lo=256, ctx_hi=4096, chunks=2, new_lo=700, new_hi=1024, cached_lo=0,
              cached_hi=2048, hd=64, tpp=32, dtype="f16", norm=True),
        # one decode step's new tokens (generated text after an image)
        _case("mrope_step", "mrope", seqs=64, new_lo=1, new_hi=1, cached_lo=512, cached_hi=4096, src="f32",
              sections="16,24,24", interleaved=False, rot=128, style="neox"),
        # prompts with images in chunked prefill, the projection in 16 bits
        _case("mrope_images", "mrope", seqs=12, new_lo=512, new_hi=2048, cached_lo=0, cached_hi=2048, src="bf16",
              sections="16,24,24", interleaved=False, rot=128, style="neox"),
        # the projection's fp32 rows into an fp8 cache of unit scales, axes interleaved
        _case("mrope_fp8", "mrope", seqs=4, new_lo=256, new_hi=1024, cached_lo=0, cached_hi=1024, src="f32", fp8=True,
              sections="24,20,20", interleaved=True, rot=128, style="neox"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["decode", "decode", "chunk", "chunk", "mrope"])
    hq, hkv = rng.choice([(32, 8), (32, 8), (64, 8), (24, 4), (32, 32), (16, 2), (40, 2)])
    fp8 = rng.random() < 0.3
    hd = rng.choice([64, 128]) if fp8 else rng.choice([32, 64, 96, 128, 128])
    case = {"kind": kind, "hq": hq, "hkv": hkv, "hd": hd, "tpp": rng.choice([16, 16, 32]),
            "dtype": rng.choice(["bf16", "bf16", "f16"]), "fp8": fp8, "lens_seed": rng.randrange(1, 1 << 30)}
    token_bytes = 4 * hkv * hd  # K and V of a token, 16 bit
    if kind == "decode":
        seqs = _log_int(rng, 1, 1500)
        # the batch's context up to 0.6 GB of 16-bit K and V
        hi = max(2, min(131072, int(6e8 / (token_bytes * seqs))))
        ctx_hi = _log_int(rng, min(48, hi), hi)
        case.update(seqs=seqs, ctx_lo=max(1, ctx_hi // rng.choice([1, 2, 8])), ctx_hi=ctx_hi,
                    norm=rng.random() < 0.8)
    elif kind == "chunk":
        chunks = _log_int(rng, 1, 8)
        new_hi = _log_int(rng, 16, 2048)
        case.update(rows_dec=rng.choice([0, 0, _log_int(rng, 1, 128)]), ctx_lo=1, ctx_hi=_log_int(rng, 32, 4096),
                    chunks=chunks, new_lo=max(2, new_hi // 4), new_hi=new_hi, cached_lo=0,
                    cached_hi=rng.randrange(0, 2049), norm=rng.random() < 0.8)
        # no more attention work than the largest listed chunk case
        while work(case)["flops"] > 1e11 and case["new_hi"] > 16:
            new_hi = max(16, case["new_hi"] // 2)
            case.update(new_lo=max(2, new_hi // 4), new_hi=new_hi)
    else:
        style = rng.choice(["neox", "neox", "gptj"])
        rot = rng.choice([hd, hd, hd // 2])
        half = rot // 2
        if rng.random() < 0.5:  # two thirds of the frequencies to the two image axes
            a = half * 3 // 8
            sections = [half - 2 * a, a, a]
        else:
            sections = [half - 2 * (half // 3), half // 3, half // 3]
        interleaved = sections[0] >= sections[1] and rng.random() < 0.5
        new_hi = _log_int(rng, 1, 2048)
        case.update(seqs=_log_int(rng, 1, 12), new_lo=max(1, new_hi // 4), new_hi=new_hi, cached_lo=0,
                    cached_hi=rng.randrange(0, 2049), src=rng.choice(["f32", "bf16", "f16"]),
                    sections=",".join(str(s) for s in sections), interleaved=interleaved, rot=rot, style=style)
        while case["seqs"] * new_hi * (hq + 2 * hkv) * hd > 8e7:
            new_hi = max(1, new_hi // 2)
            case.update(new_lo=max(1, new_hi // 4), new_hi=new_hi)
    return case


# ---------------------------------------------------------------------------
# sizes of a case
# ---------------------------------------------------------------------------


def _lengths(case: dict) -> dict:
    """Ragged lengths: keys of every sequence, and its new tokens."""
    rng = random.Random(case["lens_seed"])
    if case["kind"] == "decode":
        keys = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
        return {"keys": keys, "new": [1] * len(keys)}
    if case["kind"] == "chunk":
        keys = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["rows_dec"])]
        new = [1] * len(keys)
        for _ in range(case["chunks"]):
            n = rng.randint(case["new_lo"], case["new_hi"])
            keys.append(rng.randint(case["cached_lo"], case["cached_hi"]) + n)
            new.append(n)
        return {"keys": keys, "new": new}
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    return {"keys": [rng.randint(case["cached_lo"], case["cached_hi"]) + n for n in new], "new": new}


def work(case: dict) -> dict:
    n = _lengths(case)
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    tokens, rows = sum(n["keys"]), sum(n["new"])
    pool_bytes = 1 if case["fp8"] else 2
    if case["kind"] == "mrope":
        src = 4 if case["src"] == "f32" else 2
        # sources read, pools and rotated queries written, four indices and one table row a token
        return {"bytes": rows * ((2 * hkv + hq) * hd * src + 2 * hkv * hd * pool_bytes + hq * hd * 2 + 20 + 4 * case["rot"]),
                "flops": rows * (hkv + hq) * case["rot"] * 3}
    scales = sum(-(-k // case["tpp"]) for k in n["keys"]) * 2 * hkv * 4 if case["fp8"] else 0
    pages = 4 * sum(-(-k // case["tpp"]) for k in n["keys"])
    # keys each row sees, summed: a chunk of m rows over k keys sees k - m + 1 .. k
    seen = sum(m * k - m * (m - 1) // 2 for k, m in zip(n["keys"], n["new"]))
    # per output head and key: two score products of hd, one of the difference of the maps with 2 hd values
    return {"bytes": tokens * 2 * hkv * hd * pool_bytes + scales + pages + 2 * rows * hq * hd * 2,
            "flops": seen * (hq // 2) * 8 * hd}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _pools(case: dict, keys: list[int], g: torch.Generator):
    """Empty pools over permuted pages, and the page table (host-built plan)."""
    tpp, hkv, hd = case["tpp"], case["hkv"], case["hd"]
    per = [-(-k // tpp) for k in keys]
    width, used = max(per), sum(per)
    total = used + max(2, used // 10)
    perm = torch.randperm(total, generator=g, device=DEVICE)
    lens = torch.tensor(per, device=DEVICE)
    first = torch.cumsum(lens, 0) - lens
    col = torch.arange(width, device=DEVICE)
    idx = torch.minimum(first[:, None] + col[None, :], torch.tensor(total - 1, device=DEVICE))
    table = torch.where(col[None, :] < lens[:, None], perm[idx], torch.zeros_like(idx)).to(torch.int32)
    dtype = _FP8 if case["fp8"] else _DTYPES[case["dtype"]]
    x = 16 // torch.empty((), dtype=dtype).element_size()
    return table, total, (total, hkv, hd // x, tpp, x), (total, hkv, hd, tpp), dtype


def _normal(shape, g: torch.Generator, dtype: torch.dtype) -> torch.Tensor:
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _attention_state(case: dict, g: torch.Generator) -> dict:
    n = _lengths(case)
    hq, hkv, hd, dtype = case["hq"], case["hkv"], case["hd"], _DTYPES[case["dtype"]]
    table, total, k_shape, v_shape, pool_dtype = _pools(case, n["keys"], g)
    st = {"case": case, "table": table, "lens": torch.tensor(n["keys"], dtype=torch.int32, device=DEVICE)}
    if case["fp8"]:  # codes of a standard deviation of 64, each (page, kv head) block with a scale of its own
        st["k"] = (64 * torch.randn(k_shape, generator=g, device=DEVICE)).clamp_(-448, 448).to(_FP8)
        st["v"] = (64 * torch.randn(v_shape, generator=g, device=DEVICE)).clamp_(-448, 448).to(_FP8)
        for name in ("k_scales", "v_scales"):
            st[name] = (0.75 + 0.5 * torch.rand((total, hkv), generator=g, device=DEVICE)) / 64
    else:
        st["k"], st["v"] = _normal(k_shape, g, pool_dtype), _normal(v_shape, g, pool_dtype)
        st["k_scales"] = st["v_scales"] = None
    rows = sum(n["new"])
    st["q"] = _normal((rows, hq, hd), g, dtype)
    # lambdas near a middle layer's start value; the norm's weight near one
    st["lam"] = 0.6 + 0.1 * torch.randn(hq // 2, generator=g, device=DEVICE)
    st["weight"] = 1 + 0.1 * torch.randn(2 * hd, generator=g, device=DEVICE) if case["norm"] else None
    st["out_scale"] = 0.4
    if case["kind"] == "chunk":
        new = torch.tensor(n["new"], device=DEVICE)
        st["q2s"] = torch.repeat_interleave(torch.arange(len(n["new"]), device=DEVICE), new).to(torch.int32)
        starts = torch.cumsum(new, 0) - new
        within = torch.arange(rows, device=DEVICE) - starts[st["q2s"].long()]
        st["off"] = (st["lens"][st["q2s"].long()] - new[st["q2s"].long()] + within + 1).to(torch.int32)
        st["rows_dec"] = case["rows_dec"]
        st["new_max"] = max(n["new"])
    return st


def _grid_positions(n: int, start: int, rng: random.Random) -> list[tuple[int, int, int]]:
    """(time, height, width) positions of a prompt: text, an image of rows of
    patches, text again; a decode step is one text token."""
    out, p = [], start
    while len(out) < n:
        for _ in range(min(n - len(out), rng.randint(8, 64))):
            out.append((p, p, p))
            p += 1
        w = rng.randint(6, 24)
        size = min(n - len(out), w * rng.randint(6, 24))
        out.extend((p, p + i // w, p + i % w) for i in range(size))
        p += max(w, -(-size // w)) if size else 0
    return out


def _mrope_state(case: dict, g: torch.Generator) -> dict:
    n = _lengths(case)
    hq, hkv, hd, src = case["hq"], case["hkv"], case["hd"], _DTYPES[case["src"]]
    table, total, k_shape, v_shape, pool_dtype = _pools(case, n["keys"], g)
    rows = sum(n["new"])
    rng = random.Random(case["lens_seed"] + 1)
    grid, write = [], []
    for k, m in zip(n["keys"], n["new"]):
        grid += _grid_positions(m, (k - m) // 2, rng)
        write += range(k - m, k)
    half = case["rot"] // 2
    rows_table = 4352  # a served context, counted in positions
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
    angle = torch.arange(rows_table, dtype=torch.float64, device=DEVICE)[:, None] * freq[None, :]
    st = {
        "case": case, "table": table,
        "k": torch.zeros(k_shape, dtype=torch.float32, device=DEVICE).to(pool_dtype),
        "v": torch.zeros(v_shape, dtype=torch.float32, device=DEVICE).to(pool_dtype),
        "k_scales": torch.ones((total, hkv), device=DEVICE) if case["fp8"] else None,
        "v_scales": torch.ones((total, hkv), device=DEVICE) if case["fp8"] else None,
        "new_k": _normal((rows, hkv, hd), g, src), "new_v": _normal((rows, hkv, hd), g, src),
        "q": _normal((rows, hq, hd), g, src),
        "write": torch.tensor(write, dtype=torch.int32, device=DEVICE),
        "q2s": torch.repeat_interleave(torch.arange(len(n["new"]), device=DEVICE),
                                       torch.tensor(n["new"], device=DEVICE)).to(torch.int32),
        "pos": torch.tensor(grid, dtype=torch.int32).t().contiguous().to(DEVICE),
        "cos_sin": torch.cat([torch.cos(angle), torch.sin(angle)], 1).to(torch.float32),
        "sections": tuple(int(s) for s in case["sections"].split(",")),
        "q_dtype": _DTYPES[case["dtype"]],
    }
    return st


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return _mrope_state(case, g) if case["kind"] == "mrope" else _attention_state(case, g)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _gather(pool: torch.Tensor, scales, table: torch.Tensor, keys: bool) -> torch.Tensor:
    """fp32 [S, Hkv, W * TPP, HD] of the pages of a table."""
    t = pool.view(torch.uint8)[table.long()].view(_FP8).float() if pool.dtype == _FP8 else pool[table.long()].float()
    if scales is not None:  # [S, W, Hkv, ...]
        f = scales[table.long()]
        t = t * f.reshape(*f.shape, *([1] * (t.dim() - 3)))
    if keys:  # [S, W, Hkv, HD/x, TPP, x]
        s, w, h, c, p, x = t.shape
        return t.permute(0, 2, 1, 4, 3, 5).reshape(s, h, w * p, c * x)
    s, w, h, d, p = t.shape
    return t.permute(0, 2, 1, 4, 3).reshape(s, h, w * p, d)


def _plain_rows(st: dict, q: torch.Tensor, table: torch.Tensor, visible: torch.Tensor) -> torch.Tensor:
    """q [S, M, Hq, HD] over the pages of table [S, W]; row m of sequence s
    sees its first visible[s, m] keys.  Returns fp32 [S, M, Hq/2, 2 HD]."""
    s, m, hq, hd = q.shape
    k = _gather(st["k"], st["k_scales"], table, True)
    v = _gather(st["v"], st["v_scales"], table, False)
    hkv, n = k.shape[1], k.shape[2]
    group = hq // hkv
    # query head 2i + a of pair i = j group + e  ->  kv head 2j + a
    qf = q.float().reshape(s, m, hkv // 2, group, 2, hd).permute(0, 2, 4, 3, 1, 5).reshape(s, hkv, group * m, hd)
    score = torch.matmul(qf, k.transpose(-1, -2)) / math.sqrt(hd)
    del k, qf
    hidden = torch.arange(n, device=q.device)[None, None, :] >= visible[:, :, None]
    score = score.reshape(s, hkv, group, m, n).masked_fill_(hidden[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    del score
    z = e.sum(-1, keepdim=True)
    e = (e / torch.where(z == 0, torch.ones_like(z), z)).reshape(s, hkv // 2, 2, group, m, n)
    lam = st["lam"].reshape(1, hkv // 2, group, 1, 1)
    a = (e[:, :, 0] - lam * e[:, :, 1]).reshape(s, hkv // 2, group * m, n)
    del e
    # the value of a pair: kv head 2j's dims, then kv head 2j + 1's
    v = v.reshape(s, hkv // 2, 2, n, hd).permute(0, 1, 3, 2, 4).reshape(s, hkv // 2, n, 2 * hd)
    x = torch.matmul(a, v).reshape(s, hkv // 2, group, m, 2 * hd)
    if st["weight"] is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * st["weight"]
    return (x * st["out_scale"]).permute(0, 3, 1, 2, 4).reshape(s, m, hq // 2, 2 * hd)


def _plain_decode(st: dict) -> torch.Tensor:
    return _plain_rows(st, st["q"][:, None], st["table"], st["lens"][:, None])[:, 0].to(st["q"].dtype)


def _plain_chunk(st: dict) -> torch.Tensor:
    q, dec = st["q"], st["rows_dec"]
    out = torch.empty((q.shape[0], q.shape[1] // 2, 2 * q.shape[2]), dtype=q.dtype, device=q.device)
    visible = torch.minimum(st["off"], st["lens"][st["q2s"].long()])
    if dec:  # single rows ahead of the chunks, one a sequence
        seq = st["q2s"][:dec].long()
        out[:dec] = _plain_rows(st, q[:dec, None], st["table"][seq], visible[:dec, None])[:, 0].to(q.dtype)
    # the chunks' rows, padded to the longest
    seq = st["q2s"][dec:].long() - dec
    count = torch.bincount(seq, minlength=st["table"].shape[0] - dec)
    at = torch.arange(seq.numel(), device=q.device) - (torch.cumsum(count, 0) - count)[seq]
    padded = q.new_zeros((count.numel(), st["new_max"], *q.shape[1:]))
    padded[seq, at] = q[dec:]
    seen = torch.zeros((count.numel(), st["new_max"]), dtype=visible.dtype, device=q.device)
    seen[seq, at] = visible[dec:]
    out[dec:] = _plain_rows(st, padded, st["table"][dec:], seen)[seq, at].to(q.dtype)
    return out


def _axes(sections: tuple, interleaved: bool, device) -> torch.Tensor:
    """Axis of every frequency."""
    n = torch.tensor(sections, device=device)
    if not interleaved:
        return torch.repeat_interleave(torch.arange(len(sections), device=device), n)
    f = torch.arange(sum(sections), device=device)
    a = f % len(sections)
    return torch.where(f < len(sections) * n[a], a, torch.zeros_like(a))


def _plain_turn(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, style: str) -> torch.Tensor:
    rot = 2 * cos.shape[-1]
    f = x.float()
    c, s = cos[:, None], sin[:, None]
    if style == "neox":
        a, b = f[..., :rot // 2], f[..., rot // 2:rot]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = f[..., 0:rot:2], f[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([turned, f[..., rot:]], -1)


def _plain_mrope(st: dict):
    case, half = st["case"], st["case"]["rot"] // 2
    axis = _axes(st["sections"], case["interleaved"], st["pos"].device)
    row = st["pos"].long()[axis].t()  # [N, half]: the table row of every frequency
    f = torch.arange(half, device=row.device)[None, :]
    cos, sin = st["cos_sin"][row, f], st["cos_sin"][row, half + f]
    k, q = _plain_turn(st["new_k"], cos, sin, case["style"]), _plain_turn(st["q"], cos, sin, case["style"])
    v = st["new_v"].float()
    tpp = case["tpp"]
    page = st["table"][st["q2s"].long(), st["write"].long() // tpp].long()
    slot = st["write"].long() % tpp
    if case["fp8"]:
        k = (k / st["k_scales"][page][..., None]).clamp(-448, 448)
        v = (v / st["v_scales"][page][..., None]).clamp(-448, 448)
    kp, vp = st["k"], st["v"]
    k, v = k.to(kp.dtype).unflatten(-1, (-1, kp.shape[-1])), v.to(vp.dtype)
    if case["fp8"]:
        kp, vp, k, v = (t.view(torch.uint8) for t in (kp, vp, k, v))
    kp[page, :, :, slot, :] = k
    vp[page, :, :, slot] = v
    return st["k"], st["v"], q.to(st["q_dtype"])


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def _package():
    at = str(Path.cwd() / "proxy-attention-lab_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import proxy_attention_lab as pal

    return pal


def run(st: dict):
    case = st["case"]
    if not own:
        return {"decode": _plain_decode, "chunk": _plain_chunk, "mrope": _plain_mrope}[case["kind"]](st)
    pal = _package()
    if case["kind"] == "mrope":
        return pal.mrope_fill_kv_pages(
            st["new_k"], st["new_v"], st["k"], st["v"], st["table"], st["write"], st["q2s"], st["pos"], st["cos_sin"],
            st["sections"], interleaved=case["interleaved"], queries=st["q"], rotary_dim=case["rot"],
            style=case["style"], query_dtype=st["q_dtype"], k_scales=st["k_scales"], v_scales=st["v_scales"])
    more = {"norm_weight": st["weight"], "norm_eps": _EPS, "out_scale": st["out_scale"], "k_scales": st["k_scales"],
            "v_scales": st["v_scales"]}
    if case["kind"] == "decode":
        return pal.paged_differential_attention_decode(st["q"], st["k"], st["v"], st["table"], st["lens"], st["lam"],
                                                       **more)
    return pal.paged_differential_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], st["q2s"], st["off"],
                                            st["lam"], **more)


# ---------------------------------------------------------------------------
# the definition in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------


def _exact_sequence(st: dict, s: int, rows: range) -> torch.Tensor:
    """Rows of sequence s: [len(rows), Hq/2, 2 HD] in float64."""
    case = st["case"]
    hd, hkv, hq, tpp = case["hd"], case["hkv"], case["hq"], case["tpp"]
    n = int(st["lens"][s])
    pages = st["table"][s, : -(-n // tpp)].long()
    group = hq // hkv

    def cached(pool, scales, head):
        block = pool[:, head].view(torch.uint8)[pages].view(_FP8) if case["fp8"] else pool[:, head][pages]
        block = block.double()
        if scales is not None:
            block = block * scales[pages, head].double().view(-1, *([1] * (block.dim() - 1)))
        if block.dim() == 4:  # keys [pages, HD/x, TPP, x]
            return block.transpose(1, 2).reshape(-1, hd)[:n]
        return block.transpose(1, 2).reshape(-1, hd)[:n]

    q = st["q"][rows.start:rows.stop].double()
    if case["kind"] == "chunk":
        limit = torch.minimum(st["off"][rows.start:rows.stop], st["lens"][s]).long()
    else:
        limit = torch.tensor([n], device=DEVICE)
    seen = torch.arange(n, device=DEVICE)[None, :] < limit[:, None]
    out = torch.empty((len(rows), hq // 2, 2 * hd), dtype=torch.float64, device=DEVICE)
    for pair in range(hkv // 2):
        key = [cached(st["k"], st["k_scales"], 2 * pair + a) for a in (0, 1)]
        value = torch.cat([cached(st["v"], st["v_scales"], 2 * pair + a) for a in (0, 1)], 1)
        for i in range(pair * group, (pair + 1) * group):
            maps = []
            for a in (0, 1):
                z = (q[:, 2 * i + a] @ key[a].T) * hd ** -0.5
                maps.append(torch.softmax(z.masked_fill(~seen, -math.inf), -1))
            x = (maps[0] - float(st["lam"][i]) * maps[1]) @ value
            if st["weight"] is not None:
                x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * st["weight"].double()
            out[:, i] = x * st["out_scale"]
    return out


def _exact_mrope(st: dict):
    case = st["case"]
    rot, hd, tpp = case["rot"], case["hd"], case["tpp"]
    half, sections = rot // 2, st["sections"]
    if case["interleaved"]:
        axis = [f % len(sections) if f < len(sections) * sections[f % len(sections)] else 0 for f in range(half)]
    else:
        axis = [a for a, count in enumerate(sections) for _ in range(count)]
    table = st["cos_sin"].double()
    cos = torch.stack([table[st["pos"][a].long(), f] for f, a in enumerate(axis)], 1)
    sin = torch.stack([table[st["pos"][a].long(), half + f] for f, a in enumerate(axis)], 1)
    first = list(range(half)) if case["style"] == "neox" else list(range(0, rot, 2))
    second = [d + half for d in first] if case["style"] == "neox" else [d + 1 for d in first]

    def turn(t):
        r = t.double().clone()
        re, im = t[..., first].double(), t[..., second].double()
        r[..., first] = re * cos[:, None] - im * sin[:, None]
        r[..., second] = im * cos[:, None] + re * sin[:, None]
        return r

    q, k, v = turn(st["q"]), turn(st["new_k"]), st["new_v"].double()
    seq, write = st["q2s"].long(), st["write"].long()
    page, slot = st["table"][seq, write // tpp].long(), write % tpp
    kp = torch.zeros(st["k"].shape, dtype=torch.float64, device=DEVICE)
    vp = torch.zeros(st["v"].shape, dtype=torch.float64, device=DEVICE)
    x = kp.shape[-1]
    for c in range(hd // x):
        kp[page, :, c, slot] = k[..., c * x:(c + 1) * x]
    vp[page, :, :, slot] = v
    return kp, vp, q


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "mrope":
        return _exact_mrope(st)
    n = _lengths(case)
    if len(n["keys"]) * (case["hq"] // 2) > 50000:  # too many small products for the time there is
        return None
    out, at = [], 0
    for s, m in enumerate(n["new"]):
        out.append(_exact_sequence(st, s, range(at, at + m)))
        at += m
    return torch.cat(out)
