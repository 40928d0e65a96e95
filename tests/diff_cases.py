"""The definition of differential attention over paged pools in 64 bits, with a
bound on what a kernel's roundings may change, for the tests.

u is the most a rounding to the type changes a value, relative to it (bf16
2^-8, fp16 2^-11).  A kernel that keeps everything in fp32 but the
probabilities it multiplies the values with (rounded to the type, and perhaps
summed as rounded) has, for a map with probabilities A and scores s:

  |d score| <= (hd + 4) 2^-24 sum_d |q_d k_d| scale =: ds   (fp32 products and sums)
  |d A| / A <= 2 ds + 2 u  (numerator and normaliser)  + (keys + 16) 2^-24  (fp32 sums)

so x = A1 V - lambda A2 V is off by at most tx = sum_m |lambda_m| rel_m (A_m |V|)
(fp16: plus its subnormal half step 2^-25 per key, of values up to 1 times
the lazy maximum's 2^8 headroom, over an exp-sum that is 2^-8 of that or more).
With the norm, y = c_d x_d / r: r = sqrt(mean x^2 + eps) is off, relative, by at most
|tx| / (r sqrt(2 hd)), so |dy| <= |c| / r (tx + |x| |tx| / (r sqrt(2 hd))) to
first order; half more is allowed for the second order.  The result is rounded
once: u |y|, and half the smallest subnormal.

Over many values with random signs those roundings add as squares: each is
uniform, 0.58 u at most in the mean square, the probabilities' and the
result's; ``check`` therefore also holds the 2-norm of all differences to 2 u
of the 2-norm of the result (random values only).
"""

from __future__ import annotations

import numpy as np
import torch

import proxy_attention_lab as pal
from gpu_util import DEV, announce, dev_bits, dev_index
from oracle import pal_oracle as orc
from pal_cases import PagedCase, make_fused_case, make_paged_case, randn_bits
from test_gpu_fp8_rope import dev_codes, fp8_case

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25}


def k_tokens(pool: np.ndarray) -> np.ndarray:
    """[P, H, HD/x, TPP, x] -> [P, H, TPP, HD]."""
    p, h, c, t, x = pool.shape
    return pool.transpose(0, 1, 3, 2, 4).reshape(p, h, t, c * x)


class Diff:
    """A case on host and device: pools, page table, lengths, rows."""

    def __init__(self, case: PagedCase, queries: np.ndarray, q2s=None, off=None, fp8=False, seed=0, norm=True,
                 out_scale=0.4, lam=None, weight=None, eps=1e-5):
        rng = np.random.default_rng(seed + 77)
        self.case, self.q, self.q2s, self.off, self.fp8 = case, queries, q2s, off, fp8
        hq, hd = case.num_q_heads, case.head_dim
        self.lam = (0.6 + 0.2 * rng.standard_normal(hq // 2)).astype(np.float32) if lam is None else lam
        self.weight = None if not norm else (1 + 0.2 * rng.standard_normal(2 * hd)).astype(np.float32) \
            if weight is None else weight
        self.out_scale, self.eps = out_scale, eps
        if fp8:
            self.kc, self.vc, self.ks, self.vs = fp8_case(case, rng)
        self.dev = dict(
            q=dev_bits(queries, case.dtype), pt=dev_index(case.page_table, torch.uint32), lens=dev_index(case.seq_lens),
            k=dev_codes(self.kc) if fp8 else dev_bits(case.k_pool, case.dtype),
            v=dev_codes(self.vc) if fp8 else dev_bits(case.v_pool, case.dtype),
            lam=torch.from_numpy(self.lam).to(DEV),
            w=None if self.weight is None else torch.from_numpy(self.weight).to(DEV),
            ks=torch.from_numpy(self.ks).to(DEV) if fp8 else None, vs=torch.from_numpy(self.vs).to(DEV) if fp8 else None,
            q2s=None if q2s is None else dev_index(q2s, torch.uint32), off=None if off is None else dev_index(off))

    def run(self, stream=None) -> torch.Tensor:
        d = self.dev
        kw = dict(norm_weight=d["w"], norm_eps=self.eps, out_scale=self.out_scale, k_scales=d["ks"], v_scales=d["vs"])
        if self.q2s is None:
            return pal.paged_differential_attention_decode(d["q"], d["k"], d["v"], d["pt"], d["lens"], d["lam"], stream,
                                                           **kw)
        return pal.paged_differential_attention(d["q"], d["k"], d["v"], d["pt"], d["lens"], d["q2s"], d["off"],
                                                d["lam"], stream, **kw)

    def rows(self):
        """(sequence or None, visible keys) of every output row."""
        c = self.case
        cap = c.page_table.shape[1] * c.tokens_per_page
        if self.q2s is None:
            return [(s, max(0, min(int(n), cap))) for s, n in enumerate(c.seq_lens)]
        return [(int(s), max(0, min(int(c.seq_lens[s]), int(o), cap))) if s < c.num_seqs else (None, 0)
                for s, o in zip(self.q2s, self.off)]

    def expected(self):
        """(y, bound on the error of y) in float64, [rows, Hq/2, 2 HD]."""
        c = self.case
        hq, hkv, hd, tpp, u = c.num_q_heads, c.num_kv_heads, c.head_dim, c.tokens_per_page, U[c.dtype]
        if self.fp8:
            k = k_tokens(orc.fp8_e4m3_decode(self.kc)).astype(np.float64) * self.ks[:, :, None, None]
            v = orc.fp8_e4m3_decode(self.vc).astype(np.float64) * self.vs[:, :, None, None]
        else:
            k = k_tokens(orc.bits_to_f32(c.k_pool, c.dtype)).astype(np.float64)
            v = orc.bits_to_f32(c.v_pool, c.dtype).astype(np.float64)
        q = orc.bits_to_f32(self.q, c.dtype).astype(np.float64)
        rows = self.rows()
        y = np.zeros((len(rows), hq // 2, 2 * hd))
        tol = np.zeros_like(y)
        group = hq // hkv
        num_pages = k.shape[0]
        for s in sorted({s for s, n in rows if n > 0}):
            mine = np.array([i for i, (t, n) in enumerate(rows) if t == s and n > 0])
            lim = torch.tensor([rows[i][1] for i in mine])
            n = int(lim.max())
            ids = c.page_table[s, : -(-n // tpp)].astype(np.int64)
            ok = torch.from_numpy(np.repeat(ids < num_pages, tpp)[:n])  # a page past the pool holds no keys
            ids = np.where(ids < num_pages, ids, 0)
            ks = torch.from_numpy(k[ids].transpose(1, 0, 2, 3).reshape(hkv, -1, hd)[:, :n])
            vs = torch.from_numpy(v[ids].transpose(1, 0, 3, 2).reshape(hkv, -1, hd)[:, :n])
            vis = ok[None, :] & (torch.arange(n)[None, :] < lim[:, None])
            vs = torch.where(vis.any(0)[None, :, None], vs, 0.0)
            ks = torch.where(vis.any(0)[None, :, None], ks, 0.0)
            qs = torch.from_numpy(q[mine])
            for i in range(hq // 2):
                j = i // group
                val = torch.cat([vs[2 * j], vs[2 * j + 1]], 1)
                x, tx = torch.zeros(len(mine), 2 * hd, dtype=torch.float64), 0.0
                for a, f in ((0, 1.0), (1, -float(self.lam[i]))):
                    key = ks[2 * j + a]
                    z = (qs[:, 2 * i + a] @ key.T) * hd ** -0.5
                    z = torch.where(vis, z, -np.inf)
                    top = z.amax(1, keepdim=True)
                    p = torch.exp(z - torch.where(torch.isinf(top), 0.0, top))
                    total = p.sum(1, keepdim=True)
                    p = p / torch.where(total == 0, 1.0, total)
                    x = x + f * (p @ val)
                    ds = (hd + 4) * 2.0 ** -24 * hd ** -0.5 * (qs[:, 2 * i + a].abs() @ key.abs().T).amax(1)
                    rel = 2 * ds + 2 * u + (n + 16) * 2.0 ** -24
                    tx = tx + abs(f) * rel[:, None] * (p @ val.abs())
                    if c.dtype == "f16":
                        tx = tx + abs(f) * 2.0 ** -25 * (vis.double() @ val.abs())
                c_out = self.out_scale * np.ones(2 * hd)
                if self.weight is not None:
                    r = torch.sqrt((x * x).mean(1, keepdim=True) + self.eps)
                    c_out = self.out_scale * self.weight.astype(np.float64)
                    w = torch.from_numpy(c_out)
                    dy = 1.5 * w.abs() / r * (tx + x.abs() * torch.linalg.norm(tx, dim=1, keepdim=True) / (r * (2 * hd) ** 0.5))
                    yy = w * x / r
                else:
                    w = torch.from_numpy(c_out)
                    yy, dy = w * x, w.abs() * tx
                y[mine, i] = yy.numpy()
                tol[mine, i] = (dy + u * (yy.abs() + dy)).numpy() + TINY[c.dtype]
        return y, tol

    def check(self, out: torch.Tensor, what: str, norm2=True):
        y, tol = self.expected()
        got = out.detach().double().cpu().numpy()
        assert got.shape == y.shape, f"{what}: shape {got.shape}"
        empty = [i for i, (s, n) in enumerate(self.rows()) if n == 0]
        assert not got[empty].any(), f"{what}: rows without keys must be zero"
        far = np.abs(got - y)
        bad = ~(far <= tol)
        assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} outside the bound, first at {np.argwhere(bad)[0]}: "
                               f"got {got[bad][0]}, want {y[bad][0]} within {tol[bad][0]:.3g}")
        size = np.linalg.norm(y)
        rel = np.linalg.norm(got - y) / size if size else 0.0
        worst = float((far / np.maximum(tol, 1e-300)).max()) if y.size else 0.0
        announce(f"{what}: 2-norm of the error {rel:.2e} ({rel / U[self.case.dtype]:.2f} u), worst error / bound {worst:.3f}")
        if norm2:
            assert rel <= 2 * U[self.case.dtype], f"{what}: 2-norm of the error {rel:.3e} over 2 u"


def decode_case(seed, lens, hq, hkv, hd, tpp, dtype, fp8=False, extra_rows=0, width=None, **kw) -> Diff:
    case = make_paged_case(seed, lens, hq, hkv, hd, tpp, dtype, width=width)
    q = randn_bits(np.random.default_rng(seed + 1), (len(lens) + extra_rows, hq, hd), dtype)
    return Diff(case, q, fp8=fp8, seed=seed, **kw)


def chunk_case(seed, decode_lens, chunks, hq, hkv, hd, tpp, dtype, fp8=False, block=64, **kw) -> Diff:
    fc = make_fused_case(seed, decode_lens, chunks, hq, hkv, hd, tpp, dtype, block=block)
    return Diff(fc.case, fc.queries, fc.q2seq, fc.q_offset, fp8=fp8, seed=seed, **kw)
