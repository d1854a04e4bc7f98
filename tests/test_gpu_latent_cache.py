"""The paged latent cache operators (kimi_k3_goalbox_b200/latent_cache.py) against their definitions in 64 bits.

Tolerances are the sums of the roundings that the operators make, per element:
- attend: the output's rounding (2^-8 |out|), the rounding of the probabilities (2^-8 sum p |c|), and the scores' FP32
  accumulation: 576 products in groups of 16 or more make at most 64 additions, 2^-23 of the summed magnitudes each, which
  moves every probability by that part of itself and its share of the sum by as much again;
- lse and mass: the same accumulation, 2^-20 of each weight for the exponential, its argument and lse in base 2, and one
  rounding for each FP32 addition of the sum.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from kimi_k3_goalbox_b200 import latent_cache as lc

SCALE = 192 ** -0.5
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


class Problem:
    """Random queries over a paged cache whose unused slots hold NaN and infinities."""

    def __init__(self, seed, new, lengths, heads, page, spare=3, spread=1.0):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, std=1.0):
            return (torch.randn(shape, generator=gen, device="cuda") * std).to(BF)

        B = len(new)
        self.new, self.lens, self.heads, self.page = new, lengths, heads, page
        self.columns = max(max(-(-n // page) for n in lengths), 1)
        pages = sum(-(-n // page) for n in lengths) + spare
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        self.kv = torch.full((pages, page, 512), math.nan, dtype=BF, device="cuda")
        self.pe = torch.full((pages, page, 64), math.inf, dtype=BF, device="cuda")
        self.table = torch.zeros((B, self.columns), dtype=torch.int32, device="cuda")
        self.entries = []
        at = 0
        for b, n in enumerate(lengths):
            k = -(-n // page)
            self.table[b, :k] = order[at:at + k]
            e = (normal(n, 512), normal(n, 64))
            for p0 in range(0, n, page):
                m = min(page, n - p0)
                self.kv[order[at + p0 // page].long(), :m] = e[0][p0:p0 + m]
                self.pe[order[at + p0 // page].long(), :m] = e[1][p0:p0 + m]
            self.entries.append(e)
            at += k
        self.T = sum(new)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        self.cu = cu
        self.cu_new = torch.tensor(cu, dtype=torch.int32, device="cuda")
        self.lengths = torch.tensor(lengths, dtype=torch.int64, device="cuda")
        self.q_latent = normal(self.T, heads, 512, std=0.5 * spread)
        self.q_pe = normal(self.T, heads, 64, std=spread)
        self.cache = (self.kv, self.pe, self.table)
        self.gen = gen

    def scores(self, b):
        """(scores [n, H, L] with -inf where hidden, their FP32 accumulation error, latents) of sequence b in 64 bits."""
        rows = slice(self.cu[b], self.cu[b + 1])
        c, r = (e.to(F64) for e in self.entries[b])
        q, qr = self.q_latent[rows].to(F64), self.q_pe[rows].to(F64)
        s = (q @ c.T + qr @ r.T) * SCALE
        err = (q.abs() @ c.abs().T + qr.abs() @ r.abs().T) * SCALE * 64 * 2 ** -23
        n, L = self.new[b], self.lens[b]
        sees = L - n + 1 + torch.arange(n, device="cuda")
        hidden = torch.arange(L, device="cuda")[None] >= sees[:, None]
        return s.masked_fill(hidden[:, None], -math.inf), err, c

    def check_attend(self, out, lse):
        for b in range(len(self.new)):
            if self.new[b] == 0:
                continue
            rows = slice(self.cu[b], self.cu[b + 1])
            s, err, c = self.scores(b)
            if s.shape[-1] == 0:
                assert bool((out[rows] == 0).all()) and bool((lse[rows] == -math.inf).all())
                continue
            want = torch.logsumexp(s, -1)
            p = torch.exp(s - want[..., None]).nan_to_num(0.0)
            ref = p @ c
            ds = (p * err).sum(-1)
            empty = want == -math.inf
            assert bool((lse[rows][empty] == -math.inf).all()) and bool((out[rows][empty] == 0).all())
            tol = ds + 2 ** -20 + (s.shape[-1] ** 0.5 + 8) * 2 ** -23 + want.abs() * 2 ** -22
            assert bool(((lse[rows].to(F64) - want).abs() <= tol)[~empty].all()), (b, (lse[rows].to(F64) - want).abs().max())
            mag = p @ c.abs()
            top = err.masked_fill(s == -math.inf, 0.0).amax(-1)[..., None]
            tol = ref.abs() * 2 ** -8 + mag * (1.02 * 2 ** -8 + 2 * top) + 1e-30
            off = (out[rows].to(F64) - ref).abs()
            assert bool((off <= tol)[~empty].all()), (b, float((off / tol)[~empty].max()))

    def check_mass(self, got, before, lse):
        for b in range(len(self.new)):
            L = self.lens[b]
            base = before[b].to(F64)
            assert torch.equal(got[b, L:], before[b, L:])
            if self.new[b] == 0 or L == 0:
                assert torch.equal(got[b], before[b])
                continue
            s, err, _ = self.scores(b)
            l = lse[self.cu[b]:self.cu[b + 1]].to(F64)
            w = torch.exp(s - l[..., None]).nan_to_num(0.0, posinf=math.inf)
            w = w.masked_fill((l == -math.inf)[..., None], 0.0)
            want = base[:L] + w.sum((0, 1))
            arg = (s.abs() + l.abs()[..., None]).nan_to_num(0.0, posinf=0.0) * 2 ** -22
            tol = (w * (err + arg + 2 ** -20)).sum((0, 1)) + (w.sum((0, 1)) + base[:L].abs()) * (self.new[b] * self.heads) * 2 ** -23
            off = (got[b, :L].to(F64) - want).abs()
            assert bool((off <= tol + 1e-37).all()), (b, float((off / (tol + 1e-37)).max()))


CASES = [
    # new tokens, cached positions, heads, page size
    ([1], [1], 12, 16),
    ([1], [517], 12, 16),
    ([1, 1, 1], [33, 1, 160], 1, 16),
    ([1] * 9, [64, 63, 65, 1, 129, 500, 31, 32, 128], 12, 64),
    ([3, 1, 6], [3, 200, 77], 7, 10),            # an odd page size, a fresh prompt
    ([5, 0, 2], [300, 40, 9], 12, 48),           # a sequence without new tokens
    ([4, 3], [2, 0], 12, 8),                     # tokens that see nothing, an empty cache
    ([130], [130], 3, 32),
    ([40, 17], [1000, 17], 12, 64),
    ([2, 1], [700, 1400], 96, 128),
    ([33, 150, 1], [333, 150, 900], 31, 64),
    ([1], [9000], 128, 1),
]


@pytest.mark.parametrize("new,lengths,heads,page", CASES)
def test_attend_and_mass(new, lengths, heads, page):
    x = Problem(11, new, lengths, heads, page)
    out, lse = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
    x.check_attend(out, lse)
    before = torch.rand((len(new), x.columns * page), generator=x.gen, device="cuda")
    got = lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new, mass=before)
    x.check_mass(got, before, lse)
    # the same results again, bit for bit, and in place
    out2, lse2 = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    mine = before.clone()
    assert lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new, mass=mine, out=mine) is mine
    assert torch.equal(mine, got)
    x.check_mass(lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new), torch.zeros_like(before), lse)
