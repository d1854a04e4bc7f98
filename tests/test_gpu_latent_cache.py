"""The paged latent cache operators (kimi_k3_goalbox_b200/latent_cache.py) against their definitions in 64 bits.

Tolerances are the sums of the roundings that the operators make, per element:
- attend: the output's rounding (2^-8 |out|), the rounding of the probabilities (2^-8 sum p |c|), and the scores' FP32
  accumulation: 576 products in groups of 16 or more make at most 64 additions, 2^-23 of the summed magnitudes each, which
  moves every probability by that part of itself and its share of the sum by as much again;
- append: the mean of squares is a sum of 512 FP32 terms, rsqrt and two products follow (2^-20 in all is ample: 512 terms
  in a tree of 9 additions, half of that error after the root), then one rounding to BF16 (2^-8);
- evict: moves and copies, exact;
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
        self.table = torch.full((B, self.columns), -1, dtype=torch.int32, device="cuda")   # no page behind the end
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

    def check_attend(self, out, lse, first=0):
        for b in range(first, len(self.new)):
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
    ([1] * 300, [1 + (37 * i) % 400 for i in range(300)], 4, 16),   # many sequences
    ([1], [6000], 16, 64),                       # one tile over many workers
    ([2, 300], [9000, 2500], 64, 32),            # single tokens next to a chunk
    ([1], [64], 128, 64),
    ([1, 2, 1], [95, 96, 97], 5, 32),
    ([1], [100003], 12, 64),
    ([2], [70001], 40, 16),
    ([3, 3], [65, 64], 21, 64),                  # few rows in all
]


@pytest.mark.parametrize("new,lengths,heads,page", CASES)
def test_attend_and_mass(new, lengths, heads, page):
    x = Problem(11, new, lengths, heads, page)
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new, error_word=error)
    x.check_attend(out, lse)
    before = torch.rand((len(new), x.columns * page), generator=x.gen, device="cuda")
    got = lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new, mass=before, error_word=error)
    x.check_mass(got, before, lse)
    assert error.item() == 0
    # the same results again, bit for bit, and in place
    out2, lse2 = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    mine = before.clone()
    assert lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new, mass=mine, out=mine) is mine
    assert torch.equal(mine, got)
    x.check_mass(lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new), torch.zeros_like(before), lse)


def test_attend_rescales_when_later_scores_are_larger():
    """Scores that rise by far more than the exponent range of a probability from unit to unit, and fall again."""
    for heads, new in ((12, 1), (40, 7)):
        x = Problem(3, [new], [3000], heads, 64)
        up = torch.linspace(0.01, 12.0, 3000, device="cuda")
        up[2000:] = up[:1000].flip(0)
        c = (x.entries[0][0].float() * up[:, None]).to(BF)
        x.entries[0] = (c, x.entries[0][1])
        for p0 in range(0, 3000, 64):
            m = min(64, 3000 - p0)
            x.kv[x.table[0, p0 // 64].long(), :m] = c[p0:p0 + m]
        out, lse = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
        x.check_attend(out, lse)
        before = torch.zeros((1, x.columns * 64), device="cuda")
        x.check_mass(lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new), before, lse)


@pytest.mark.parametrize("heads,new", [(12, [1, 1]), (24, [9, 30])])
@pytest.mark.parametrize("scale", [0.0, -0.05, 0.25])
def test_scales(heads, new, scale):
    x = Problem(5, new, [300, 77], heads, 16)
    out, lse = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new, scale=scale)
    for b in range(2):
        rows = slice(x.cu[b], x.cu[b + 1])
        c, r = (e.to(F64) for e in x.entries[b])
        q, qr = x.q_latent[rows].to(F64), x.q_pe[rows].to(F64)
        s = (q @ c.T + qr @ r.T) * scale
        err = (q.abs() @ c.abs().T + qr.abs() @ r.abs().T) * abs(scale) * 64 * 2 ** -23
        sees = x.lens[b] - x.new[b] + 1 + torch.arange(x.new[b], device="cuda")
        s = s.masked_fill((torch.arange(x.lens[b], device="cuda")[None] >= sees[:, None])[:, None], -math.inf)
        p = torch.softmax(s, -1)
        tol = (p @ c).abs() * 2 ** -8 + (p @ c.abs()) * (1.02 * 2 ** -8 + 2 * err.amax(-1)[..., None])
        assert bool(((out[rows].to(F64) - p @ c).abs() <= tol).all())
        assert bool(((lse[rows].to(F64) - torch.logsumexp(s, -1)).abs() <= (p * err).sum(-1) + 2 ** -18).all())


def _pool(x, wide=576 + 64, extra=2):
    """The cache of `x` as slices of one pool whose rows hold latent and rope values, with columns and pages between."""
    pages, page = x.kv.shape[:2]
    pool = torch.full((pages * extra, page, wide), math.nan, dtype=BF, device="cuda")
    pool[::extra, :, :512] = x.kv
    pool[::extra, :, 512:576] = x.pe
    table = torch.full((x.table.shape[0], x.table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    table[:, :x.table.shape[1]] = x.table
    return pool, (pool[::extra, :, :512], pool[::extra, :, 512:576], table[:, :x.table.shape[1]])


@pytest.mark.parametrize("heads,new", [(12, [1, 1, 1]), (12, [40, 3, 1])])
@pytest.mark.parametrize("page", [64, 6])
def test_strided_arguments_give_the_same(heads, new, page):
    x = Problem(7, new, [400, 90, 33], heads, page)
    out, lse = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
    mass = lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new)
    _, cache = _pool(x)
    T = x.T
    both = torch.empty((T, heads, 576), dtype=BF, device="cuda")
    both[..., :512], both[..., 512:] = x.q_latent, x.q_pe
    by_head = both.transpose(0, 1).contiguous().transpose(0, 1)      # heads outermost
    apart = torch.zeros((T, heads + 2, 584), dtype=BF, device="cuda")
    apart[:, :heads, :576] = both
    odd = torch.zeros(T * heads * 576 + 1, dtype=BF, device="cuda")[1:].view(T, heads, 576)   # not 16-byte aligned
    odd.copy_(both)
    for q in (both, by_head, apart[:, :heads], odd):
        out2, lse2 = lc.attend(q[..., :512], q[..., 512:576], *cache, x.lengths, x.cu_new)
        assert torch.equal(out, out2) and torch.equal(lse, lse2)
        before = torch.rand((3, cache[2].shape[1] * page + 7), device="cuda")[:, :cache[2].shape[1] * page]
        got = lc.attention_mass(q[..., :512], q[..., 512:576], lse2, *cache, x.lengths, x.cu_new, mass=before)
        x.check_mass(got, before, lse2)
    assert torch.equal(mass, lc.attention_mass(both[..., :512], both[..., 512:], lse, *cache, x.lengths, x.cu_new))


@pytest.mark.parametrize("heads,new", [(12, [1, 1, 1]), (24, [20, 9, 4])])
def test_sequences_that_share_pages(heads, new):
    """Three sequences of one prefix: the same pages in three rows of the table, and one of them twice in a row."""
    x = Problem(8, new, [150, 160, 170], heads, 16)
    x.table[1:, :9] = x.table[0, :9]
    x.table[2, 3] = x.table[2, 5]
    for b in (1, 2):
        for e, first in zip(x.entries[b], x.entries[0]):
            e[:144] = first[:144]
    for e in x.entries[2]:
        e[48:64] = e[80:96].clone()
    out, lse = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
    x.check_attend(out, lse)
    before = torch.zeros((3, x.columns * 16), device="cuda")
    x.check_mass(lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new), before, lse)


@pytest.mark.parametrize("heads,new", [(12, [1, 1]), (24, [30, 9])])
def test_rows_behind_the_last_sequence_stay(heads, new):
    x = Problem(9, new, [200, 60], heads, 16)
    pad = 5
    q = torch.full((x.T + pad, heads, 512), math.nan, dtype=BF, device="cuda")
    qr = torch.full((x.T + pad, heads, 64), math.nan, dtype=BF, device="cuda")
    q[:x.T], qr[:x.T] = x.q_latent, x.q_pe
    out = torch.full((x.T + pad, heads, 512), 7.0, dtype=BF, device="cuda")
    lse = torch.full((x.T + pad, heads), 7.0, device="cuda")
    assert lc.attend(q, qr, *x.cache, x.lengths, x.cu_new, out=out, lse=lse)[0] is out
    assert bool((out[x.T:] == 7).all()) and bool((lse[x.T:] == 7).all())
    x.check_attend(out[:x.T], lse[:x.T])
    before = torch.zeros((2, x.columns * 16), device="cuda")
    x.check_mass(lc.attention_mass(q, qr, lse, *x.cache, x.lengths, x.cu_new), before, lse[:x.T])


def test_no_tokens():
    x = Problem(2, [0, 0], [5, 0], 4, 16)
    out, lse = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
    assert out.shape == (0, 4, 512) and lse.shape == (0, 4)
    before = torch.rand((2, x.columns * 16), device="cuda")
    assert torch.equal(lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new, mass=before), before)
    assert not lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new).any()
    raw = torch.zeros((0, 576), dtype=BF, device="cuda")
    assert lc.append(raw, torch.ones(512, dtype=BF, device="cuda"), *x.cache, x.lengths, x.cu_new).tolist() == [5, 0]


@pytest.mark.parametrize("heads,new,page", [(12, [1, 1, 1], 16), (24, [30, 9, 4], 16), (12, [1, 1, 1], 10), (24, [30, 9, 4], 10)])
def test_bad_pages_and_lengths_are_reported_and_not_followed(heads, new, page):
    x = Problem(13, new, [200, 60, 50], heads, page)
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    ok, ok_lse = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new, error_word=error)
    lc.attention_mass(x.q_latent, x.q_pe, ok_lse, *x.cache, x.lengths, x.cu_new, error_word=error)
    assert error.item() == 0
    others = slice(x.cu[1], x.T)
    for bad in (-1, x.kv.shape[0], 2 ** 31 - 1, -2 ** 31):
        table = x.table.clone()
        table[0, 2] = bad
        for run in range(2):
            error.zero_()
            if run == 0:
                out, lse = lc.attend(x.q_latent, x.q_pe, x.kv, x.pe, table, x.lengths, x.cu_new, error_word=error)
                assert torch.equal(out[others], ok[others]) and torch.equal(lse[others], ok_lse[others])
                # the page reads as zeros
                held = x.entries[0]
                x.entries[0] = tuple(e.clone() for e in held)
                for e in x.entries[0]:
                    e[2 * page:3 * page] = 0
                x.check_attend(out, lse)
                x.entries[0] = held
            else:
                lc.attention_mass(x.q_latent, x.q_pe, ok_lse, x.kv, x.pe, table, x.lengths, x.cu_new, error_word=error)
            assert error.item() != 0
    for length in (-5, x.columns * page + 1, 2 ** 40, -2 ** 40, 2 ** 63 - 1):
        lengths = x.lengths.clone()
        lengths[0] = length
        error.zero_()
        out, lse = lc.attend(x.q_latent, x.q_pe, *x.cache, lengths, x.cu_new, error_word=error)
        torch.cuda.synchronize()
        assert error.item() != 0
        x.check_attend(out, lse, first=1)   # not bit for bit: every length has a part in how the work is split
        error.zero_()
        lc.attention_mass(x.q_latent, x.q_pe, ok_lse, *x.cache, lengths, x.cu_new, error_word=error)
        torch.cuda.synchronize()
        assert error.item() != 0


def test_outputs_that_do_not_fit_are_refused():
    x = Problem(15, [1, 1], [20, 9], 4, 16)
    args = (x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
    out, lse = lc.attend(*args)
    for bad in (out[:1], out.float(), torch.empty((2, 512, 4), dtype=BF, device="cuda").transpose(1, 2), out.cpu()):
        with pytest.raises(ValueError):
            lc.attend(*args, out=bad)
    for bad in (lse[:, :2], lse.to(BF), lse.cpu()):
        with pytest.raises(ValueError):
            lc.attend(*args, lse=bad)
    margs = (x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new)
    wide = torch.zeros((2, 2 * 32), device="cuda")
    flat = torch.zeros(2 * 32 + 1, device="cuda")
    for mass, result in ((wide[:, :32], wide.view(-1)[:64].view(2, 32)), (flat[1:].view(2, 32), flat[:-1].view(2, 32))):
        with pytest.raises(ValueError, match="overlap"):
            lc.attention_mass(*margs, mass=mass, out=result)
    for scale in (math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            lc.attend(*args, scale=scale)
    with pytest.raises(ValueError, match="heads"):
        lc.attend(torch.zeros((2, 129, 512), dtype=BF, device="cuda"), torch.zeros((2, 129, 64), dtype=BF, device="cuda"), *args[2:])
    mass = torch.zeros((2, 32), device="cuda")
    for budget, sinks, recent in ((0, 0, 0), (33, 0, 0), (8, 0, -1), (8, -1, 0), (8, 1 << 40, 0)):
        with pytest.raises(ValueError):
            lc.evict(*x.cache, x.lengths, mass, budget, sinks=sinks, recent=recent)
    with pytest.raises(ValueError, match="hold the budget"):
        lc.evict(*x.cache, x.lengths, mass, 20, dst_table=x.table[:, :1])
    with pytest.raises(ValueError, match="error_word"):
        lc.evict(*x.cache, x.lengths, mass, 20, error_word=torch.zeros(1, device="cuda"))


# --- append ----------------------------------------------------------------------------------------------------

def _appended(raw, weight, eps):
    c = raw[:, :512].to(F64)
    return c * torch.rsqrt((c * c).mean(-1, keepdim=True) + eps) * weight.to(F64)


@pytest.mark.parametrize("new,lengths,page", [([1], [0], 16), ([1, 1, 0, 1], [0, 15, 7, 31], 16), ([33, 0, 70], [5, 9, 100], 10),
                                               ([300], [1], 1), ([1] * 200, list(range(200)), 64)])
@pytest.mark.parametrize("sliced", [False, True])
def test_append(new, lengths, page, sliced):
    total = [n + m for n, m in zip(new, lengths)]
    x = Problem(17, new, total, 1, page)
    cache = _pool(x)[1] if sliced else x.cache
    kv0, pe0 = cache[0].clone(), cache[1].clone()
    T = x.T
    gen = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn((T + 3, 592 if sliced else 576), generator=gen, device="cuda").to(BF)   # three rows behind the last
    raw = wide[:, :576]
    weight = torch.rand(512, generator=gen, device="cuda").to(BF)
    before = torch.tensor(lengths, device="cuda")
    after = lc.append(raw, weight, *cache, before, x.cu_new, eps=1e-5)
    assert after.tolist() == total and before.tolist() == lengths
    want = _appended(raw, weight, 1e-5)
    touched = torch.zeros(kv0.shape[:2], dtype=torch.bool, device="cuda")
    for b, n in enumerate(new):
        pos = torch.arange(lengths[b], total[b], device="cuda")
        pages, slots = cache[2][b, pos // page].long(), pos % page
        rows = slice(x.cu[b], x.cu[b + 1])
        off = (cache[0][pages, slots].to(F64) - want[rows]).abs()
        assert bool((off <= want[rows].abs() * (2 ** -8 + 2 ** -20) + 1e-38).all())
        assert torch.equal(cache[1][pages, slots], raw[rows, 512:])
        touched[pages, slots] = True
    assert torch.equal(cache[0][~touched].view(torch.int16), kv0[~touched].view(torch.int16))
    assert torch.equal(cache[1][~touched].view(torch.int16), pe0[~touched].view(torch.int16))


def test_append_reports_what_does_not_fit():
    x = Problem(19, [4, 2, 2], [30, 20, 10], 1, 16)
    kv0 = x.kv.clone()
    raw = torch.randn((8, 576), device="cuda").to(BF)
    weight = torch.ones(512, dtype=BF, device="cuda")
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    cap = x.columns * 16
    lengths = torch.tensor([cap - 1, -3, 8], device="cuda")   # three of the first one's tokens lie behind the table
    table = x.table.clone()
    table[1] = -7
    lc.append(raw, weight, x.kv, x.pe, table, lengths, x.cu_new, error_word=error)
    torch.cuda.synchronize()
    assert error.item() != 0
    want = _appended(raw, weight, 1e-6)
    last = x.kv[table[0, -1].long(), 15]
    assert bool(((last.to(F64) - want[0]).abs() <= want[0].abs() * (2 ** -8 + 2 ** -20)).all())
    got = x.kv[table[2, 0].long(), 8:10]
    assert bool(((got.to(F64) - want[6:8]).abs() <= want[6:8].abs() * (2 ** -8 + 2 ** -20)).all())
    same = torch.ones(kv0.shape[:2], dtype=torch.bool, device="cuda")
    same[table[0, -1].long(), 15] = False
    same[table[2, 0].long(), 8:10] = False
    assert torch.equal(x.kv[same].view(torch.int16), kv0[same].view(torch.int16))
    # lengths whose sum with the new tokens passes 64 bits
    kv0 = x.kv.clone()
    for length in (2 ** 63 - 1, 2 ** 62, cap + 1, cap, -2 ** 63):
        error.zero_()
        lengths = torch.tensor([length, length, length], device="cuda")
        after = lc.append(raw, weight, x.kv, x.pe, table, lengths, x.cu_new, error_word=error)
        assert after.tolist() == ([cap] * 3 if length > 0 else [4, 2, 2]) and error.item() != 0
        if length > 0:
            assert torch.equal(x.kv.view(torch.int16), kv0.view(torch.int16))


# --- evict -----------------------------------------------------------------------------------------------------

def _kept(mass, length, budget, sinks, recent):
    """Positions that stay, ascending: the protected ones, then by weight, the lowest index among equal ones."""
    keep = min(length, budget)
    if keep == length:
        return list(range(length))
    m = mass[:length].tolist()
    guarded = [p for p in range(length) if p < sinks or p >= length - recent]
    rest = [p for p in range(length) if sinks <= p < length - recent]
    rest.sort(key=lambda p: (0 if math.isnan(m[p]) else 1, 0.0 if math.isnan(m[p]) else -m[p], p))
    return sorted((guarded + rest)[:keep])


def _mass(kind, B, n, gen):
    if kind == "equal":
        return torch.full((B, n), 0.25, device="cuda")
    if kind == "few":
        return torch.randint(0, 3, (B, n), generator=gen, device="cuda").float() * 0.5 - 0.5     # zeros of both signs
    m = torch.randn((B, n), generator=gen, device="cuda").exp()
    if kind == "odd":
        m *= torch.randint(-1, 2, (B, n), generator=gen, device="cuda")
        m[torch.rand((B, n), generator=gen, device="cuda") < 0.1] = math.nan
        m[torch.rand((B, n), generator=gen, device="cuda") < 0.05] = math.inf
        m[torch.rand((B, n), generator=gen, device="cuda") < 0.05] = -math.inf
        m[:, ::7] = 1e-42
    return m


EVICTIONS = [
    # lengths, page, budget, sinks, recent
    ([0, 1, 5, 16, 17, 33], 16, 16, 0, 0),
    ([100, 64, 63, 65], 16, 64, 4, 8),
    ([1000, 37, 999], 10, 250, 0, 100),
    ([2100], 64, 1, 0, 0),
    ([700, 300], 48, 300, 150, 150),      # nothing but protected positions
    ([513, 40], 1, 512, 1, 0),
    ([60, 9, 4, 5], 16, 4, 4, 1),         # more protected positions than the budget
    ([100, 50, 3], 16, 10, 7, 20),
    ([40, 10], 8, 5, 9, 1000),
    ([64, 30], 16, 16, 0, 16),
    ([40000, 33000, 20], 64, 20000, 5, 9),
]


@pytest.mark.parametrize("lengths,page,budget,sinks,recent", EVICTIONS)
@pytest.mark.parametrize("kind", ["spread", "few", "equal", "odd"])
@pytest.mark.parametrize("place", ["pages", "in place"])
def test_evict(lengths, page, budget, sinks, recent, kind, place):
    B = len(lengths)
    x = Problem(23, [0] * B, lengths, 1, page, spare=B * -(-budget // page) + 2)
    cap = x.columns * page
    if cap < budget:
        pytest.skip("the budget exceeds the capacity, which is refused")
    mass = _mass(kind, B, cap + 3, x.gen)[:, :cap]
    dst = None
    if place == "pages":
        k = -(-budget // page)
        used = set(x.table[b, i].item() for b in range(B) for i in range(-(-lengths[b] // page)))
        free = [p for p in range(x.kv.shape[0]) if p not in used][:B * k]
        dst = torch.tensor(free, dtype=torch.int32, device="cuda").view(B, k)
    kv0, pe0 = x.kv.clone(), x.pe.clone()
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    new_lengths, new_mass, kept = lc.evict(*x.cache, x.lengths, mass, budget, sinks=sinks, recent=recent, dst_table=dst,
                                           error_word=error)
    assert error.item() == 0
    table = x.table if dst is None else dst
    written = torch.zeros(kv0.shape[:2], dtype=torch.bool, device="cuda")
    for b in range(B):
        want = _kept(mass[b], lengths[b], budget, sinks, recent)
        n = len(want)
        assert new_lengths[b].item() == n and kept[b].tolist() == want + [-1] * (budget - n)
        at = torch.tensor(want, dtype=torch.int64, device="cuda")
        assert torch.equal(new_mass[b, :n].view(torch.int32), mass[b, at].view(torch.int32)) and not new_mass[b, n:].any()
        pos = torch.arange(n, device="cuda")
        pages, slots = table[b, pos // page].long(), pos % page
        assert torch.equal(x.kv[pages, slots], x.entries[b][0][at]) and torch.equal(x.pe[pages, slots], x.entries[b][1][at])
        written[pages, slots] = True
    assert torch.equal(x.kv[~written].view(torch.int16), kv0[~written].view(torch.int16))
    assert torch.equal(x.pe[~written].view(torch.int16), pe0[~written].view(torch.int16))


def test_evict_reports_bad_pages_and_lengths():
    for place in (False, True):
        x = Problem(29, [0, 0], [100, 90], 1, 16, spare=8)
        mass = torch.rand((2, x.columns * 16), device="cuda")
        used = set(x.table[0, :7].tolist() + x.table[1, :6].tolist())
        free = [p for p in range(x.kv.shape[0]) if p not in used]
        dst = torch.tensor(free[:8], dtype=torch.int32, device="cuda").view(2, 4) if place else None
        table = x.table.clone()
        table[0] = x.kv.shape[0]
        lengths = torch.tensor([100, -1], device="cuda")
        kv0 = x.kv.clone()
        error = torch.zeros(1, dtype=torch.int32, device="cuda")
        new_lengths, new_mass, kept = lc.evict(x.kv, x.pe, table, lengths, mass, 64, dst_table=dst, error_word=error)
        torch.cuda.synchronize()
        assert error.item() != 0 and new_lengths.tolist() == [64, 0]
        assert kept[0].tolist() == _kept(mass[0], 100, 64, 0, 0) and kept[1].tolist() == [-1] * 64
        assert torch.equal(x.kv.view(torch.int16), kv0.view(torch.int16)) and not new_mass[1].any()


# --- larger pools, streams, graphs -----------------------------------------------------------------------------

def test_offsets_beyond_32_bits():
    """A pool of more than 2^31 latent values (and 2^32 bytes): its last pages are used."""
    pages, page = 66000, 64
    kv = torch.zeros((pages, page, 512), dtype=BF, device="cuda")
    pe = torch.zeros((pages, page, 64), dtype=BF, device="cuda")
    for new, heads in (([1, 1], 12), ([20, 40], 24)):
        x = Problem(31, new, [200, 100], heads, page, spare=4)
        n = x.kv.shape[0]
        kv[-n:], pe[-n:] = x.kv, x.pe
        table = x.table + (pages - n)
        out, lse = lc.attend(x.q_latent, x.q_pe, kv, pe, table, x.lengths, x.cu_new)
        x.check_attend(out, lse)
        mass = lc.attention_mass(x.q_latent, x.q_pe, lse, kv, pe, table, x.lengths, x.cu_new)
        x.check_mass(mass, torch.zeros_like(mass), lse)
        new_lengths, _, kept = lc.evict(kv, pe, table, x.lengths, mass, 64)
        for b in range(2):
            assert torch.equal(kv[table[b, 0].long()], x.entries[b][0][kept[b].long()])
        raw = torch.randn((x.T, 576), device="cuda").to(BF)
        lc.append(raw, torch.ones(512, dtype=BF, device="cuda"), kv, pe, table, new_lengths, x.cu_new)
        assert torch.equal(pe[table[0, 1].long(), 0], raw[0, 512:])


def _serve(x, raw, weight, lengths, dst, heads):
    """What a serving loop enqueues: append, attend, accumulate, cut down."""
    after = lc.append(raw, weight, *x.cache, lengths, x.cu_new)
    out, lse = lc.attend(x.q_latent, x.q_pe, *x.cache, after, x.cu_new)
    mass = lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, after, x.cu_new)
    return (out, lse, mass) + lc.evict(*x.cache, after, mass, 48, sinks=2, recent=4, dst_table=dst)


@pytest.mark.parametrize("heads,new", [(12, [1, 1, 1]), (24, [20, 5, 1])])
def test_streams_and_graphs(heads, new):
    """On a stream of their own, and captured into two graphs that are replayed in turn with new inputs."""
    total = [150, 60, 40]
    x = Problem(37, new, total, heads, 16, spare=12)
    used = set(x.table[b, i].item() for b in range(3) for i in range(-(-total[b] // 16)))
    dst = torch.tensor([p for p in range(x.kv.shape[0]) if p not in used][:9], dtype=torch.int32, device="cuda").view(3, 3)
    weight = torch.rand(512, generator=x.gen, device="cuda").to(BF)
    raw = torch.randn((x.T, 576), generator=x.gen, device="cuda").to(BF)
    lengths = torch.tensor([n - m for n, m in zip(total, new)], device="cuda")
    want = _serve(x, raw, weight, lengths, dst, heads)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _serve(x, raw, weight, lengths, dst, heads)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = _serve(x, raw, weight, lengths, dst, heads)
        graphs.append((g, res))
    for i in range(6):
        raw.copy_(torch.randn((x.T, 576), generator=x.gen, device="cuda").to(BF))
        lengths.copy_(torch.tensor([n - m - 3 * i for n, m in zip(total, new)], device="cuda"))
        x.q_latent.copy_((torch.randn(x.q_latent.shape, generator=x.gen, device="cuda") * 0.5).to(BF))
        g, res = graphs[i % 2]
        g.replay()
        got = [t.clone() for t in res]
        other = [t.clone() for t in graphs[1 - i % 2][1]]
        want = _serve(x, raw, weight, lengths, dst, heads)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        if i:   # the other graph's results are its own
            assert all(torch.equal(a, b) for a, b in zip(other, last))
        last = got


def test_calls_on_two_streams_at_once():
    xs = [Problem(41 + i, [1] * 8 if i else [60, 9], [900] * 8 if i else [700, 300], 12, 64) for i in range(2)]
    want = [lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (x, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                got[i].append(lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


# --- with the decode step --------------------------------------------------------------------------------------

def test_prefill_evict_and_decode_with_the_step():
    """Prompts are appended to every MLA layer's cache, attended and cut down in place; the decode step continues the
    cut caches, graded against the oracle on what the caches hold then, and its entry is attended after it."""
    from kimi_k3_goalbox_b200.runtime import StepContext
    from oracle import kimi_oracle as ko
    from tests import gpu_helpers as gh
    from tests import test_gpu_append as ta

    B, capacity, page, budget, heads = 3, 32, 8, 12, 2
    case = gh.small_case(B, context=capacity)
    p = case["params"]
    prompts = [20, 12, 5]
    cu = torch.tensor([0, 20, 32, 37], dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(43)
    with torch.inference_mode():
        values = ko.make_inputs(case, 47, "cuda")
        conv, rec = ta._stacked_states(case, values)
        zeros = torch.zeros(B, dtype=torch.int64, device="cuda")
        views = {}
        for l in ko.mla_layer_ids(case):
            view = views[l] = lc.paged_view(values[f"l{l}_kv_cache"], values[f"l{l}_pe_cache"], page)
            raw = torch.randn((37, 576), generator=gen, device="cuda").to(BF)
            weight = torch.ones(512, dtype=BF, device="cuda")
            lengths = lc.append(raw, weight, *view, zeros, cu)
            q = (torch.randn((37, heads, 512), generator=gen, device="cuda") * 0.5).to(BF)
            qr = torch.randn((37, heads, 64), generator=gen, device="cuda").to(BF)
            out, lse = lc.attend(q, qr, *view, lengths, cu)
            mass = lc.attention_mass(q, qr, lse, *view, lengths, cu)
            total = torch.tensor([n * heads for n in prompts], device="cuda", dtype=F64)
            # the weights of a row add up to one; the summed magnitudes of a score's products stay below 2^5, so that
            # the two operators' scores differ by 2 * 2^5 * 64 * 2^-23 = 2^-11 at most
            assert bool(((mass.to(F64).sum(1) - total).abs() <= total * 2 ** -11).all())
            before = [values[f"l{l}_kv_cache"][b].clone() for b in range(B)]
            new_lengths, _, kept = lc.evict(*view, lengths, mass, budget, sinks=1, recent=2)
            assert new_lengths.tolist() == [12, 12, 5]
            for b in range(B):
                want = _kept(mass[b], prompts[b], budget, 1, 2)
                assert kept[b, :len(want)].tolist() == want
                assert torch.equal(values[f"l{l}_kv_cache"][b, :len(want)], before[b][want])
        values["token"] = torch.randint(0, p["vocab"], (B,), generator=gen, device="cuda")
        values["reset"] = torch.zeros(B, dtype=torch.bool, device="cuda")
        held = {k: (v.clone() if k.endswith(("kv_cache", "pe_cache", "conv_state", "recurrent_state")) else v) for k, v in values.items()}
        ctx = StepContext(case)
        try:
            outputs = ctx.allocate_outputs()
            outputs["conv_state"], outputs["recurrent_state"] = conv, rec
            ctx.step_append(values, outputs, new_lengths)
            torch.cuda.synchronize()
            ctx.check()
            actual = {k: v.clone() for k, v in outputs.items()}
        finally:
            ctx.close()
        assert actual["cache_length"].tolist() == [13, 13, 6]
        ta._grade_rows(case, held, actual, [0, 1], 12)
        ta._grade_rows(case, held, actual, [2], 5)
        one = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
        for i, l in enumerate(views):
            # the last position is the step's own entry: a query that looks at nothing else returns it
            q = actual["kv_write"][i][:, None] * 8
            out, lse = lc.attend(q, torch.zeros((B, 1, 64), dtype=BF, device="cuda"), *views[l], actual["cache_length"], one, scale=1.0)
            assert torch.equal(out[:, 0], actual["kv_write"][i])


def test_attend_agrees_with_the_step_oracle():
    """The absorbed queries and the attended latents of the oracle's MLA layers, with its new entries in the cache."""
    from oracle import kimi_oracle as ko
    from tests import gpu_helpers as gh

    B, context = 3, 24
    case = gh.small_case(B, context=context)
    with torch.inference_mode():
        values = ko.make_inputs(case, 53, "cuda")
        values["reset"] = torch.zeros(B, dtype=torch.bool, device="cuda")
        trace = {}
        outputs = ko.reference(case, values, serial=True, trace=trace)
        one = torch.arange(B + 1, dtype=torch.int32, device="cuda")
        lengths = torch.full((B,), context + 1, dtype=torch.int64, device="cuda")
        for i, l in enumerate(ko.mla_layer_ids(case)):
            kv = torch.full((B, 32, 512), math.nan, dtype=BF, device="cuda")
            pe = torch.full((B, 32, 64), math.nan, dtype=BF, device="cuda")
            kv[:, :context], pe[:, :context] = values[f"l{l}_kv_cache"], values[f"l{l}_pe_cache"]
            kv[:, context], pe[:, context] = outputs["kv_write"][i], outputs["pe_write"][i]
            q, want = trace[f"l{l}_absorbed"], trace[f"l{l}_attn_latent"].to(F64)
            out, lse = lc.attend(q, trace[f"l{l}_q"][..., 128:], *lc.paged_view(kv, pe, 8), lengths, one)
            c = kv[:, :context + 1].to(F64)
            s = (q.to(F64) @ c.mT + trace[f"l{l}_q"][..., 128:].to(F64) @ pe[:, :context + 1].to(F64).mT) * SCALE
            mag = torch.softmax(s, -1) @ c.abs()
            # both sides round the probabilities and the result once: 2^-8 of the summed magnitudes and of the value each
            assert bool(((out.to(F64) - want).abs() <= 2 * 2 ** -8 * 1.05 * (mag + want.abs())).all())


# --- caches with room to grow --------------------------------------------------------------------------------------

ROOMY = [
    # new tokens, cached positions, heads, page size, positions that the table has room for
    ([1], [517], 12, 16, 8192),
    ([1], [100], 12, 64, 1024),
    ([1], [500], 12, 64, 131072),
    ([1] * 16, [600] * 16, 12, 64, 8192),
    ([1] * 8, [300] * 8, 12, 64, 8192),
    ([1, 0], [300, 229], 12, 16, 4096),      # a sequence without new tokens beside a short one
    ([1, 1], [300, 300], 12, 8, 4096),
    ([40, 3], [333, 90], 96, 10, 8190),
    ([1, 2, 0, 1], [1, 2, 0, 3000], 1, 1, 5000),
    ([1] * 200, [1 + (53 * i) % 300 for i in range(200)], 3, 32, 1024),   # more sequences than CTAs
    ([0, 0], [90, 0], 4, 16, 2048),          # nothing new at all
]


@pytest.mark.parametrize("new,lengths,heads,page,capacity", ROOMY)
def test_mass_with_room_behind_the_lengths(new, lengths, heads, page, capacity):
    """Every position behind a length keeps its mass (zero without one), however far the table goes on."""
    x = Problem(61, new, lengths, heads, page)
    table = torch.full((len(new), capacity // page), -1, dtype=torch.int32, device="cuda")
    table[:, :x.columns] = x.table
    cache = (x.kv, x.pe, table)
    out, lse = lc.attend(x.q_latent, x.q_pe, *cache, x.lengths, x.cu_new)
    x.check_attend(out, lse)
    args = (x.q_latent, x.q_pe, lse, *cache, x.lengths, x.cu_new)
    before = torch.rand((len(new), capacity), generator=x.gen, device="cuda")
    for mass in (None, before):
        got = torch.full((len(new), capacity), math.nan, device="cuda")
        assert lc.attention_mass(*args, mass=mass, out=got) is got
        x.check_mass(got, torch.zeros_like(before) if mass is None else mass, lse)
    mine = before.clone()
    lc.attention_mass(*args, mass=mine, out=mine)
    assert torch.equal(mine, got)


def test_append_writes_nothing_for_a_negative_length():
    """A length below zero is reported and no token of its sequence is written, though the table has pages for them."""
    x = Problem(63, [4, 2, 3], [30, 20, 10], 1, 16)
    raw = torch.randn((9, 576), generator=x.gen, device="cuda").to(BF)
    weight = torch.rand(512, generator=x.gen, device="cuda").to(BF)
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    for length in (-1, -3, -16, -2 ** 31, -2 ** 40, -2 ** 63):
        kv0, pe0 = x.kv.clone(), x.pe.clone()
        error.zero_()
        lc.append(raw, weight, *x.cache, torch.tensor([5, length, 7], device="cuda"), x.cu_new, error_word=error)
        assert error.item() != 0
        written = torch.zeros(x.kv.shape[:2], dtype=torch.bool, device="cuda")
        written[x.table[0, 0].long(), 5:9] = True
        written[x.table[2, 0].long(), 7:10] = True
        assert torch.equal(x.kv[~written].view(torch.int16), kv0[~written].view(torch.int16))
        assert torch.equal(x.pe[~written].view(torch.int16), pe0[~written].view(torch.int16))
        assert torch.equal(x.pe[x.table[2, 0].long(), 7:10], raw[6:, 512:])


# --- entries as the step writes them -------------------------------------------------------------------------------

def _step_entries(raw, weight, eps):
    """The two values that an entry rounded as the step's can take: bf16(bf16(x rs) w), where the FP32 rs and its product
    are within 2^-20 of the exact ones (the sum of squares, its root and a product, as for append), so that the inner
    rounding gives `low` or `high`, which agree but next to a tie. A product of two bf16 values is exact in FP32."""
    x = raw[:, :512].to(F64)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    low, high = (((y * (1 + d)).to(F32).to(BF).to(F32) * weight.to(F32)).to(BF) for d in (-2 ** -20, 2 ** -20))
    return low, high


@pytest.mark.parametrize("kind", ["near one", "wide", "one"])
@pytest.mark.parametrize("new,lengths,page", [([1], [0], 16), ([33, 0, 70], [5, 9, 100], 10), ([300], [1], 1)])
def test_append_as_the_step_rounds(new, lengths, page, kind):
    total = [n + m for n, m in zip(new, lengths)]
    x = Problem(65, new, total, 1, page)
    raw = torch.randn((x.T, 576), generator=x.gen, device="cuda").to(BF)
    weight = {"near one": 1 + 0.1 * torch.randn(512, generator=x.gen, device="cuda"),
              "wide": torch.randn(512, generator=x.gen, device="cuda") * 3, "one": torch.ones(512, device="cuda")}[kind].to(BF)
    before = torch.tensor(lengths, device="cuda")
    assert lc.append(raw, weight, *x.cache, before, x.cu_new, eps=1e-5, as_step=True).tolist() == total
    low, high = _step_entries(raw, weight, 1e-5)
    for b in range(len(new)):
        pos = torch.arange(lengths[b], total[b], device="cuda")
        pages, slots = x.table[b, pos // page].long(), pos % page
        rows = slice(x.cu[b], x.cu[b + 1])
        got = x.kv[pages, slots]
        assert bool(((got == low[rows]) | (got == high[rows])).all())
        assert torch.equal(x.pe[pages, slots], raw[rows, 512:])


def test_append_writes_the_entry_that_the_step_writes():
    """The step's own `ka` products of a layer, appended, against the entry that the step cached for them."""
    from kimi_k3_goalbox_b200.runtime import StepContext
    from oracle import kimi_oracle as ko
    from tests import gpu_helpers as gh
    from tests import test_gpu_append as ta

    B, capacity = 3, 32
    case = gh.small_case(B, context=capacity)
    last = ko.mla_layer_ids(case)[-1]     # the layer whose products the scratch buffer holds after the step
    q_rank = case["params"]["q_lora_rank"]
    with torch.inference_mode():
        values = ko.make_inputs(case, 67, "cuda")
        weight = (1 + 0.1 * torch.randn(512, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")).to(BF)
        values[f"l{last}_kn"] = weight
        lengths = torch.tensor([9, 0, 30], dtype=torch.int64, device="cuda")
        values["reset"] = torch.zeros(B, dtype=torch.bool, device="cuda")
        conv, rec = ta._stacked_states(case, values)
        ctx = StepContext(case)
        try:
            outputs = ctx.allocate_outputs()
            outputs["conv_state"], outputs["recurrent_state"] = conv, rec
            ctx.step_append(values, outputs, lengths)
            torch.cuda.synchronize()
            ctx.check()
            raw = ctx.debug_buffer(gh.BUF["qkv"], BF, (B * (q_rank + 576),))[B * q_rank:].view(B, 576).clone()
            step, step_pe = outputs["kv_write"][-1].clone(), outputs["pe_write"][-1].clone()
        finally:
            ctx.close()
        assert torch.equal(raw[:, 512:], step_pe)     # these are that layer's products
        kv, pe, table = lc.paged_view(torch.zeros((B, capacity, 512), dtype=BF, device="cuda"),
                                      torch.zeros((B, capacity, 64), dtype=BF, device="cuda"), 8)
        one = torch.arange(B + 1, dtype=torch.int32, device="cuda")
        assert lc.append(raw, weight, kv, pe, table, lengths, one, as_step=True).tolist() == [10, 1, 31]
        rows = torch.arange(B, device="cuda")
        got = kv.view(B, capacity, 512)[rows, lengths]
        low, high = _step_entries(raw, weight, 1e-6)
        assert bool(((got == step) | (low != high)).all())
        for entry in (got, step):
            assert bool(((entry == low) | (entry == high)).all())
        assert torch.equal(got, values[f"l{last}_kv_cache"][rows, lengths]) or bool((low != high).any())
        assert torch.equal(pe.view(B, capacity, 64)[rows, lengths], values[f"l{last}_pe_cache"][rows, lengths])


# --- plans that pass through shared memory -------------------------------------------------------------------------

@pytest.mark.parametrize("new,lengths,heads,page", [
    ([11 + i % 7 for i in range(140)], [30 + (41 * i) % 700 for i in range(140)], 24, 16),    # more than 128 sequences
    ([700, 1], [1500, 900], 24, 64),                                                          # more than 32 tiles in one
    ([1] * 200, [300 + (59 * i) % 800 for i in range(200)], 12, 10),
    ([2, 1], [9001, 20000], 31, 10),                                                          # likewise, positions
])
def test_large_plans_before_the_copies(new, lengths, heads, page):
    """Calls whose work split lies, while it is computed, in the shared memory that the first copies fill."""
    x = Problem(71, new, lengths, heads, page)
    before = torch.zeros((len(new), x.columns * page), device="cuda")
    out, lse = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
    x.check_attend(out, lse)
    mass = lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new)
    x.check_mass(mass, before, lse)
    for _ in range(10):
        out2, lse2 = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
        assert torch.equal(out, out2) and torch.equal(lse, lse2)
        assert torch.equal(mass, lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new))


@pytest.mark.parametrize("new,heads", [(1, 12), (9, 40)])
@pytest.mark.parametrize("page", [10, 1, 16])
def test_mass_of_several_tiles_a_worker(new, heads, page):
    """Tiles follow one another in a worker, each with its own table of rows, from which odd pages are gathered."""
    B = 24
    lengths = [2600 + 61 * i for i in range(B)]      # 264 or more tiles, over fewer workers
    x = Problem(73, [new] * B, lengths, heads, page)
    _, lse = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
    mass = lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new)
    x.check_mass(mass, torch.zeros_like(mass), lse)
    for _ in range(5):
        assert torch.equal(mass, lc.attention_mass(x.q_latent, x.q_pe, lse, *x.cache, x.lengths, x.cu_new))


# --- lost rows -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("new,lengths,heads", [
    ([1, 1], [8000, 700], 12),         # single tokens, the first one's tile cut between many workers
    ([1, 3], [90, 50], 12),            # whole tiles
    ([60, 9], [9000, 333], 24),        # CTA pairs, cut tiles
    ([300, 40], [300, 40], 24),        # CTA pairs, whole tiles among them
])
def test_rows_of_nan_stay_marked_and_alone(new, lengths, heads):
    """A row whose sums are NaN (here by its query; by a wait that ran out, all rows of a tile) comes out as NaN in all of
    `out` and `lse`, through a tile's own end and through the join of a cut one, and spoils no other row."""
    x = Problem(75, new, lengths, heads, 16)
    q = x.q_latent.clone()
    bad = [0, x.T - 1, x.T // 2]
    for i, t in enumerate(bad):
        q[t, (5 * i) % heads] = math.nan
    out, lse = lc.attend(q, x.q_pe, *x.cache, x.lengths, x.cu_new)
    lost = torch.isnan(q[..., 0])
    assert bool(torch.isnan(out[lost]).all()) and bool(torch.isnan(lse[lost]).all())
    clean, clean_lse = lc.attend(x.q_latent, x.q_pe, *x.cache, x.lengths, x.cu_new)
    assert torch.equal(out[~lost], clean[~lost]) and torch.equal(lse[~lost], clean_lse[~lost])


# --- scales --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,new", [(12, [1, 1]), (24, [9, 30])])
def test_scales_that_leave_fp32_are_refused(heads, new):
    x = Problem(77, new, [40, 50], heads, 16)
    args = (*x.cache, x.lengths, x.cu_new)
    _, lse = lc.attend(x.q_latent, x.q_pe, *args)
    for scale in (2.4e38, -3e38, 1e39, -1e300, math.inf, -math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            lc.attend(x.q_latent, x.q_pe, *args, scale=scale)
        with pytest.raises(ValueError, match="scale"):
            lc.attention_mass(x.q_latent, x.q_pe, lse, *args, scale=scale)
    # the largest ones, over products of zero: every position counts alike
    none = torch.zeros_like(x.q_latent), torch.zeros_like(x.q_pe)
    flat = lc.attend(*none, *args)
    for scale in (lc.MAX_SCALE, -lc.MAX_SCALE):
        got = lc.attend(*none, *args, scale=scale)
        assert torch.equal(got[0], flat[0]) and torch.equal(got[1], flat[1])
        assert torch.equal(lc.attention_mass(*none, flat[1], *args, scale=scale), lc.attention_mass(*none, flat[1], *args))
