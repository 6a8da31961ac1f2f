"""The paged KV cache (append, gather) and the attention over it against plain
64-bit forms.

Stored elements are compared exactly: the formats' rounding is defined by the
exact quotient, and the oracle below decides it in 64 bits.

Tolerance of attention, per output element, from the arithmetic alone.  With
w_j the softmax weights, A = sum_j w_j |v_j| and X the largest
scale * sum_i |q_i k_ji| of the row:
- a score is a sum of head_dim products in fp32, whatever its order: off by at
  most (head_dim + 8) 2^-24 X; a tensor core may keep fewer bits of an aligned
  term, counted as a factor of 4; scores are scaled, exponentiated and summed
  in fp32: 2^-21 (|x| + 4) more, x <= X;
- each weight is off by that absolute error of its exponent, both in the
  numerator and the sum: a factor of 2;
- 16-bit outputs may round each weight to fp16 (2^-11); 32-bit ones hold it
  in 22 bits (2^-21);
- sums over n keys: (n / 16 + 16) 2^-23 A for any order in groups of at least 16;
- the output's own rounding: half a step of its type.
"""
from __future__ import annotations

import math
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest
import torch

from dotnetfoundryllm_b200.paged import PagedBatch, PagedKvCache
from dotnetfoundryllm_b200.runtime import ArgumentError, NotSupportedError

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
KV = {"f16": torch.float16, "q8": torch.int8, "f8": torch.float8_e4m3fn}
ACT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ── oracle ──────────────────────────────────────────────────────────────────
def e4m3_values() -> torch.Tensor:
    b = torch.arange(0, 0x7f, dtype=torch.uint8)
    return b.view(torch.float8_e4m3fn).to(torch.float32).double()


def quantise(x: torch.Tensor, kv: str):
    """Stored elements (as the numbers they are) and scales of rows x [..., hd]; on the CPU."""
    x = x.detach().cpu().to(torch.float32).double()
    if kv == "f16":
        return torch.where(x.isnan(), x, x.clamp(-65504.0, 65504.0)).float().half().double(), None
    top = 127.0 if kv == "q8" else 448.0
    a = x.abs().amax(-1)
    scale = (a / top).float()
    ok = x.isfinite().all(-1)
    scale = torch.where(ok, scale, torch.full_like(scale, float("nan")))
    live = ok & (scale > 0)
    y = torch.where(live[..., None], x / torch.where(live, scale, torch.ones_like(scale)).double()[..., None], torch.zeros_like(x))
    if kv == "q8":
        return y.round().clamp(-127, 127), scale
    val = e4m3_values()
    mid = (val[1:] + val[:-1]) / 2
    mag = y.abs()
    i = torch.bucketize(mag, mid)                       # a border goes down ...
    border = (i < len(mid)) & (mag == mid[i.clamp(max=len(mid) - 1)])
    i = torch.where(border & (i % 2 == 1), i + 1, i)    # ... unless the upper code is the even one
    return val[i] * torch.where(y < 0, -1.0, 1.0), scale


def as_numbers(t: torch.Tensor) -> torch.Tensor:
    return t.cpu().to(torch.float32).double()


class Setup:
    """A cache with random pages, and a batch; positions are mapped page by page in a random order."""

    def __init__(self, kv, hd, n_kv, page, lens, rows, seed=0, cols=None, fill=True):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.g, self.kv, self.hd, self.n_kv, self.page, self.lens, self.rows = g, kv, hd, n_kv, page, lens, rows
        need = [-(-max(0, n) // page) for n in lens]
        self.cols = cols or max(1, *need)
        n_pages = sum(need) + 2
        order = torch.randperm(n_pages, generator=g, device=DEV).tolist()
        table = [[-1] * self.cols for _ in lens]
        for b, k in enumerate(need):
            for j in range(min(k, self.cols)):
                table[b][j] = order.pop()
        self.table = torch.tensor(table, dtype=torch.int32, device=DEV).view(len(lens), self.cols)
        start = [0]
        for r in rows:
            start.append(start[-1] + r)
        self.start = start
        self.cache = PagedKvCache.empty(n_pages, page, n_kv, hd, KV[kv], DEV)
        if fill:
            for x, s in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)):
                if kv == "f16":
                    x.copy_(torch.randn(x.shape, generator=g, device=DEV))
                elif kv == "q8":
                    x.copy_(torch.randint(-127, 128, x.shape, generator=g, device=DEV, dtype=torch.int8))
                else:
                    x.copy_((torch.randn(x.shape, generator=g, device=DEV) * 100).clamp(-448, 448).to(torch.float8_e4m3fn))
                if s is not None:
                    s.copy_((torch.rand(s.shape, generator=g, device=DEV) + 0.5) / (70 if kv == "q8" else 100))
        self.seq_len = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.row_start = torch.tensor(start, dtype=torch.int32, device=DEV)
        self.batch = PagedBatch(self.table, self.seq_len, self.row_start, max_rows=max(rows))

    @property
    def n_rows(self):
        return self.start[-1]

    def values(self, which):
        """[n_pages, n_kv, page, hd] doubles the pool stands for, on the GPU."""
        x = getattr(self.cache, which)
        s = getattr(self.cache, which + "_scale")
        x = x.to(torch.float32).double()
        return x if s is None else x * s.double()[..., None]

    def place(self, b, p):
        """(page, offset) of position p of sequence b, or None."""
        col = p // self.page
        if p < 0 or col >= self.cols:
            return None
        pg = int(self.table[b, col])
        return (pg, p % self.page) if 0 <= pg < self.cache.k.shape[0] else None


def attend(su: Setup, q, scale, window=0, softcap=0.0):
    """out, lse and the tolerance scale (A, X) in 64 bits, row by row of sequences."""
    K, V = su.values("k"), su.values("v")
    H = q.shape[1]
    grp = H // su.n_kv
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    A = torch.zeros_like(out)
    X = torch.zeros(q.shape[0], H, dtype=torch.float64, device=DEV)
    lse = torch.full((q.shape[0], H), -math.inf, dtype=torch.float64, device=DEV)
    for b, (n, r) in enumerate(zip(su.lens, su.rows)):
        for i in range(r):
            row, p = su.start[b] + i, n - r + i
            seen = [su.place(b, j) for j in range(max(0, p - window + 1) if window > 0 else 0, p + 1)]
            seen = [x for x in seen if x is not None]
            if not seen:
                continue
            pg, off = (torch.tensor(c, device=DEV) for c in zip(*seen))
            k = K[pg, :, off].repeat_interleave(grp, 1)  # [keys, H, hd]
            v = V[pg, :, off].repeat_interleave(grp, 1)
            qq = q[row].double()
            x = torch.einsum("hd,nhd->hn", qq, k) * scale
            X[row] = (torch.einsum("hd,nhd->hn", qq.abs(), k.abs()) * abs(scale)).amax(1)
            if softcap > 0:
                x = softcap * torch.tanh(x / softcap)
            w = torch.softmax(x, 1)
            lse[row] = torch.logsumexp(x, 1)
            out[row] = torch.einsum("hn,nhd->hd", w, v)
            A[row] = torch.einsum("hn,nhd->hd", w, v.abs())
    return out, lse, A, X


def check_attention(su, q, scale, window=0, softcap=0.0, out=None, lse=None):
    want, want_lse, A, X = attend(su, q, scale, window, softcap)
    f32 = q.dtype == torch.float32
    n = max(1, max(su.lens))
    score = 4 * (su.hd + 8) * 2.0 ** -24 * X + 2.0 ** -21 * (X + 4)
    rel = 2 * score[..., None] + (2.0 ** -21 if f32 else 2.0 ** -11) + (n / 16 + 16) * 2.0 ** -23
    tol = rel * A + torch.finfo(q.dtype).eps / 2 * want.abs() * (1 + rel) + 1e-30
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"off by {(err / tol).max().item():.3g} of the tolerance"
    if lse is not None:
        live = want_lse > -math.inf
        assert torch.equal(lse == -math.inf, ~live)
        e = (lse.double() - want_lse).abs()[live]
        t = (score + 2.0 ** -22 * (want_lse.abs() + 16) + (n / 16 + 16) * 2.0 ** -23)[live]
        assert (e <= t).all(), f"lse off by {(e / t).max().item():.3g} of the tolerance"


# ── append and gather ───────────────────────────────────────────────────────
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv", ["f16", "q8", "f8"])
def test_append_writes_the_nearest_element_and_nothing_else(kv, act, hd):
    su = Setup(kv, hd, 3, 16, lens=[5, 0, 40, 17, 33], rows=[5, 0, 1, 16, 3], seed=hd)
    n = su.n_rows
    packed = torch.randn(n, 7, hd, generator=su.g, device=DEV).to(ACT[act])
    packed[2] *= 2.0 ** -9
    packed[3, 0] = 0.0
    packed[4, 1, 5:] = 0.0
    k, v = packed[:, 1:4], packed[:, 4:]  # strided rows of one matrix
    before = [as_numbers(t) for t in (su.cache.k, su.cache.v)]
    su.cache.append(su.batch, k, v)
    for which, x, old in (("k", k, before[0]), ("v", v, before[1])):
        elems, scale = quantise(x, kv)
        want = old.clone()
        want_s = None if scale is None else getattr(su.cache, which + "_scale").cpu().clone()
        for b, (ln, r) in enumerate(zip(su.lens, su.rows)):
            for i in range(r):
                pg, off = su.place(b, ln - r + i)
                want[pg, :, off] = elems[su.start[b] + i]
                if scale is not None:
                    want_s[pg, :, off] = scale[su.start[b] + i]
        assert torch.equal(as_numbers(getattr(su.cache, which)), want)
        if scale is not None:
            assert torch.equal(getattr(su.cache, which + "_scale").cpu(), want_s)


@pytest.mark.parametrize("kv", ["q8", "f8"])
def test_borders_between_elements_round_to_even_by_the_exact_quotient(kv):
    """Rows whose scale is exact and not a power of two, with elements at every
    border between two codes and one ulp to either side of it."""
    hd, rows = 256, 12
    su = Setup(kv, hd, 1, 16, lens=[rows], rows=[rows])
    if kv == "q8":
        top, mid = 127.0, torch.arange(0, 127).double() + 0.5
    else:
        val = e4m3_values()
        top, mid = 448.0, (val[1:] + val[:-1]) / 2
    x = torch.zeros(rows, 1, hd)
    for r in range(rows):
        s = torch.tensor([1.0, 1.5, 1.25, 0.75, 3.0, 1 + 2.0 ** -10, 1.0, 1.5, 1.25, 0.75, 3.0, 5.0])[r]
        border = (mid * s.double()).float()[torch.randperm(len(mid))[:hd - 1]]
        bits = border.view(torch.int32) + torch.randint(-1, 2, border.shape, dtype=torch.int32)
        x[r, 0, :len(bits)] = bits.view(torch.float32) * torch.where(torch.rand(len(bits)) < 0.5, -1.0, 1.0)
        x[r, 0, -1] = top * s
    k = x.to(DEV)
    su.cache.append(su.batch, k, -k)
    elems, scale = quantise(k, kv)
    got = torch.stack([as_numbers(su.cache.k)[su.place(0, p)[0], :, su.place(0, p)[1]] for p in range(rows)])
    neg = torch.stack([as_numbers(su.cache.v)[su.place(0, p)[0], :, su.place(0, p)[1]] for p in range(rows)])
    assert torch.equal(got, elems)
    assert torch.equal(neg, -elems)


@pytest.mark.parametrize("kv", ["f16", "q8", "f8"])
def test_rows_with_nan_infinity_zeros_and_subnormals(kv):
    hd = 128
    x = torch.randn(8, 1, hd)
    x[0, 0, 7] = float("nan")
    x[1, 0, 100] = float("inf")
    x[2] = 0.0
    x[3] = -0.0
    x[4] *= 1e-40   # subnormal rows: the scale may round, elements stay in range
    x[5] = torch.randint(-200, 201, (hd,)).float() * 2.0 ** -149
    x[6] *= 3e38 / x[6].abs().max()
    x[7, 0, :-1] = 1e-30
    x[7, 0, -1] = 1e30
    su = Setup(kv, hd, 1, 16, lens=[8], rows=[8])
    k = x.to(DEV)
    su.cache.append(su.batch, k, k)
    kk, vv = su.cache.gather(su.batch, 8, torch.float32)
    assert torch.equal(kk.view(torch.int32), vv.view(torch.int32)) or kv == "f16"
    elems, scale = quantise(k, kv)
    want = elems.float() if scale is None else elems.float() * scale[..., None]
    got = kk.cpu()
    assert torch.equal(got.isnan(), want.isnan())
    if kv == "f16":
        assert got[0, 0, 7].isnan() and got[0].isnan().sum() == 1 and got[1, 0, 100] == 65504.0
    else:
        assert got[0].isnan().all() and got[1].isnan().all()
    live = ~want.isnan()
    assert torch.equal(got[live], want[live])


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,hd,page", [("f16", 64, 16), ("q8", 64, 128), ("f8", 64, 16), ("f16", 128, 1024), ("q8", 128, 16),
                                         ("f8", 128, 32), ("f16", 256, 64), ("q8", 256, 16), ("f8", 256, 16)])
def test_gather_reads_the_values_rounded_once(kv, hd, page, act):
    su = Setup(kv, hd, 2, page, lens=[1, 130, 64, 0, 31], rows=[1, 50, 64, 0, 2], seed=3)
    su.table[1, 100 // page] = -1 if page == 16 else su.table[1, 100 // page]  # an unmapped page reads as zero
    K, V = su.values("k").float(), su.values("v").float()
    k, v = su.cache.gather(su.batch, su.n_rows, ACT[act])
    for b, (n, r) in enumerate(zip(su.lens, su.rows)):
        for i in range(r):
            at = su.place(b, n - r + i)
            for got, pool in ((k, K), (v, V)):
                want = torch.zeros(2, hd, device=DEV) if at is None else pool[at[0], :, at[1]]
                assert torch.equal(got[su.start[b] + i], want.to(ACT[act]))


def test_rows_behind_the_last_sequence_and_unmapped_places_are_left_alone():
    su = Setup("q8", 128, 2, 16, lens=[3, 20], rows=[5, 4])   # the first sequence's rows start at position -2
    n = su.n_rows + 3
    su.table[1, 1] = 10 ** 6                                  # positions 16.. of the second point nowhere
    k = torch.randn(n, 2, 128, generator=su.g, device=DEV)
    before = su.cache.k.clone(), su.cache.k_scale.clone()
    su.cache.append(su.batch, k, k)
    elems, scale = quantise(k, "q8")
    want = before[0].clone()
    for i in range(2, 5):
        pg, off = su.place(0, i - 2)
        want[pg, :, off] = elems[i].to(torch.int8).to(DEV)
    assert torch.equal(su.cache.k, want)
    out = torch.full((n, 2, 128), 7.0, device=DEV), torch.full((n, 2, 128), 7.0, device=DEV)
    su.cache.gather(su.batch, n, torch.float32, out=out)
    assert (out[0][su.n_rows:] == 7.0).all() and (out[1][su.n_rows:] == 7.0).all()
    assert (out[0][:2] == 0).all() and (out[0][5:9] == 0).all()
    assert (out[0][2:5] != 0).any(-1).all()
    q = torch.randn(n, 4, 128, generator=su.g, device=DEV)
    o = torch.full_like(q, 7.0)
    lse = torch.full((n, 4), 7.0, device=DEV)
    su.cache.attention(su.batch, q, 0.1, out=o, lse=lse)
    assert (o[su.n_rows:] == 7.0).all() and (lse[su.n_rows:] == 7.0).all()
    assert (o[:2] == 0).all() and (lse[:2] == -math.inf).all()
    check_attention(su, q[:su.n_rows], 0.1, out=o[:su.n_rows], lse=lse[:su.n_rows])


def test_lengths_past_the_page_table_are_cut():
    su = Setup("f16", 64, 1, 16, lens=[100], rows=[4], cols=3)   # positions 48.. have no page
    k = torch.randn(4, 1, 64, generator=su.g, device=DEV)
    before = su.cache.k.clone()
    su.cache.append(su.batch, k, k)
    assert torch.equal(su.cache.k, before)
    q = torch.randn(4, 2, 64, generator=su.g, device=DEV)
    check_attention(su, q, 0.2, out=su.cache.attention(su.batch, q, 0.2))


@pytest.mark.parametrize("kv", ["q8", "f16"])
def test_offsets_past_32_bits(kv):
    """A pool of more than 2^32 elements: the last page, written, read and attended to."""
    n_kv, page, hd = 8, 128, 128
    n_pages = 2 ** 32 // (n_kv * page * hd) + 3
    k = torch.empty(n_pages, n_kv, page, hd, dtype=KV[kv], device=DEV)
    v = torch.empty_like(k)
    sc = [None, None] if kv == "f16" else [torch.empty(n_pages, n_kv, page, device=DEV) for _ in range(2)]
    cache = PagedKvCache(k, v, *sc)
    table = torch.tensor([[n_pages - 1]], dtype=torch.int32, device=DEV)
    batch = PagedBatch(table, torch.tensor([70], dtype=torch.int32, device=DEV), torch.tensor([0, 70], dtype=torch.int32, device=DEV))
    x = torch.randn(70, n_kv, hd, device=DEV)
    cache.append(batch, x, x * 0.5)
    kk, vv = cache.gather(batch, 70)
    assert (kk - x).abs().max() < 0.05 and (vv - x * 0.5).abs().max() < 0.05
    q = torch.randn(70, 2 * n_kv, hd, device=DEV)
    o = cache.attention(batch, q, 0.1)
    w = torch.softmax((torch.einsum("rhd,nhd->rhn", q.double(), kk.double().repeat_interleave(2, 1)) * 0.1).masked_fill(
        torch.ones(70, 70, dtype=torch.bool, device=DEV).triu(1)[:, None], -math.inf), -1)
    want = torch.einsum("rhn,nhd->rhd", w, vv.double().repeat_interleave(2, 1))
    assert (o.double() - want).abs().max() < 1e-4
    del cache, k, v, sc
    torch.cuda.empty_cache()


# ── attention ───────────────────────────────────────────────────────────────
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv", ["f16", "q8", "f8"])
@pytest.mark.parametrize("kind", ["decode", "verify", "chunk"])
def test_attention_matches_the_formula(kind, kv, act, hd):
    lens, rows = {"decode": ([1, 130, 700, 0, 33], [1, 1, 1, 0, 1]), "verify": ([5, 200, 64], [5, 3, 4]),
                  "chunk": ([150, 300], [150, 77])}[kind]
    su = Setup(kv, hd, 2, 16, lens, rows, seed=hd + len(lens))
    q = (torch.randn(su.n_rows, 8, hd, generator=su.g, device=DEV)).to(ACT[act])
    lse = torch.empty(su.n_rows, 8, device=DEV)
    o = su.cache.attention(su.batch, q, 1 / math.sqrt(hd), lse=lse)
    check_attention(su, q, 1 / math.sqrt(hd), out=o, lse=lse)


@pytest.mark.parametrize("group", [1, 2, 3, 7, 8, 16, 33])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_attention_groups(group, rows):
    su = Setup("q8", 128, 2, 32, [200, rows], [rows, rows], seed=group)
    q = torch.randn(su.n_rows, 2 * group, 128, generator=su.g, device=DEV).to(torch.bfloat16)
    check_attention(su, q, 0.09, out=su.cache.attention(su.batch, q, 0.09))


@pytest.mark.parametrize("window", [1, 7, 64, 129, 5000])
@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("kv,act,hd,rows", [("f16", "f32", 64, 1), ("f8", "bf16", 256, 5), ("q8", "f16", 128, 90)])
def test_attention_window_and_softcap(window, softcap, kv, act, hd, rows):
    su = Setup(kv, hd, 2, 64, [300, rows + 2], [rows, rows], seed=window)
    q = (2 * torch.randn(su.n_rows, 6, hd, generator=su.g, device=DEV)).to(ACT[act])
    o = su.cache.attention(su.batch, q, 1 / math.sqrt(hd), window=window, softcap=softcap)
    check_attention(su, q, 1 / math.sqrt(hd), window, softcap, out=o)


@pytest.mark.parametrize("page", [16, 128, 1024])
@pytest.mark.parametrize("rows", [1, 70])
def test_attention_pages_and_holes(page, rows):
    """Lengths that end inside a tile and a page, and unmapped pages in the middle."""
    su = Setup("q8", 64, 1, page, [2 * page + 77, 4 * page, page + 1], [rows] * 3, seed=page)
    su.table[1, 1] = -1
    q = torch.randn(su.n_rows, 4, 64, generator=su.g, device=DEV)
    check_attention(su, q, 0.125, out=su.cache.attention(su.batch, q, 0.125))


@pytest.mark.parametrize("kv", ["f16", "q8", "f8"])
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 6, 200])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_what_is_masked_does_not_touch_a_row(kv, act, rows, hd):
    """NaN and infinities behind a row's position, before its window, in stale
    places of a page and in unmapped pages leave it exactly as it is."""
    lens = [230, 210]
    su = Setup(kv, hd, 2, 32, lens, [rows, 1], seed=rows)
    q = torch.randn(su.n_rows, 4, hd, generator=su.g, device=DEV).to(ACT[act])
    kw = dict(scale=1 / math.sqrt(hd), window=50)
    clean = su.cache.attention(su.batch, q, **kw)
    check_attention(su, q, kw["scale"], 50, out=clean)
    bad = [float("nan"), float("inf"), -float("inf")]

    def poison(b, p):
        pg, off = su.place(b, p)
        for i, t in enumerate((su.cache.k, su.cache.v)):
            if kv == "f16":
                t[pg, :, off] = bad[(p + i) % 3]
            else:
                if kv == "f8":
                    t.view(torch.uint8)[pg, :, off] = 0x7F if p % 2 else 0xFF
                (su.cache.k_scale, su.cache.v_scale)[i][pg, :, off] = bad[(p + i) % 3]

    first = lens[0] - rows                           # the chunk's first row's position
    for p in range(0, max(0, first - 49)):
        poison(0, p)                                 # before every row's window
    for p in range(0, 150):
        poison(1, p)
    for b in range(2):
        for p in range(lens[b], -(-lens[b] // 32) * 32):
            poison(b, p)                             # stale places behind the sequence
    assert torch.equal(su.cache.attention(su.batch, q, **kw), clean)
    if rows > 1:                                     # the last position: only the last row sees it
        poison(0, lens[0] - 1)
        got = su.cache.attention(su.batch, q, **kw)
        assert torch.equal(got[:rows - 1], clean[:rows - 1])
        assert got[rows - 1].isnan().any()
        assert torch.equal(got[rows:], clean[rows:])


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_32_bit_rows_over_long_sequences_do_not_drift(hd):
    """Equal weights over values of one sign: the output is their mean.  A tensor
    core truncates each of its sums of 16 products, by at most 2^-23 of the sum;
    in a run of 512 keys there are 64 of them (two halves of a weight), and each
    run's sum, the weights' sum and the quotient are rounded to nearest: at
    16,000 keys (64 + 32 / 2 + 4) 2^-23 = 1.0e-5 in all."""
    n, seqs, rows = 16000, 20, 6
    su = Setup("f16", hd, 4, 64, [n], [rows], seed=hd)
    su.cache.v.copy_(1 + torch.rand(su.cache.v.shape, generator=su.g, device=DEV))
    batch = PagedBatch(su.table.repeat(seqs, 1), su.seq_len.repeat(seqs),
                       torch.arange(seqs + 1, dtype=torch.int32, device=DEV) * rows, max_rows=rows)
    out = su.cache.attention(batch, torch.zeros(seqs * rows, 32, hd, device=DEV), 0.1).view(seqs, rows, 4, 8, hd).double()
    V = su.cache.v[su.table[0].long()].double().transpose(1, 2).reshape(-1, 4, hd)[:n].cumsum(0)
    for i in range(rows):
        seen = n - rows + i + 1
        ref = V[seen - 1] / seen
        worst = ((out[:, i] - ref[None, :, None]).abs() / ref[None, :, None]).max()
        assert float(worst) < 84 * 2.0 ** -23


def test_scores_of_any_size():
    """Scores far apart, all far below zero, and past the largest finite value of 16 bits."""
    for strength in (1.0, 200.0, 30000.0):
        for act in ("f32", "bf16"):
            su = Setup("f16", 64, 1, 16, [90, 45], [3, 1], seed=int(strength))
            su.cache.k.copy_(su.cache.k.sign() * 0.01 + 0.002 * su.cache.k)
            q = (strength * torch.randn(su.n_rows, 2, 64, generator=su.g, device=DEV)).to(ACT[act])
            check_attention(su, q, 1.0, out=su.cache.attention(su.batch, q, 1.0))


def test_tiny_and_large_values_in_the_cache():
    """Scales of very different size in one sequence; queries near the ends of the exponent range."""
    su = Setup("q8", 128, 1, 16, [300], [4], seed=5)
    su.cache.v_scale.mul_(torch.exp2(torch.randint(-12, 13, su.cache.v_scale.shape, generator=su.g, device=DEV).float()))
    q = torch.randn(4, 2, 128, generator=su.g, device=DEV)
    check_attention(su, q, 0.09, out=su.cache.attention(su.batch, q, 0.09))
    for f in (1e-30, 1e25):
        out = su.cache.attention(su.batch, q * f, 0.09 / f)
        check_attention(su, q * f, 0.09 / f, out=out)


def test_strided_queries_and_outputs():
    su = Setup("f8", 128, 2, 16, [50, 9], [7, 2])
    packed = torch.randn(9, 12, 128, generator=su.g, device=DEV).to(torch.float16)
    q = packed[:, 2:10]
    o = torch.full((9, 10, 128), 7.0, dtype=torch.float16, device=DEV)
    su.cache.attention(su.batch, q, 0.1, out=o[:, 1:9])
    check_attention(su, q, 0.1, out=o[:, 1:9])
    assert (o[:, 0] == 7.0).all() and (o[:, 9] == 7.0).all()


def test_the_same_call_gives_the_same_bits_and_sequences_do_not_touch_each_other():
    lens, rows = [900, 77, 1500, 3], [2, 2, 2, 2]
    su = Setup("q8", 128, 4, 16, lens, rows)
    q = torch.randn(su.n_rows, 16, 128, generator=su.g, device=DEV).to(torch.bfloat16)
    a = su.cache.attention(su.batch, q, 0.09)
    for _ in range(3):
        assert torch.equal(su.cache.attention(su.batch, q, 0.09), a)
    check_attention(su, q, 0.09, out=a)


def test_max_rows_is_a_hint_only():
    """A wrong bound on the rows of a sequence costs speed, never results."""
    su = Setup("q8", 128, 2, 16, [400, 130, 20], [170, 1, 9])
    q = torch.randn(su.n_rows, 8, 128, generator=su.g, device=DEV).to(torch.bfloat16)
    for hint in (0, 1, 5, 170, 100000):
        batch = PagedBatch(su.table, su.seq_len, su.row_start, max_rows=hint)
        check_attention(su, q, 0.09, out=su.cache.attention(batch, q, 0.09))


def test_graphs_replay_with_new_lengths_and_hold_their_own_workspaces():
    """Two captured steps share the cache; lengths, tables and rows change between replays."""
    su = Setup("q8", 128, 2, 16, [260, 40], [1, 1], cols=20)
    q = [torch.randn(2, 8, 128, generator=su.g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    kv = torch.randn(2, 2, 128, generator=su.g, device=DEV).to(torch.bfloat16)
    su.cache.attention(su.batch, q[0], 0.09)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            su.cache.append(su.batch, kv, kv)
            outs.append(su.cache.attention(su.batch, q[i], 0.09))
        graphs.append(g)
    for lens in ([260, 40], [17, 272], [1, 1], [250, 0]):
        su.lens = lens
        su.seq_len.copy_(torch.tensor(lens, dtype=torch.int32))
        for g in graphs:
            g.replay()
        for i in range(2):
            check_attention(su, q[i], 0.09, out=outs[i])


def test_another_stream_than_the_default():
    su = Setup("f16", 64, 2, 16, [500, 300], [3, 3])
    q = torch.randn(6, 4, 64, generator=su.g, device=DEV)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([su.cache.attention(su.batch, q, 0.1) for _ in range(4)])
    torch.cuda.synchronize()
    for os in outs:
        for o in os:
            assert torch.equal(o, outs[0][0])
    check_attention(su, q, 0.1, out=outs[0][0])


def test_threads_on_their_own_streams():
    """Calls from several host threads at once, each on a stream of its own."""
    su = Setup("q8", 128, 2, 32, [700, 650], [4, 40], seed=4)
    q = torch.randn(44, 8, 128, generator=su.g, device=DEV).to(torch.bfloat16)
    one = PagedBatch(su.table, su.seq_len, torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), max_rows=1)
    want = su.cache.attention(su.batch, q, 0.09), su.cache.attention(one, q[:2], 0.09)
    torch.cuda.synchronize()

    def work(_):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [(su.cache.attention(su.batch, q, 0.09), su.cache.attention(one, q[:2], 0.09)) for _ in range(8)]
            torch.cuda.current_stream().synchronize()
        return all(torch.equal(a, b) for g in got for a, b in zip(g, want))

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(4)))


COLD = """
import torch
from dotnetfoundryllm_b200.paged import PagedBatch, PagedKvCache
from dotnetfoundryllm_b200.speculate import verify_drafts
i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
cache = PagedKvCache.empty(4, 16, 2, 64, torch.int8, "cuda")
cache.k.zero_(), cache.v.zero_(), cache.k_scale.zero_(), cache.v_scale.zero_()
batches = [PagedBatch(i32(0, 1, 2, 3).view(1, 4), i32(n), i32(0, n), max_rows=n) for n in (1, 60)]
x = torch.randn(60, 2, 64, device="cuda")
q = torch.randn(60, 8, 64, device="cuda")
logits = torch.randn(2, 1000, device="cuda")
args = i32(0, 2), i32(5, 0), torch.ones(1, device="cuda"), torch.rand(2, device="cuda"), torch.rand(1, device="cuda")
def step():
    out = []
    for n, b in zip((1, 60), batches):
        cache.append(b, x[:n], x[:n])
        out += [cache.attention(b, q[:n], 0.1), *cache.gather(b, n, torch.float16)]
    return out + list(verify_drafts(logits, *args))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a = step()
g.replay()
torch.cuda.synchronize()
b = step()
assert all(torch.equal(p, q) for p, q in zip(a, b)), "replayed and called results differ"
"""


def test_first_calls_of_a_process_may_be_captured():
    r = subprocess.run([sys.executable, "-c", COLD], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("rows", [1, 50])
def test_a_batch_of_absent_sequences_leaves_everything_alone(rows):
    """Row arrays that are padding throughout: no sequence has a row."""
    su = Setup("f8", 128, 2, 16, [40, 0], [0, 0])
    q = torch.randn(rows, 4, 128, generator=su.g, device=DEV)
    batch = PagedBatch(su.table, su.seq_len, su.row_start, max_rows=rows)
    out = torch.full_like(q, 7.0)
    before = su.cache.k.view(torch.uint8).clone()
    su.cache.append(batch, q[:, :2].contiguous(), q[:, 2:].contiguous())
    su.cache.attention(batch, q, 0.1, out=out)
    assert bool((out == 7.0).all()) and torch.equal(su.cache.k.view(torch.uint8), before)


def test_refusals_of_tensors():
    su = Setup("q8", 128, 2, 16, [20], [2])
    q = torch.randn(2, 4, 128, device=DEV)
    k = torch.randn(2, 2, 128, device=DEV)
    c, b = su.cache, su.batch
    for bad in (q[:, :3], q[..., :64], q[0], q.cpu(), q.transpose(0, 1)[:, :4]):
        with pytest.raises(ArgumentError):
            c.attention(b, bad, 0.1)
    with pytest.raises(NotSupportedError):
        c.attention(b, q.double(), 0.1)
    with pytest.raises(ArgumentError):
        c.attention(b, q, float("inf"))
    with pytest.raises(ArgumentError):
        c.attention(b, q, 0.1, out=torch.empty(2, 4, 128, dtype=torch.float16, device=DEV))
    with pytest.raises(ArgumentError):
        c.attention(b, q, 0.1, lse=torch.empty(2, 4, dtype=torch.float64, device=DEV))
    with pytest.raises(ArgumentError):
        c.append(b, k, k.half())
    with pytest.raises(ArgumentError):
        c.append(b, k, k[:1])
    with pytest.raises(ArgumentError):
        c.append(b, torch.randn(2, 2, 256, device=DEV)[..., ::2], k)
    with pytest.raises(ArgumentError):
        c.gather(b, 3, out=(k, k))
    with pytest.raises(NotSupportedError):
        c.gather(b, 2, torch.int32)
    with pytest.raises(ArgumentError):
        PagedKvCache(c.k, c.v)                       # scales missing
    with pytest.raises(ArgumentError):
        PagedKvCache(c.k, c.v, c.k_scale, c.v_scale.half())
    with pytest.raises(ArgumentError):
        PagedKvCache(c.k.transpose(1, 2), c.v.transpose(1, 2), c.k_scale, c.v_scale)
    with pytest.raises(ArgumentError):
        PagedBatch(su.table, su.seq_len, su.row_start[:1])
    with pytest.raises(ArgumentError):
        PagedBatch(su.table.long(), su.seq_len, su.row_start)
