"""Attention over a paged KV cache for batches that give every SM several items
(a sequence's kv head, up to 128 or 256 query rows with the heads of its group),
short and long ones in turn, and for masks and units at the ends of their range.
The tolerance is derived in test_gpu_paged.py; where scores are far apart one more
part of it counts, since an output may be made of small weights alone (the value of
the largest is 0 there).  A weight p <= 2^8 is stored as fp16 of 2^6 p times its
value's scale in units of the largest scale's power of two.  Below 2^-14 the steps of
fp16 are 2^-24: half a step is 2^-25, so each weight times scale is off by at most
2^-31 of the largest scale, each product by 2^-31 of that scale and the largest
element (of the largest value, without scales).  n keys are off by n times that; the
sum that divides them is at least 1, the weight of the reference.
"""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from dotnetfoundryllm_b200 import _native as N
from dotnetfoundryllm_b200.paged import PagedBatch
from dotnetfoundryllm_b200.runtime import ArgumentError, DeviceTimeoutError
from test_gpu_paged import ACT, DEV, Setup

pytestmark = pytest.mark.gpu


def attend(su: Setup, q, scale, window=0, softcap=0.0):
    """out, lse and the tolerance scales A, X in 64 bits, a sequence at a time."""
    K, V = su.values("k"), su.values("v")
    n_rows, H, hd = q.shape
    grp = H // su.n_kv
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    A = torch.zeros_like(out)
    X = torch.zeros(n_rows, H, dtype=torch.float64, device=DEV)
    lse = torch.full((n_rows, H), -math.inf, dtype=torch.float64, device=DEV)
    for b, (n, r) in enumerate(zip(su.lens, su.rows)):
        n_pages = min(-(-n // su.page), su.cols)
        if r == 0 or n_pages <= 0:
            continue
        pages = su.table[b, :n_pages].long()
        there = ((pages >= 0) & (pages < K.shape[0])).repeat_interleave(su.page)[:n]
        pages = pages.clamp(0, K.shape[0] - 1)
        k = K[pages].transpose(1, 2).reshape(-1, su.n_kv, hd)[:n].repeat_interleave(grp, 1)  # [keys, H, hd]
        v = V[pages].transpose(1, 2).reshape(-1, su.n_kv, hd)[:n].repeat_interleave(grp, 1)
        at = slice(su.start[b], su.start[b] + r)
        qq = q[at].double()
        x = torch.einsum("rhd,nhd->rhn", qq, k) * scale
        bound = torch.einsum("rhd,nhd->rhn", qq.abs(), k.abs()) * abs(scale)
        if softcap > 0:
            x = softcap * torch.tanh(x / softcap)
        pos = n - r + torch.arange(r, device=DEV)[:, None]
        key = torch.arange(len(k), device=DEV)[None]
        seen = (key <= pos) & there[None]
        if window > 0:
            seen &= key > pos - window
        some = seen.any(1)
        seen = seen[:, None]
        w = torch.softmax(x.masked_fill(~seen, -math.inf), -1).masked_fill(~some[:, None, None], 0.0)
        lse[at] = torch.logsumexp(x.masked_fill(~seen, -math.inf), -1)
        out[at] = torch.einsum("rhn,nhd->rhd", w, v)
        A[at] = torch.einsum("rhn,nhd->rhd", w, v.abs())
        X[at] = bound.masked_fill(~seen, 0.0).amax(-1)
    return out, lse, A, X


def check(su, q, scale, window=0, softcap=0.0, **kw):
    """Calls the operator and compares out and lse, as check_attention of test_gpu_paged.py does."""
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    out = su.cache.attention(su.batch, q, scale, window=window, softcap=softcap, lse=lse, **kw)
    compare(su, q, scale, window, softcap, out, lse)
    return out


def compare(su, q, scale, window, softcap, out, lse, rows=slice(None)):
    want, want_lse, A, X = (t[rows] for t in attend(su, q, scale, window, softcap))
    out, lse = out[rows], lse[rows]
    f32 = q.dtype == torch.float32
    n = max(1, max(su.lens))
    score = 4 * (su.hd + 8) * 2.0 ** -24 * X + 2.0 ** -21 * (X + 4)
    rel = 2 * score[..., None] + (2.0 ** -21 if f32 else 2.0 ** -11) + (n / 16 + 16) * 2.0 ** -23
    largest = su.cache.v.float().abs().max().item()
    if su.cache.v_scale is not None:
        largest *= su.cache.v_scale.abs().max().item()
    tol = rel * A + torch.finfo(q.dtype).eps / 2 * want.abs() * (1 + rel) + n * 2.0 ** -31 * largest
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"off by {(err / tol).nan_to_num(math.inf).max().item():.3g} of the tolerance"
    live = want_lse > -math.inf
    assert torch.equal(lse == -math.inf, ~live)
    e = (lse.double() - want_lse).abs()[live]
    t = (score + 2.0 ** -22 * (want_lse.abs() + 16) + (n / 16 + 16) * 2.0 ** -23)[live]
    assert (e <= t).all(), f"lse off by {(e / t).nan_to_num(math.inf).max().item():.3g} of the tolerance"


def queries(su, heads, act, f=1.0):
    return (f * torch.randn(su.n_rows, heads, su.hd, generator=su.g, device=DEV)).to(ACT[act])


@pytest.mark.parametrize("kv,hd,rows", [("f8", 64, 32), ("q8", 64, 32), ("f8", 128, 32), ("q8", 128, 32), ("q8", 256, 32)])
def test_weights_of_16_bit_rows_are_rounded_once(kv, hd, rows):
    """Causal prompts, whose first rows have a few large weights: a weight and the scale of its value make one
    product, and the tolerance has room for one rounding of it to 11 bits."""
    for seed in range(12):
        su = Setup(kv, hd, 8, 16, [rows] * 18, [rows] * 18, seed=seed)
        check(su, queries(su, 32, "bf16"), 1 / math.sqrt(hd))


# cache, rows' type, head size, drafted rows that the tcgen05 kernel takes at 4 heads a group
SHORT = [("f16", "bf16", 128, 5), ("f16", "f16", 64, 9), ("f16", "f32", 64, 13), ("f16", "f32", 128, 5), ("f16", "bf16", 256, 5),
         ("q8", "bf16", 128, 13), ("q8", "f16", 64, 13), ("q8", "f32", 64, 21), ("f8", "bf16", 64, 9), ("f8", "f16", 128, 9),
         ("f8", "f32", 64, 17)]


@pytest.mark.parametrize("kv,act,hd,rows", SHORT)
def test_many_sequences_of_a_few_drafted_rows(kv, act, hd, rows):
    """100 sequences x 8 kv heads: five or six items an SM, none with a second row tile."""
    g = torch.Generator().manual_seed(hd + rows)
    lens = [rows + int(x) for x in torch.randint(0, 700, (100,), generator=g)]
    su = Setup(kv, hd, 8, 16, lens, [rows] * 100, seed=1)
    check(su, queries(su, 32, act), 1 / math.sqrt(hd))


@pytest.mark.parametrize("kv,act,hd,rows", SHORT)
def test_many_short_prompts(kv, act, hd, rows):
    su = Setup(kv, hd, 8, 16, [32] * 96, [32] * 96, seed=2)
    check(su, queries(su, 32, act), 1 / math.sqrt(hd))


@pytest.mark.parametrize("kv,act,hd,rows", SHORT)
def test_single_tokens_beside_a_chunk(kv, act, hd, rows):
    g = torch.Generator().manual_seed(hd)
    lens = [1 + int(x) for x in torch.randint(0, 900, (80,), generator=g)]
    lens[40] = 1100
    su = Setup(kv, hd, 8, 32, lens, [1] * 40 + [512] + [1] * 39, seed=3)
    check(su, queries(su, 32, act), 1 / math.sqrt(hd))


@pytest.mark.parametrize("kv,act,hd,rows", SHORT)
def test_items_with_one_and_with_two_row_tiles_in_turn(kv, act, hd, rows):
    """Rows that fill a row tile (32 x 4), fall short of it, pass it by one row, fill two and pass two."""
    kinds = [1, 32, 33, 2, 64, 17, 65, 31, 40, 1, 1, 1, 64, 0, 5]
    g = torch.Generator().manual_seed(hd + 7)
    n_rows = [kinds[int(x)] for x in torch.randint(0, len(kinds), (120,), generator=g)]
    lens = [r + int(x) for r, x in zip(n_rows, torch.randint(0, 300, (120,), generator=g))]
    su = Setup(kv, hd, 8, 16, lens, n_rows, seed=4)
    q = queries(su, 32, act)
    out = check(su, q, 1 / math.sqrt(hd), window=150)
    for _ in range(3):
        assert torch.equal(su.cache.attention(su.batch, q, 1 / math.sqrt(hd), window=150), out)


@pytest.mark.parametrize("kv,act,hd", [("f16", "bf16", 64), ("f16", "f32", 128), ("q8", "bf16", 128), ("q8", "f16", 256), ("f8", "f32", 64),
                                       ("f8", "bf16", 256)])
@pytest.mark.parametrize("rows", [1, 3, 90])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-3, -1e-3, 1e-30, 1e-38])
def test_units_of_zero_and_queries_of_zero(kv, act, hd, rows, scale):
    """A scale of 0 gives the mean of what a row sees; so does a row of zeros, whatever the scale; rows of tiny
    queries are next to it.  The page in the middle is not mapped."""
    su = Setup(kv, hd, 2, 16, [rows + 200, rows, rows + 37], [rows] * 3, seed=rows)
    su.table[0, 2] = -1
    q = queries(su, 8, act)
    q[::2, ::3] = 0.0
    q[1::3, 1] *= 1e-30
    check(su, q, scale)
    check(su, q, scale, window=70)
    check(su, q, scale, softcap=30.0)


@pytest.mark.parametrize("kv,act,hd", [("f16", "bf16", 64), ("f16", "f16", 128), ("f16", "f32", 128), ("q8", "bf16", 128),
                                       ("f8", "f16", 256), ("f8", "f32", 64)])
@pytest.mark.parametrize("rows", [1, 90])
@pytest.mark.parametrize("softcap", [0.02, 127.0, 129.0, 1e3, 1e4, 1e6, 1e8])
def test_softcaps_of_any_size(softcap, kv, act, hd, rows):
    """A cap far above the scores leaves them as they are; q runs to scores of some tens and, of 90 rows, hundreds."""
    su = Setup(kv, hd, 2, 16, [rows + 250, rows], [rows, rows], seed=int(softcap) % 97)
    su.table[0, 1] = -1
    q = queries(su, 8, act, 8.0)
    q[::5] *= 16
    check(su, q, 1 / math.sqrt(hd), softcap=softcap)


@pytest.mark.parametrize("kv,act,hd,lens,rows", [
    ("f16", "bf16", 128, [700, 300], [500, 90]),            # items cut and whole, two row tiles and one
    ("q8", "f16", 64, [40] * 60 + [300], [32] * 60 + [17]),  # several short items an SM
    ("f8", "bf16", 256, [200, 600], [150, 33]),
    ("q8", "f32", 128, [900], [200]),
    ("f16", "f32", 64, [64, 2000], [64, 70]),
])
def test_a_wait_that_runs_out_is_reported(kv, act, hd, lens, rows):
    """Copies held back: every row is NaN, whatever the buffers held, rows behind the last sequence stay as they were,
    the device reports it once, and the next call is right."""
    su = Setup(kv, hd, 4, 16, lens, rows, seed=hd)
    c, n = su.cache, su.n_rows + 3
    q = torch.randn(n, 16, hd, generator=su.g, device=DEV).to(ACT[act])
    out = torch.full_like(q, 7.0)
    lse = torch.full((n, 16), 7.0, device=DEV)
    want = c.attention(su.batch, q[:su.n_rows], 0.1)
    need = C.c_uint64()
    assert c.lib.fl_attn_paged_workspace(c._ref, su.batch._ref, n, 16, C.byref(need)) == N.FL_OK
    ws = torch.zeros(need.value, dtype=torch.uint8, device=DEV)
    d = N.FlPagedAttnDesc(C.sizeof(N.FlPagedAttnDesc), {"f32": 0, "f16": 1, "bf16": 30}[act], n, 16, 0, 0.1, 0.0, 0, q.data_ptr(),
                          q.stride(0), out.data_ptr(), out.stride(0), lse.data_ptr(), ws.data_ptr(), need.value)
    stream = torch.cuda.current_stream().cuda_stream
    c.synchronize()
    assert c.lib.fl_attn_paged_stall(c._ref, su.batch._ref, C.byref(d), stream) == N.FL_OK
    with pytest.raises(DeviceTimeoutError):
        c.synchronize()
    c.synchronize()
    assert out[:su.n_rows].isnan().all() and lse[:su.n_rows].isnan().all()
    assert (out[su.n_rows:] == 7.0).all() and (lse[su.n_rows:] == 7.0).all()
    assert torch.equal(c.attention(su.batch, q[:su.n_rows], 0.1), want)
    c.synchronize()


@pytest.mark.parametrize("kv,act,hd", [("q8", "bf16", 64), ("f8", "f16", 64), ("q8", "f32", 64), ("q8", "bf16", 128), ("f16", "bf16", 64)])
@pytest.mark.parametrize("rows", [1, 4, 90])
@pytest.mark.parametrize("mapped", [0.02, 0.4])
def test_most_pages_unmapped(kv, act, hd, rows, mapped):
    """Single pages and runs of them among unmapped ones: places of a ring are zeroed and copied into in turn."""
    lens = [3000, 1777, rows, 640]
    su = Setup(kv, hd, 2, 16, lens, [rows] * 4, seed=rows)
    su.table[torch.rand(su.table.shape, generator=su.g, device=DEV) > mapped] = -1
    q = queries(su, 8, act)
    out = check(su, q, 1 / math.sqrt(hd))
    for _ in range(3):
        assert torch.equal(su.cache.attention(su.batch, q, 1 / math.sqrt(hd)), out)


@pytest.mark.parametrize("kv,act,hd", [("f16", "bf16", 64), ("q8", "bf16", 128), ("f8", "f32", 256)])
@pytest.mark.parametrize("rows", [7, 90])
@pytest.mark.parametrize("window", [1, 2 ** 30, 2 ** 31 - 50, 2 ** 31 - 1])
def test_the_largest_windows_with_rows_before_the_first_position(window, kv, act, hd, rows):
    """A padded sequence: fewer positions than rows, so that its first rows lie at negative positions and see nothing."""
    su = Setup(kv, hd, 2, 16, [rows // 2, rows + 300, 1], [rows, rows, rows], seed=rows)
    check(su, queries(su, 8, act), 1 / math.sqrt(hd), window=window)


@pytest.mark.parametrize("kv,act,hd", [("f16", "bf16", 64), ("q8", "bf16", 128), ("f8", "f32", 256)])
@pytest.mark.parametrize("rows", [3, 90])
@pytest.mark.parametrize("window", [0, 1, 40, 2 ** 31 - 60])
def test_lengths_that_are_far_past_the_table_or_negative(window, kv, act, hd, rows):
    """Rows at positions up to 2^31 - 2, none of whose keys but the table's are there; beside a sequence of the usual kind."""
    su = Setup(kv, hd, 2, 16, [rows + 90, rows, rows + 30, 48], [rows] * 4, seed=rows)
    q = queries(su, 8, act)
    su.seq_len.copy_(torch.tensor([2 ** 31 - 1, -2 ** 31, rows + 30, -1], dtype=torch.int32))
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    out = su.cache.attention(su.batch, q, 0.1, window=window, lse=lse)
    su.cache.synchronize()
    compare(su, q, 0.1, window, 0.0, out, lse, slice(2 * rows, 3 * rows))
    for at in ([1, 3] if window in (0, 2 ** 31 - 60) else [0, 1, 3]):
        assert (out[at * rows:(at + 1) * rows] == 0).all() and (lse[at * rows:(at + 1) * rows] == -math.inf).all()
    if window == 0:  # every position of the table
        su.lens[0] = su.cols * su.page + rows
        compare(su, q, 0.1, window, 0.0, out, lse, slice(0, rows))
    su.cache.append(su.batch, q[:, :2].contiguous(), q[:, 2:4].contiguous())
    torch.cuda.synchronize()


def test_numbers_out_of_range_are_refused():
    su = Setup("q8", 128, 2, 16, [20], [2])
    q = queries(su, 4, "bf16")
    for kw in (dict(window=2 ** 31), dict(window=-2 ** 31 - 1), dict(window=1.5), dict(scale=1e39), dict(softcap=1e300),
               dict(scale="1"), dict(softcap=None)):
        with pytest.raises(ArgumentError):
            su.cache.attention(su.batch, q, **{"scale": 0.1, **kw})
    for max_rows in (-1, 2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ArgumentError):
            PagedBatch(su.table, su.seq_len, su.row_start, max_rows=max_rows)


@pytest.mark.parametrize("kv,act,hd", [("q8", "bf16", 128), ("f16", "f32", 64)])
@pytest.mark.parametrize("hint", [1, 64])
def test_more_sequences_than_threads_of_a_block(kv, act, hd, hint):
    """Schedules in which a thread adds up several sequences; most have a row, some none, a few a prompt."""
    g = torch.Generator().manual_seed(hd)
    rows = [(1, 1, 1, 0, 2, 20)[int(x)] for x in torch.randint(0, 6, (1700,), generator=g)]
    lens = [r + int(x) for r, x in zip(rows, torch.randint(0, 60, (1700,), generator=g))]
    su = Setup(kv, hd, 2, 16, lens, rows, seed=hint)
    su.batch = PagedBatch(su.table, su.seq_len, su.row_start, max_rows=hint)
    check(su, queries(su, 8, act), 1 / math.sqrt(hd), window=40)
