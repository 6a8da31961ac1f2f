"""Argument checks of the paged-cache operators and of verify: refused before
any device work, so none of this needs a GPU (pointers are never followed)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from dotnetfoundryllm_b200 import _native as N
from dotnetfoundryllm_b200 import paged, speculate
from dotnetfoundryllm_b200.runtime import ArgumentError, NotSupportedError

P = 4096  # a pointer that is never followed


def kv(**over):
    f = dict(struct_size=C.sizeof(N.FlPagedKv), kv_dtype=N.FL_KV_Q8, n_pages=4, page_size=16, n_kv_heads=2, head_dim=128,
             k=P, v=P, k_scale=P, v_scale=P)
    f.update(over)
    return N.FlPagedKv(**f)


def batch(**over):
    f = dict(struct_size=C.sizeof(N.FlPagedBatch), n_seqs=2, table_cols=3, max_rows=0, page_table=P, seq_len=P, row_start=P)
    f.update(over)
    return N.FlPagedBatch(**f)


def attn(**over):
    f = dict(struct_size=C.sizeof(N.FlPagedAttnDesc), type=1, n_rows=4, n_heads=8, window=0, scale=0.1, softcap=0.0, reserved=0,
             q=P, q_stride=1024, out=P, out_stride=1024, lse=None, workspace=P, workspace_bytes=1 << 40)
    f.update(over)
    return N.FlPagedAttnDesc(**f)


def verify(**over):
    f = dict(struct_size=C.sizeof(N.FlVerifyDesc), type=0, n_rows=4, n_seqs=2, vocab=100, reserved=0, logits=P,
             logits_stride=100, draft_probs=None, probs_stride=0, row_start=P, draft=P, temperature=P, u_accept=P, u_sample=P,
             tokens=P, accepted=P, workspace=P, workspace_bytes=1 << 40)
    f.update(over)
    return N.FlVerifyDesc(**f)


BAD_CACHE = [
    (dict(struct_size=4), N.FL_ERR_ARG),
    (dict(kv_dtype=N.FL_KV_F32), N.FL_ERR_UNSUPPORTED),
    (dict(kv_dtype=9), N.FL_ERR_UNSUPPORTED),
    (dict(head_dim=96), N.FL_ERR_UNSUPPORTED),
    (dict(page_size=24), N.FL_ERR_ARG),
    (dict(page_size=8), N.FL_ERR_ARG),
    (dict(page_size=2048), N.FL_ERR_ARG),
    (dict(n_pages=0), N.FL_ERR_ARG),
    (dict(n_kv_heads=0), N.FL_ERR_ARG),
    (dict(k=None), N.FL_ERR_ARG),
    (dict(v=P + 8), N.FL_ERR_ARG),
    (dict(k_scale=None), N.FL_ERR_ARG),
    (dict(v_scale=None), N.FL_ERR_ARG),
]
BAD_BATCH = [
    (dict(struct_size=8), N.FL_ERR_ARG),
    (dict(n_seqs=-1), N.FL_ERR_ARG),
    (dict(table_cols=-1), N.FL_ERR_ARG),
    (dict(table_cols=1 << 28), N.FL_ERR_ARG),
    (dict(max_rows=-1), N.FL_ERR_ARG),
    (dict(page_table=None), N.FL_ERR_ARG),
    (dict(seq_len=None), N.FL_ERR_ARG),
    (dict(row_start=None), N.FL_ERR_ARG),
]


@pytest.mark.parametrize("over,code", BAD_CACHE)
def test_bad_cache_is_refused_by_every_call(over, code):
    lib, c, b = N.cuda(), kv(**over), batch()
    n = C.c_uint64()
    assert lib.fl_kv_append_device(C.byref(c), C.byref(b), 1, 4, P, 256, P, 256, None) == code
    assert lib.fl_kv_gather_device(C.byref(c), C.byref(b), 1, 4, P, 256, P, 256, None) == code
    assert lib.fl_attn_paged_workspace(C.byref(c), C.byref(b), 4, 8, C.byref(n)) == code
    assert lib.fl_attn_paged_device(C.byref(c), C.byref(b), C.byref(attn()), None) == code
    assert N.last_error() != ""


@pytest.mark.parametrize("over,code", BAD_BATCH)
def test_bad_batch_is_refused_by_every_call(over, code):
    lib, c, b = N.cuda(), kv(), batch(**over)
    assert lib.fl_kv_append_device(C.byref(c), C.byref(b), 1, 4, P, 256, P, 256, None) == code
    assert lib.fl_kv_gather_device(C.byref(c), C.byref(b), 1, 4, P, 256, P, 256, None) == code
    assert lib.fl_attn_paged_device(C.byref(c), C.byref(b), C.byref(attn()), None) == code


@pytest.mark.parametrize("args,code", [
    ((2, 4, P, 256, P, 256), N.FL_ERR_UNSUPPORTED),   # Q4_0 rows
    ((1, -1, P, 256, P, 256), N.FL_ERR_ARG),
    ((1, 4, None, 256, P, 256), N.FL_ERR_ARG),
    ((1, 4, P, 256, None, 256), N.FL_ERR_ARG),
    ((1, 4, P, 255, P, 256), N.FL_ERR_ARG),           # rows overlap
    ((1, 4, P, 260, P, 256), N.FL_ERR_ARG),           # rows not 16-byte aligned
    ((0, 4, P, 256, P, 258), N.FL_ERR_ARG),
    ((1, 4, P + 2, 256, P, 256), N.FL_ERR_ARG),
])
def test_bad_rows_are_refused(args, code):
    lib, c, b = N.cuda(), kv(), batch()
    assert lib.fl_kv_append_device(C.byref(c), C.byref(b), *args, None) == code
    assert lib.fl_kv_gather_device(C.byref(c), C.byref(b), *args, None) == code


@pytest.mark.parametrize("over,code", [
    (dict(struct_size=4), N.FL_ERR_ARG),
    (dict(type=12), N.FL_ERR_UNSUPPORTED),
    (dict(n_heads=7), N.FL_ERR_ARG),                  # not a multiple of the kv heads
    (dict(n_heads=0), N.FL_ERR_ARG),
    (dict(n_rows=-2), N.FL_ERR_ARG),
    (dict(n_rows=1 << 30), N.FL_ERR_ARG),             # rows x heads past 32 bits
    (dict(scale=float("nan")), N.FL_ERR_ARG),
    (dict(softcap=float("inf")), N.FL_ERR_ARG),
    (dict(scale=3e38), N.FL_ERR_ARG),                 # out of range in units of log2
    (dict(softcap=1e-40), N.FL_ERR_ARG),              # scale / softcap likewise
    (dict(reserved=1), N.FL_ERR_ARG),
    (dict(q=None), N.FL_ERR_ARG),
    (dict(q=P + 4), N.FL_ERR_ARG),
    (dict(q_stride=1000), N.FL_ERR_ARG),
    (dict(out=None), N.FL_ERR_ARG),
    (dict(out_stride=1028), N.FL_ERR_ARG),
    (dict(workspace=P + 16), N.FL_ERR_ARG),
])
def test_bad_attention_is_refused(over, code):
    lib, c, b = N.cuda(), kv(), batch()
    assert lib.fl_attn_paged_device(C.byref(c), C.byref(b), C.byref(attn(**over)), None) == code
    assert N.last_error() != ""


def test_a_workspace_that_is_too_small_is_refused():
    lib, c, b = N.cuda(), kv(), batch()
    n = C.c_uint64()
    assert lib.fl_attn_paged_workspace(C.byref(c), C.byref(b), 4, 8, C.byref(n)) == N.FL_OK
    if n.value:
        a = attn(workspace_bytes=n.value - 1)
        assert lib.fl_attn_paged_device(C.byref(c), C.byref(b), C.byref(a), None) == N.FL_ERR_ARG
    assert lib.fl_verify_workspace(4, 2, 100, C.byref(n)) == N.FL_OK and n.value > 0
    assert lib.fl_verify_device(C.byref(verify(workspace_bytes=n.value - 1)), None) == N.FL_ERR_ARG
    assert "workspace" in N.last_error()


@pytest.mark.parametrize("over,code", [
    (dict(struct_size=4), N.FL_ERR_ARG),
    (dict(type=8), N.FL_ERR_UNSUPPORTED),
    (dict(n_rows=-1), N.FL_ERR_ARG),
    (dict(n_seqs=-1), N.FL_ERR_ARG),
    (dict(n_seqs=1 << 29), N.FL_ERR_ARG),
    (dict(draft_probs=P + 2, probs_stride=100), N.FL_ERR_ARG),
    (dict(vocab=0), N.FL_ERR_ARG),
    (dict(vocab=(1 << 24) + 1, logits_stride=1 << 25), N.FL_ERR_ARG),
    (dict(reserved=3), N.FL_ERR_ARG),
    (dict(logits=None), N.FL_ERR_ARG),
    (dict(logits=P + 2), N.FL_ERR_ARG),
    (dict(logits_stride=99), N.FL_ERR_ARG),
    (dict(draft_probs=P, probs_stride=50), N.FL_ERR_ARG),
    (dict(row_start=None), N.FL_ERR_ARG),
    (dict(draft=None), N.FL_ERR_ARG),
    (dict(temperature=None), N.FL_ERR_ARG),
    (dict(u_accept=None), N.FL_ERR_ARG),
    (dict(u_sample=None), N.FL_ERR_ARG),
    (dict(tokens=None), N.FL_ERR_ARG),
    (dict(accepted=None), N.FL_ERR_ARG),
    (dict(workspace=None), N.FL_ERR_ARG),
])
def test_bad_verification_is_refused(over, code):
    assert N.cuda().fl_verify_device(C.byref(verify(**over)), None) == code
    assert N.last_error() != ""


def test_nothing_to_do_is_not_an_error():
    lib, c = N.cuda(), kv()
    none = batch(n_seqs=0, page_table=None, seq_len=None, row_start=None)
    assert lib.fl_kv_append_device(C.byref(c), C.byref(none), 1, 0, None, 0, None, 0, None) == N.FL_OK
    assert lib.fl_kv_gather_device(C.byref(c), C.byref(batch()), 1, 0, None, 0, None, 0, None) == N.FL_OK
    a = attn(n_rows=0, q=None, out=None, workspace=None, workspace_bytes=0)
    assert lib.fl_attn_paged_device(C.byref(c), C.byref(batch()), C.byref(a), None) == N.FL_OK
    assert lib.fl_verify_device(C.byref(verify(n_seqs=0, n_rows=0)), None) == N.FL_OK


def test_descriptor_layouts_match_the_header():
    assert C.sizeof(N.FlPagedKv) == 6 * 4 + 4 * 8
    assert C.sizeof(N.FlPagedBatch) == 4 * 4 + 3 * 8
    assert C.sizeof(N.FlPagedAttnDesc) == 8 * 4 + 7 * 8
    assert C.sizeof(N.FlVerifyDesc) == 6 * 4 + 13 * 8


def test_host_tensors_are_refused():
    t = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ArgumentError):
        paged.PagedBatch(t, t[0], t[0])
    x = torch.zeros(4, 2, 16, 128, dtype=torch.float16)
    with pytest.raises(ArgumentError):
        paged.PagedKvCache(x, x)
    with pytest.raises(NotSupportedError):
        paged.PagedKvCache.empty(4, 16, 2, 128, torch.float32, device="cpu")
    with pytest.raises(ArgumentError):
        speculate.verify_drafts(torch.zeros(2, 10), t[0], t[0], t[0], t[0], t[0])
