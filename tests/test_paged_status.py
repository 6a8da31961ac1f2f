"""Argument checks of the paged attention's status query and of its test hook, and of overlapping and
unaligned arrays, before any device work (pointers are never followed)."""
from __future__ import annotations

import ctypes as C

import pytest

from dotnetfoundryllm_b200 import _native as N
from test_paged_refusals import P, attn, batch, kv, verify


def test_status_needs_a_place_for_the_count():
    assert N.cuda().fl_attn_paged_status(None, None) == N.FL_ERR_ARG


def test_stall_is_refused_without_waits():
    lib, c = N.cuda(), kv()
    one, many = batch(n_seqs=1, max_rows=1), batch(n_seqs=1, max_rows=500)
    assert lib.fl_attn_paged_stall(C.byref(c), C.byref(one), C.byref(attn()), None) == N.FL_ERR_ARG
    assert "no waits" in N.last_error()
    assert lib.fl_attn_paged_stall(C.byref(c), C.byref(many), C.byref(attn(n_heads=7)), None) == N.FL_ERR_ARG


def test_verified_tokens_may_not_go_over_the_drafts():
    lib = N.cuda()
    for off in (-12, -4, 0, 4, 12):
        assert lib.fl_verify_device(C.byref(verify(draft=1 << 20, tokens=(1 << 20) + off)), None) == N.FL_ERR_ARG
        assert "overlap" in N.last_error()


@pytest.mark.parametrize("name", ["page_table", "seq_len", "row_start"])
def test_batches_off_their_alignment_are_refused_by_every_call(name):
    lib, c, b = N.cuda(), kv(), batch(**{name: (1 << 20) + 2})
    assert lib.fl_kv_append_device(C.byref(c), C.byref(b), 1, 4, P, 256, P, 256, None) == N.FL_ERR_ARG
    assert lib.fl_kv_gather_device(C.byref(c), C.byref(b), 1, 4, P, 256, P, 256, None) == N.FL_ERR_ARG
    assert lib.fl_attn_paged_device(C.byref(c), C.byref(b), C.byref(attn()), None) == N.FL_ERR_ARG
    assert "aligned" in N.last_error()


def test_lse_off_its_alignment_is_refused():
    assert N.cuda().fl_attn_paged_device(C.byref(kv()), C.byref(batch()), C.byref(attn(lse=P + 2)), None) == N.FL_ERR_ARG
    assert "lse" in N.last_error()


@pytest.mark.parametrize("name", ["row_start", "draft", "temperature", "u_accept", "u_sample", "tokens", "accepted"])
def test_verify_arrays_off_their_alignment_are_refused(name):
    over = dict(draft=1 << 20, tokens=1 << 21)
    over[name] = (1 << 22) + 1
    assert N.cuda().fl_verify_device(C.byref(verify(**over)), None) == N.FL_ERR_ARG
    assert "aligned" in N.last_error()
