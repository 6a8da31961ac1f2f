"""Argument checks of the paged attention's status query, of its test hook and of overlapping arrays, before any device work."""
from __future__ import annotations

import ctypes as C

from dotnetfoundryllm_b200 import _native as N
from test_paged_refusals import attn, batch, kv, verify


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
