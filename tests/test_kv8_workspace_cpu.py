"""The workspace of prefill calls over 8-bit pages: what it holds beyond the same call's over bf16 pages (no GPU)."""

from __future__ import annotations

import ctypes

import pytest

from lastkv_amd import _lib, ops
from test_pages_cpu import _prefill


def sizes(**kw):
    lib = _lib.load()
    a = _prefill(**kw)
    b = _prefill(older_k=16, older_v=16, older_num_pages=10, older_page_stride=4096, older_head_stride=40960, **kw)
    return lib.lkv_prefill_kv8_workspace_bytes(ctypes.byref(a)), lib.lkv_prefill_workspace_bytes(ctypes.byref(b))


@pytest.mark.parametrize("batch,tokens,older", [(1, 40, 100), (3, 17, 128), (32, 1024, 8192), (2, 100, 31)])
def test_tiles_take_the_bf16_call_s_and_one_copy_of_k(batch, tokens, older):
    """As much again as the codes, so that pages, copies and fp16 V together are never more than bf16 pages and fp16 V."""

    cap = -(-older // 32) * 32
    eight, bf16 = sizes(batch=batch, tokens=tokens, older_len_const=older, older_capacity_tokens=cap, older_table_stride=cap // 32)
    assert eight - bf16 == batch * 2 * (cap // 32) * 8192 == ops.kv8_copy_bytes(batch, 2, older)


@pytest.mark.parametrize("tokens", [1, 4, 16])
def test_short_calls_take_nothing_more(tokens):
    eight, bf16 = sizes(tokens=tokens)
    assert eight == bf16
