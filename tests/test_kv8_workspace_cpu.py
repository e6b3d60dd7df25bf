"""The workspace of prefill calls over 8-bit pages: what it holds beyond the same call's over bf16 pages (no GPU)."""

from __future__ import annotations

import ctypes

import numpy as np
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


def _ragged(counts, host=True, **kw):
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    args = dict(batch=len(counts), tokens=int(cu[-1]), cu_seqlens_q=16, max_seqlen_q=max(counts), older_len=16, older_capacity_tokens=8192,
                older_table_stride=256, **kw)
    return sizes(**args, **(dict(cu_seqlens_q_host=cu.ctypes.data) if host else {}))


@pytest.mark.parametrize("counts,tiles", [([1] * 31 + [512], 1), ([17, 16, 40, 1, 1, 16], 2), ([16] * 9, 0), ([17] * 5, 5)])
def test_only_sequences_on_the_tiles_have_copies(counts, tiles):
    """Groups of 4: those above 16 tokens, as the host's offsets say."""

    eight, bf16 = _ragged(counts)
    assert eight - bf16 == ops.kv8_copy_bytes(tiles, 2, 8192, len(counts))
    eight, bf16 = _ragged(counts, host=False)  # (as many as the rows allow)
    most = min(len(counts), sum(counts) // 17) if max(counts) > 16 else 0
    assert eight - bf16 == ops.kv8_copy_bytes(most, 2, 8192, len(counts)) and most >= tiles
    if max(counts) <= 16:  # (a call of short ones alone that is put on the tile kernel)
        eight, bf16 = _ragged(counts, tile_waves=4)
        assert eight - bf16 == ops.kv8_copy_bytes(len(counts), 2, 8192, len(counts))
