"""The custom operators of the 8-bit cache, page copies and beam selection without a GPU: the tensors their schemas say they
write, the shapes their fake forms give, and the key splits of a decode call."""

from __future__ import annotations

import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from lastkv_amd import ops
import lastkv_amd.torch_ops  # noqa: F401

L = torch.ops.lastkv


def written(name):
    schema = getattr(L, name).default._schema
    return {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write}


def test_schemas_name_what_is_written():
    assert written("kv8_quantize") == {"dst_k", "dst_v", "dst_k_scales", "dst_v_scales"}
    assert written("copy_pages") == {"k", "v", "k_scales", "v_scales"}
    for name in ("kv8_unpack", "decode_attention_kv8", "prefill_attention_kv8", "beam_select"):
        assert written(name) == set(), name


def test_fake_shapes():
    with FakeTensorMode():
        codes = torch.empty((8, 12, 4096), dtype=torch.float8_e4m3fn)
        scales = torch.empty((8, 12), dtype=torch.uint8)
        table = torch.empty((3, 4), dtype=torch.int32)
        k, v = L.kv8_unpack(codes, codes, scales, scales, table, 5, 40)
        assert k.shape == v.shape == (3, 8, 40, 128) and k.dtype == v.dtype == torch.bfloat16
        q = torch.empty((3, 32, 128), dtype=torch.bfloat16)
        out = L.decode_attention_kv8(q, codes, codes, scales, scales, None, 100, table, None, None, None, None, 0, None, 0, None,
                                     0, 0.0, 0)
        assert out.shape == q.shape and out.dtype == q.dtype
        qp = torch.empty((3, 7, 32, 128), dtype=torch.bfloat16)
        out = L.prefill_attention_kv8(qp, codes, codes, scales, scales, None, 100, table, None, None, None, None, 0, None, 0,
                                      None, 0, True, 0.0)
        assert out.shape == qp.shape
        got = L.beam_select(torch.empty((2, 4, 999)), torch.empty((2, 4)), 8)
        assert [t.shape for t in got] == [(2, 8)] * 3
        assert [t.dtype for t in got] == [torch.float32, torch.int32, torch.int32]
        assert L.copy_pages(codes, codes, scales, scales, [0], [1]) is None
        pool = torch.empty((8, 12, 4096), dtype=torch.bfloat16)
        assert L.kv8_quantize(pool, pool, codes, codes, scales, scales, table, table, None, 64) is None


def test_default_decode_splits():
    splits = lambda B, tokens, older8: ops.default_decode_splits(B, 8, tokens, 256, older8)
    for B, tokens in ((1, 500), (7, 9300), (20, 9300), (32, 9300), (56, 9300), (64, 9300), (40, 2000)):
        assert splits(B, tokens, True) == splits(B, tokens, False), (B, tokens)
    for B, tokens, want in ((34, 9300, 4), (40, 9300, 4), (48, 9300, 2), (72, 9300, 4), (33, 40000, 8)):
        assert splits(B, tokens, True) == want and splits(B, tokens, False) == 1, (B, tokens)
