"""Host logic of shared pages: forks and compaction of the allocator, and the C entry points' refusals (no GPU)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from lastkv_amd import _lib
from lastkv_amd.serving import PageAllocator


class Pages:
    """What the pages hold, as the copies of a compaction move it."""

    def __init__(self, n):
        self.data = np.full(n, -1)

    def copy(self, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst) and len(src) == len(dst) > 0
        self.data[dst] = self.data[src]


@pytest.mark.parametrize("seed", range(6))
def test_random_forks_and_compactions(seed):
    rng = np.random.default_rng(seed)
    n, width, slots = 60, 12, 8
    al, mem = PageAllocator(max_slots=slots, pages=n, width=width, scratch=n), Pages(n)
    want = {}  # slot -> the values its blocks hold
    fresh = iter(range(10 ** 6))
    for step in range(600):
        op = rng.integers(5)
        if op == 0 and len(want) < slots:
            want[al.open_slot()] = []
        elif op == 1 and want:
            s = int(rng.choice(list(want)))
            grow = int(rng.integers(1, 4))
            if len(want[s]) + grow <= width and grow <= al.free_pages:
                al.reserve(s, 32 * (len(want[s]) + grow))
                for j in range(len(want[s]), len(want[s]) + grow):
                    v = next(fresh)
                    mem.data[al.table[s, j]] = v
                    want[s].append(v)
        elif op == 2 and want and len(want) < slots:
            s = int(rng.choice(list(want)))
            shared = int(rng.integers(0, len(want[s]) + 1))
            if len(want[s]) - shared > al.free_pages:
                with pytest.raises(RuntimeError):
                    al.fork(s, shared)
                continue
            f = al.fork(s, shared)
            assert f not in want
            want[f] = want[s][:shared]
            for j in range(shared, len(want[s])):  # pages of its own
                v = next(fresh)
                mem.data[al.table[f, j]] = v
                want[f].append(v)
        elif op == 3 and want and rng.random() < 0.5:
            s = int(rng.choice(list(want)))
            al.close_slot(s)
            del want[s]
            assert (al.table[s] == n).all()
        elif op == 4 and rng.random() < 0.3:
            free = al.free_pages
            for src, dst in al.compact():
                mem.copy(src, dst)
            assert al.free_pages == free
            if free:  # every page stands where the slots' order puts it
                order = list(dict.fromkeys(int(p) for s in range(slots) for p in al.table[s, :al.used[s]]))
                assert order == list(range(len(order)))
            assert al.compact() == [] or not free
        for s, v in want.items():
            assert mem.data[al.table[s, :al.used[s]]].tolist() == v and (al.table[s, al.used[s]:] == n).all()
        used = {int(p) for s in want for p in al.table[s, :al.used[s]]}
        assert len(used) + al.free_pages == n and not used & set(al._free_pages)
        for p in range(n):
            assert al.refs[p] == sum((al.table[s, :al.used[s]] == p).sum() for s in want)


def _copy_args(pages, to, **kw):
    a = _lib.CopyPagesArgs()
    a.struct_size = ctypes.sizeof(a)
    s, d = np.array(pages, dtype=np.int32), np.array(to, dtype=np.int32)
    a.count, a.heads, a.num_pages, a.page_bytes = len(pages), 2, 64, 8192
    a.page_stride, a.head_stride = 8192, 64 * 8192
    a.src, a.dst, a.k, a.v = s.ctypes.data, d.ctypes.data, 4096, 8192
    for k, v in kw.items():
        setattr(a, k, v)
    return a, (s, d)


@pytest.mark.parametrize("src,dst,message", [([1], [1], b"source and a destination"), ([1, 2], [5, 5], b"destination twice"),
                                             ([5, 1], [6, 5], b"source and a destination"), ([-1], [2], b"outside"),
                                             ([1], [64], b"outside"), ([64], [1], b"outside")])
def test_copy_pages_refuses_lists_without_one_result(src, dst, message):
    lib = _lib.load()
    a, keep = _copy_args(src, dst)
    assert lib.lkv_copy_pages(ctypes.byref(a), None) == 1 and message in lib.lkv_last_error()


@pytest.mark.parametrize("kw,message", [(dict(struct_size=8), b"size"), (dict(page_bytes=100), b"page_bytes"), (dict(heads=0), b"sizes"),
                                        (dict(count=-1), b"sizes"), (dict(num_pages=0), b"sizes"), (dict(k=0), b"null"),
                                        (dict(v=8), b"aligned"), (dict(page_stride=4096), b"overlap"), (dict(src=0), b"null"),
                                        (dict(k_scales=64), b"both"), (dict(heads=70000), b"65535")])
def test_copy_pages_refuses_bad_arguments(kw, message):
    lib = _lib.load()
    a, keep = _copy_args([1], [2], **kw)
    assert lib.lkv_copy_pages(ctypes.byref(a), None) == 1 and message in lib.lkv_last_error()


@pytest.mark.parametrize("pages", [64, 4096, 1 << 20])
@pytest.mark.parametrize("n", [2, 9, 40, 64])
def test_copy_pages_finds_a_wrong_pair_anywhere(n, pages):
    """Lists of few and many pairs, of small and large pools, with one page that is a destination twice or on both sides."""

    lib = _lib.load()
    rng = np.random.default_rng(n + pages)
    for _ in range(20):
        ids = rng.permutation(min(pages, 500))[:2 * n] if 2 * n <= min(pages, 500) else rng.permutation(pages)
        n = min(n, len(ids) // 2)
        src, dst = ids[:n].tolist(), ids[n:2 * n].tolist()
        i, j = (int(x) for x in rng.choice(n, 2, replace=False))
        for lists, message in ((([*src], [dst[j] if k == i else d for k, d in enumerate(dst)]), b"destination twice"),
                               (([dst[j] if k == i else x for k, x in enumerate(src)], dst), b"source and a destination"),
                               ((src, [pages if k == i else d for k, d in enumerate(dst)]), b"outside")):
            a, keep = _copy_args(*lists, num_pages=pages, head_stride=pages * 8192)
            assert lib.lkv_copy_pages(ctypes.byref(a), None) == 1 and message in lib.lkv_last_error()


def test_copy_pages_of_nothing_launches_nothing():
    lib = _lib.load()
    a, keep = _copy_args([], [])
    assert lib.lkv_copy_pages(ctypes.byref(a), None) == 0


def _pool(**kw):
    p = _lib.Kv8Pool()
    p.struct_size = ctypes.sizeof(p)
    p.num_pages, p.heads = 10, 2
    p.k, p.v, p.k_scales, p.v_scales = 4096, 8192, 16, 32
    p.page_stride, p.head_stride, p.scale_head_stride = 4096, 40960, 12
    for k, v in kw.items():
        setattr(p, k, v)
    return p


POOLS = [(dict(struct_size=0), b"size"), (dict(k=0), b"null"), (dict(v_scales=0), b"null"), (dict(num_pages=0), b"pages"),
         (dict(k=8), b"aligned"), (dict(page_stride=2048), b"strides"), (dict(head_stride=8), b"strides"),
         (dict(k_scales=18), b"scales"), (dict(scale_head_stride=10), b"scales"), (dict(scale_head_stride=8), b"scales")]


def _decode(**kw):
    a = _lib.DecodeArgs()
    a.struct_size = ctypes.sizeof(a)
    a.batch, a.num_q_heads, a.num_kv_heads, a.head_dim, a.num_splits = 1, 8, 2, 128, 1
    a.q = a.out = a.older_block_table = 16
    a.older_table_stride, a.older_capacity_tokens = 4, 128
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _prefill(**kw):
    a = _lib.PrefillArgs()
    a.struct_size = ctypes.sizeof(a)
    a.batch, a.tokens, a.num_q_heads, a.num_kv_heads, a.head_dim = 1, 40, 8, 2, 128
    a.q = a.out = a.older_block_table = 16
    a.older_table_stride, a.older_capacity_tokens, a.older_len_const = 4, 128, 100
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,message", POOLS)
def test_every_call_refuses_a_bad_8_bit_pool(kw, message):
    lib = _lib.load()
    pool = _pool(**kw)
    q = _lib.Kv8QuantizeArgs()
    q.struct_size = ctypes.sizeof(q)
    for status in (lib.lkv_kv8_quantize(ctypes.byref(q), ctypes.byref(pool), None),
                   lib.lkv_kv8_unpack(ctypes.byref(pool), 16, 1, 1, 1, 0, 1, 16, 0, 0, 128, 16, 0, 0, 128, None),
                   lib.lkv_decode_attn_kv8(ctypes.byref(_decode()), ctypes.byref(pool), None),
                   lib.lkv_prefill_attn_kv8(ctypes.byref(_prefill()), ctypes.byref(pool), None)):
        assert status == 1 and message in lib.lkv_last_error()


@pytest.mark.parametrize("kw,message", [(dict(older_k=16, older_v=16), b"NULL"), (dict(older_block_table=0), b"older_block_table"),
                                        (dict(num_kv_heads=4), b"kv heads"), (dict(older_capacity_tokens=33), b"multiple of 32"),
                                        (dict(older_table_stride=3), b"older_table_stride")])
def test_attention_refuses_bad_8_bit_segments(kw, message):
    lib = _lib.load()
    pool = _pool()
    assert lib.lkv_decode_attn_kv8(ctypes.byref(_decode(**kw)), ctypes.byref(pool), None) == 1 and message in lib.lkv_last_error()
    a = _prefill(workspace=16, workspace_bytes=1 << 40, **kw)
    assert lib.lkv_prefill_attn_kv8(ctypes.byref(a), ctypes.byref(pool), None) == 1 and message in lib.lkv_last_error()


def test_prefill_over_8_bits_needs_room_for_its_copies():
    lib = _lib.load()
    need = lib.lkv_prefill_kv8_workspace_bytes(ctypes.byref(_prefill()))
    copies = 1 * 2 * 4 * 2 * 8192
    assert need > copies
    a = _prefill(workspace=16, workspace_bytes=copies)
    assert lib.lkv_prefill_attn_kv8(ctypes.byref(a), ctypes.byref(_pool()), None) == 1 and b"workspace" in lib.lkv_last_error()
    a = _prefill(workspace=16, workspace_bytes=copies + 16)
    assert lib.lkv_prefill_attn_kv8(ctypes.byref(a), ctypes.byref(_pool()), None) == 1 and b"workspace" in lib.lkv_last_error()
    # short calls, which run on the decode kernel, copy nothing
    assert lib.lkv_prefill_kv8_workspace_bytes(ctypes.byref(_prefill(tokens=4))) < copies


def _quantize(**kw):
    a = _lib.Kv8QuantizeArgs()
    a.struct_size = ctypes.sizeof(a)
    a.batch, a.heads, a.head_dim, a.blocks, a.src_num_pages = 1, 2, 128, 1, 4
    a.src_k = a.src_v = a.src_table = a.dst_table = 16
    a.src_table_width = a.dst_table_width = 2
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,message", [(dict(struct_size=1), b"size"), (dict(head_dim=64), b"head_dim"), (dict(batch=-1), b"sizes"),
                                        (dict(heads=3), b"heads"), (dict(src_k=0), b"null"), (dict(src_num_pages=0), b"src_num_pages"),
                                        (dict(src_v=8), b"aligned"), (dict(tokens_const=-1), b"negative"), (dict(blocks=3), b"exceed"),
                                        (dict(first_block=2), b"exceed"), (dict(first_block=-1), b"sizes"), (dict(dst_table_width=0), b"exceed"),
                                        (dict(batch=70000), b"65535")])
def test_quantize_refuses_bad_arguments(kw, message):
    lib = _lib.load()
    assert lib.lkv_kv8_quantize(ctypes.byref(_quantize(**kw)), ctypes.byref(_pool()), None) == 1 and message in lib.lkv_last_error()


def _beam(**kw):
    a = _lib.BeamSelectArgs()
    a.struct_size = ctypes.sizeof(a)
    a.batch, a.beams, a.vocab, a.count = 1, 2, 100, 4
    a.logits = a.scores = a.out_scores = a.out_beams = a.out_tokens = a.workspace = 16
    a.workspace_bytes = 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,status,message", [
    (dict(struct_size=1), 1, b"size"), (dict(batch=-1), 1, b"sizes"), (dict(beams=0), 1, b"beams"), (dict(beams=65), 1, b"beams"),
    (dict(vocab=0), 1, b"vocab"), (dict(vocab=(1 << 20) + 1), 1, b"vocab"), (dict(count=0), 1, b"count"), (dict(count=65), 1, b"count"),
    (dict(logits_fp32=2), 1, b"logits_fp32"), (dict(logits=0), 1, b"null"), (dict(logits=17), 1, b"aligned"),
    (dict(logits=18, logits_fp32=1), 1, b"aligned"), (dict(batch=40000), 1, b"65535"), (dict(workspace_bytes=8), 3, b"workspace"),
    (dict(workspace=0), 3, b"workspace"), (dict(workspace=24), 1, b"aligned")])
def test_beam_select_refuses_bad_arguments(kw, status, message):
    lib = _lib.load()
    assert lib.lkv_beam_select(ctypes.byref(_beam(**kw)), None) == status and message in lib.lkv_last_error()


def test_beam_workspace_size():
    lib = _lib.load()
    assert lib.lkv_beam_workspace_bytes(0, 2, 100, 4) == 0
    assert lib.lkv_beam_workspace_bytes(1, 2, 100, 4) == 2 * (16 + 4 * 8)
    assert lib.lkv_beam_workspace_bytes(1, 1, 2048, 4) == 2 * (16 + 4 * 8)  # (a row may begin inside a 16-byte piece)
    assert lib.lkv_beam_workspace_bytes(16, 8, 128256, 16) == 128 * 16 * (16 + 16 * 8)
