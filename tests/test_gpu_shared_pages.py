"""The serving path over an 8-bit shared cache, forked sequences, compaction and beam search (gpu)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from lastkv_amd import ops
from lastkv_amd.serving import LastKVFastPath, LastKVPagePool, LastKVServingModel

from test_gpu_kv8 import attention64, check
from test_gpu_llm import _tiny
from test_gpu_serving import _rotary

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _path(shared_cache, C, Hq, Hkv, layers, cap, slots, seed, contract):
    g = torch.Generator(device=DEV).manual_seed(seed)
    params = []
    for _ in range(layers):
        w = (torch.rand(128, generator=g, device=DEV) + 0.5).bfloat16()
        vs = (torch.rand(Hkv, generator=g, device=DEV) + 0.4).bfloat16().float()
        params.append((w, w.flip(0).contiguous(), 1e-5, vs))
    alpha = torch.rand(layers * Hkv, generator=g, device=DEV).bfloat16().float()
    blend = (alpha, (1 - alpha).bfloat16().float(), torch.cat([p[3] for p in params]))
    pool = LastKVPagePool(num_layers=layers, kv_heads=Hkv, chunk_size=C, max_slots=slots, source_pages=slots * cap // 32 + 8,
                          max_tokens_per_slot=cap, device=DEV, shared_cache=shared_cache)
    return pool, LastKVFastPath(pool, num_q_heads=Hq, layer_params=params, blend=blend, rotary=_rotary, max_batch=slots + 2,
                                num_splits=2, contract=contract)


def _tokens(pool, table, kind, lo, hi):
    """Tokens [lo, hi) of one table row of a bf16 pool, [H, hi - lo, 128]."""

    pages = pool.kp[table.long()] if kind == 0 else pool.vp[table.long()]  # [W, H, 4096]
    cache = pages.transpose(0, 1).contiguous()[None]                       # as one slot of a tiled cache
    return ops.cache_unpack(cache, kind, lo, hi - lo, 1)[0]


@pytest.mark.parametrize("contract", ["hf", "vllm"])
@pytest.mark.parametrize("seed,C", [(0, 8), (1, 24), (2, 32), (3, 40), (4, 100)])
def test_8_bit_history_next_to_a_bf16_twin(seed, C, contract):
    """Random schedules with forks, frees and compactions on both kinds of pool: the rings are the twin's bit for bit, the 8-bit
    pages are the twin's history quantised in one go, and the outputs are the attention over them in 64 bits."""

    rng = np.random.default_rng(seed)
    Hkv, layers, cap, slots = 2, 2, 352, 4
    Hq = Hkv * int(rng.choice([1, 4]))
    (ref, a), (pool, b) = (_path(kind, C, Hq, Hkv, layers, cap, slots, seed, contract) for kind in ("bf16", "kv8"))
    free = pool.free_pages
    g = torch.Generator(device=DEV).manual_seed(seed + 50)
    live = []
    for step in range(70):
        while len(live) < 2:
            live.append(a.add_sequence())
            assert b.add_sequence() == live[-1]
        if rng.random() < 0.15 and len(live) < slots:
            s = int(rng.choice(live))
            live.append(a.fork_sequence(s))
            assert b.fork_sequence(s) == live[-1]
        if rng.random() < 0.1:
            ref.compact()
            pool.compact()
        rows = []
        for s in live:
            p = a.seen(s)
            n = min(cap - p, C - p % C)
            if n > 0 and rng.random() < 0.8:
                rows.append((s, int(rng.integers(1, n + 1)) if rng.random() < 0.6 else 1))
        if not rows:
            continue
        T = sum(n for _, n in rows)
        x = [torch.randn((T, h * 128), generator=g, device=DEV).bfloat16() for h in (Hq, Hkv, Hkv)]
        # (a row of a fork must not repeat its parent's tokens: every row has its own)
        for path in (a, b):
            path.prepare(rows)
        for l in range(layers):
            outs = [torch.empty((T, Hq, 128), dtype=torch.bfloat16, device=DEV) for _ in range(2)]  # (the twin's is not compared)
            for path, o in zip((a, b), outs):
                path.run_layer(l, *x, o)
            start = 0
            for i, (s, n) in enumerate(rows):
                r = b.rows[i]
                lo = r.position + n - r.local
                ring = []
                for P in (ref, pool):
                    for kind in (0, 1):
                        whole = _tokens(P.pool, P.ring_table[l, s], kind, 0, P.ring_tokens)
                        ring.append(whole[:, [t % P.ring_tokens for t in range(lo, r.position + n)]])
                assert torch.equal(ring[0], ring[2]) and torch.equal(ring[1], ring[3])
                hist = (torch.zeros(Hkv, 0, 128),) * 2
                if r.older:
                    W = -(-r.older // 32)
                    new = ops.PagedKV8.zeros(W, Hkv, DEV)
                    own = torch.arange(W, dtype=torch.int32, device=DEV)[None]
                    ops.kv8_quantize(ref.pool, new, src_table=ref.src_table[s:s + 1, :W], dst_table=own, tokens=r.older)
                    hist = ops.kv8_unpack(new, own, 0, r.older)
                    got = ops.kv8_unpack(pool.shared, pool.src_table[s:s + 1], 0, r.older)
                    assert torch.equal(hist[0], got[0]) and torch.equal(hist[1], got[1]), (step, s)
                    hist = (hist[0][0].cpu(), hist[1][0].cpu())
                if step % 5 == 0 or r.older == 0:
                    vs, os = b.layer_params[l][3].cpu(), None
                    v = hist[1]
                    if contract == "hf":
                        v = (v.float() * vs[:, None, None]).bfloat16()
                    else:
                        os = vs.repeat_interleave(Hq // Hkv).double()[None, :, None]
                    q = b._q_out.reshape(-1, Hq, 128)[start:start + n].cpu()
                    k = torch.cat((hist[0], ring[2].cpu()), 1)
                    want, mean, err, _ = attention64(q, k, torch.cat((v, ring[3].cpu()), 1), n)
                    o = outs[1][start:start + n]
                    if os is None:
                        check(o, want, mean, err, 2.0 ** -10, (step, l, s))
                    else:  # two roundings: the output's, and its product's with the scale
                        off = (o.double().cpu() - want * os).abs()
                        assert bool((off <= os.abs() * (want.abs() * 2.0 ** -7 * 1.01 + mean * (2 * err + 2.0 ** -10))).all())
                start += n
        for s in [s for s in live if a.seen(s) >= cap or rng.random() < 0.02]:
            for path in (a, b):
                path.free_sequence(s)
            live.remove(s)
    for s in live:
        for path in (a, b):
            path.free_sequence(s)
    assert pool.free_pages == free


def _prefill(runner, ids, slot=None):
    slot = runner.add_sequence() if slot is None else slot
    C, fed = runner.config.chunk_size, 0
    while fed < ids.numel():
        take = min(ids.numel() - fed, C - runner.fast.seen(slot) % C)
        logits = runner.step([(slot, ids[fed:fed + take])])
        fed += take
    return slot, logits


def _ids(seed, n):
    return torch.randint(3, 97, (n,), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("shared_cache", ["bf16", "kv8"])
def test_a_fork_continues_as_its_parent(shared_cache):
    """Two sequences of one prompt, the second forked from the first or prefilled by itself: the same logits at every step, with
    the same and with other tokens."""

    _, model = _tiny(chunk=24)
    made = []
    for fork in (True, False):
        r = LastKVServingModel(model, max_batch=4, max_tokens_per_slot=256, num_splits=2, shared_cache=shared_cache)
        s0, _ = _prefill(r, _ids(1, 101))
        s1 = r.fork_sequence(s0) if fork else _prefill(r, _ids(1, 101))[0]
        made.append((r, s0, s1))
    tok = _ids(2, 400).view(200, 2)
    for t in range(70):
        rows = [tok[t, 0:1], tok[t, 0:1] if t < 3 else tok[t, 1:2]]
        a, b = (r.step([(s0, rows[0]), (s1, rows[1])]) for r, s0, s1 in made)
        assert torch.equal(a, b), t
        if t < 3:
            assert torch.equal(a[0], a[1])
    (r, s0, s1), _ = made
    used = int(r.pool.pages.used[s1])
    r.free_sequence(s0)
    assert int((r.pool.pages.refs > 0).sum()) == used  # the fork keeps the pages that it shared
    r.free_sequence(s1)
    assert r.pool.free_pages == r.pool.source_pages


@pytest.mark.parametrize("shared_cache", ["bf16", "kv8"])
def test_compaction_changes_no_logits(shared_cache):
    _, model = _tiny(chunk=16)
    runners = [LastKVServingModel(model, max_batch=5, max_tokens_per_slot=192, num_splits=2, shared_cache=shared_cache)
               for _ in range(2)]
    slots = []
    for r in runners:
        s = [_prefill(r, _ids(i, 40 + 13 * i))[0] for i in range(4)]
        s.append(r.fork_sequence(s[2]))
        for k in (0, 1):
            r.free_sequence(s[k])
        slots.append(s[2:])
    assert runners[0].pool.compact() > 0 and runners[0].pool.compact() == 0
    P = runners[0].pool
    order = list(dict.fromkeys(int(p) for s in range(P.max_slots) for p in P.pages.table[s, :P.pages.used[s]]))
    assert order == list(range(len(order)))
    tok = _ids(9, 90).view(30, 3)
    for t in range(30):
        a, b = (r.step([(x, tok[t, i:i + 1]) for i, x in enumerate(s)]) for r, s in zip(runners, slots))
        assert torch.equal(a, b)


@pytest.mark.parametrize("contract", ["hf", "vllm"])
def test_decode_graph_over_8_bits_equals_eager_steps(contract):
    _, model = _tiny(chunk=16)
    runners = [LastKVServingModel(model, max_batch=3, max_tokens_per_slot=256, num_splits=3, contract=contract, shared_cache="kv8")
               for _ in range(2)]
    slots = [[_prefill(r, _ids(i, 50 + 9 * i))[0] for i in range(3)] for r in runners]
    graph = runners[0].decode_graph(slots[0], num_splits=3)
    tok = _ids(5, 180).view(60, 3)
    for t in range(60):
        got, _ = graph.step(tok[t].to(DEV))
        want = runners[1].step([(s, tok[t, i:i + 1]) for i, s in enumerate(slots[1])])
        torch.cuda.synchronize()
        assert torch.equal(got, want), t
        if t == 30:
            runners[0].pool.compact()


def test_serving_options_are_checked():
    _, model = _tiny()
    with pytest.raises(ValueError, match="shared_cache"):
        LastKVServingModel(model, max_batch=2, max_tokens_per_slot=64, shared_cache="fp8")
    r = LastKVServingModel(model, max_batch=2, max_tokens_per_slot=64)
    with pytest.raises(ValueError, match="not in use"):
        r.fork_sequence(0)
    a, b = r.add_sequence(), r.add_sequence()
    with pytest.raises(RuntimeError, match="slot"):
        r.fork_sequence(a)
    for s in (a, b):
        r.free_sequence(s)
    p = _ids(1, 5)
    for kw in (dict(num_beams=0, max_new_tokens=3), dict(num_beams=65, max_new_tokens=3), dict(num_beams=2, max_new_tokens=0),
               dict(num_beams=3, max_new_tokens=2), dict(num_beams=33, max_new_tokens=2, eos_token_id=1)):
        with pytest.raises(ValueError):
            r.beam_search([p], **kw)
    with pytest.raises(ValueError):
        r.beam_search([p[:0]], num_beams=1, max_new_tokens=2)
    assert r.pool.free_pages == r.pool.source_pages and not r.fast._open.any()


def _reference_beams(model, prompt, K, steps, eos, penalty, shared_cache):
    """The search with every beam's sequence fed again from its prompt at every step, selections in 64 bits."""

    def fresh():
        return LastKVServingModel(model, max_batch=K, max_tokens_per_slot=256, num_splits=2, shared_cache=shared_cache)

    new, scores, done = [[]], [0.0], []
    count = K if eos is None else 2 * K
    for t in range(steps):
        r = fresh()
        if t == 0:
            logits = _prefill(r, prompt)[1]
        else:
            slots = [_prefill(r, prompt)[0] for _ in range(K)]
            for j in range(t):
                logits = r.step([(s, torch.tensor([ids[j]])) for s, ids in zip(slots, new)])
        total = torch.tensor(scores, dtype=torch.float32).double()[:, None] + torch.log_softmax(logits.double().cpu(), -1)
        best, index = torch.sort(total.flatten(), descending=True, stable=True)
        V = logits.shape[-1]
        kids = []
        for rank in range(count):
            k, tok, sc = int(index[rank]) // V, int(index[rank]) % V, float(best[rank].float())
            if tok == eos:
                if rank < K:
                    done.append((sc, new[k] + [tok]))
            elif len(kids) < K:
                kids.append((sc, k, tok))
        if len(done) >= K or t + 1 == steps:
            if len(done) < K:
                done += [(sc, new[k] + [tok]) for sc, k, tok in kids]
            break
        new, scores = [new[k] + [tok] for _, k, tok in kids], [sc for sc, _, _ in kids]
    return sorted(((s / len(x) ** penalty, x) for s, x in done), key=lambda h: -h[0])[:K]


@pytest.mark.parametrize("shared_cache", ["bf16", "kv8"])
@pytest.mark.parametrize("K,eos,penalty", [(1, None, 1.0), (3, None, 1.0), (4, 11, 0.7)])
def test_beam_search_against_sequences_fed_from_the_start(K, eos, penalty, shared_cache):
    """Forked beams over copied pages give the ids of beams that are fed whole every time, across chunk boundaries."""

    _, model = _tiny(chunk=8, seed=23)
    if eos is not None:  # a token that beams do choose
        with torch.no_grad():
            model.lm_head.weight[eos] = model.lm_head.weight[[5, 17, 40]].mean(0) * 2.5
    r = LastKVServingModel(model, max_batch=K, max_tokens_per_slot=256, num_splits=2, shared_cache=shared_cache)
    prompt = _ids(3, 21)
    got = r.beam_search([prompt], num_beams=K, max_new_tokens=14, eos_token_id=eos, length_penalty=penalty)[0]
    want = _reference_beams(model, prompt, K, 14, eos, penalty, shared_cache)
    assert [ids[21:].tolist() for ids, _ in got] == [x for _, x in want]
    # 14 steps' scores, each rounded to fp32 (below 128: 2^-18 apart) from sums with errors of 40 * 2^-24
    assert all(abs(s - w) <= 14 * (2.0 ** -18 + 40 * 2.0 ** -24) for (_, s), (w, _) in zip(got, want))
    assert all(torch.equal(ids[:21], prompt) for ids, _ in got)
    assert r.pool.free_pages == r.pool.source_pages and not r.fast._open.any()


def test_beam_search_of_one_beam_is_greedy_and_prompts_share_steps():
    _, model = _tiny(chunk=8)
    r = LastKVServingModel(model, max_batch=6, max_tokens_per_slot=128, num_splits=2)
    prompts = [_ids(4, 9), _ids(5, 17)]
    greedy = r.generate(prompts, 12)
    one = r.beam_search(prompts, num_beams=1, max_new_tokens=12)
    assert all(torch.equal(g, h[0][0]) for g, h in zip(greedy, one))
    both = r.beam_search(prompts, num_beams=3, max_new_tokens=12)
    for hyps, p in zip(both, prompts):
        assert len(hyps) == 3 and all(ids.numel() == p.numel() + 12 for ids, _ in hyps)
        assert [s for _, s in hyps] == sorted((s for _, s in hyps), reverse=True)
        assert len({tuple(ids.tolist()) for ids, _ in hyps}) == 3
    assert r.pool.free_pages == r.pool.source_pages


@pytest.mark.parametrize("shared_cache", ["bf16", "kv8"])
@pytest.mark.parametrize("contract", ["hf", "vllm"])
def test_forks_at_and_around_boundaries(shared_cache, contract):
    """Forks of prompts that end before, at and behind a chunk's or page's end, and forks of forks, beside sequences prefilled by
    themselves; then a captured step over all of them."""

    _, model = _tiny(chunk=24)
    lengths = [1, 23, 24, 25, 31, 32, 48, 72, 96, 97]
    logits = []
    for fork in (True, False):
        r = LastKVServingModel(model, max_batch=3, max_tokens_per_slot=256, num_splits=2, shared_cache=shared_cache, contract=contract)
        seen = []
        for n in lengths:
            ids = _ids(n, n)
            s = [_prefill(r, ids)[0]]
            for i in range(2):
                s.append(r.fork_sequence(s[i]) if fork else _prefill(r, ids)[0])
            tok = _ids(n + 1, 60 * 3).view(60, 3)
            for t in range(50):
                seen.append(r.step([(x, tok[t, i:i + 1]) for i, x in enumerate(s)]).clone())
            graph = r.decode_graph(s, num_splits=2)
            for t in range(50, 60):
                seen.append(graph.step(tok[t].to(DEV))[0].clone())
            torch.cuda.synchronize()
            del graph
            for x in s:
                r.free_sequence(x)
        assert r.pool.free_pages == r.pool.source_pages
        logits.append(seen)
    for t, (a, b) in enumerate(zip(*logits)):
        assert torch.equal(a, b), (lengths[t // 60], t % 60)


def test_fork_of_an_empty_sequence():
    _, model = _tiny(chunk=24)
    r = LastKVServingModel(model, max_batch=2, max_tokens_per_slot=128, shared_cache="kv8")
    a = r.add_sequence()
    b = r.fork_sequence(a)
    tok = _ids(3, 60)
    for t in range(60):
        got = r.step([(a, tok[t:t + 1]), (b, tok[t:t + 1])])
        assert torch.equal(got[0], got[1])


@pytest.mark.parametrize("contract", ["hf", "vllm"])
def test_the_runtime_self_check_covers_8_bits(contract, monkeypatch, capsys):
    """Every layer's call next to its two passes (history alone, ring alone, merged): each of the passes, their merge and the call
    round to bf16, 2^-8 of a value each, and the vLLM contract rounds the first three twice."""

    monkeypatch.setenv("LASTKV_MERGED_CHECK", "1")
    _, model = _tiny(chunk=24)
    r = LastKVServingModel(model, max_batch=2, max_tokens_per_slot=256, contract=contract, shared_cache="kv8")
    slots = [_prefill(r, _ids(i, 75 + 40 * i))[0] for i in range(2)]
    for t in range(3):
        r.step([(slots[0], _ids(t, 1)), (slots[1], _ids(t + 9, 1 + 3 * (t == 1)))])
    lines = [line for line in capsys.readouterr().out.splitlines() if "lastkv_merged_check" in line]
    rels = [float(line.split("'rel': ")[1].split(",")[0]) for line in lines]
    assert len(rels) > 20 and any("'older': [48" in line for line in lines) and max(rels) <= 7 * 2.0 ** -8
