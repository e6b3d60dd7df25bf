"""The low-bit operators through the framework's own paths: the serving model over 4-bit weights, the native launch
path against the Python bodies, the custom operators against the plain calls."""

from __future__ import annotations

import pytest
import torch

from lastkv_amd import ops
from lastkv_amd import torch_ops as L
from lastkv_amd.serving import LastKVServingModel

from test_gpu_host_path import _both, _randn
from test_gpu_llm import _no_worse_than_reference_bf16, _o16, _o32, _tiny
from test_gpu_mx import random_mx4, random_mx8

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _prefill(runner, slots, prompts, chunk):
    nxt = []
    for slot, p in zip(slots, prompts):
        fed = 0
        while fed < p.numel():
            take = min(p.numel() - fed, chunk - runner.fast.seen(slot) % chunk)
            logits = runner.step([(slot, p[fed:fed + take])])
            fed += take
        nxt.append(logits[0].argmax())
    return torch.stack(nxt)


def _quantized_oracle(oracle):
    """The oracle with its layers' projections at the values of their 4-bit weights (exact in bf16)."""

    with torch.no_grad():
        for layer in oracle.model.layers:
            a, m = layer.self_attn, layer.mlp
            for lin in (a.q_proj, a.k_proj, a.v_proj, a.o_proj, m.gate_proj, m.up_proj, m.down_proj):
                lin.weight.copy_(ops.mx4_unpack(ops.mx4_quantize(lin.weight)))
    return oracle


def test_serving_over_4_bit_weights_matches_the_oracle_with_their_values():
    """Ragged continuous batching, bf16 activations: no further from the fp32-attention oracle on the same weights than
    the reference's own bf16 path is."""

    oracle, ours = _tiny(chunk=8)
    runner = LastKVServingModel(ours, max_batch=3, max_tokens_per_slot=64, num_splits=1, weights="mxfp4")
    seqs = [torch.randint(3, 97, (n,), generator=torch.Generator().manual_seed(n)).to(DEV) for n in (37, 29, 41)]
    slots = [runner.add_sequence() for _ in seqs]
    fed, got = [0] * 3, [[] for _ in seqs]
    with torch.inference_mode():
        step = 0
        while any(f < len(s) for f, s in zip(fed, seqs)):
            rows, owners = [], []
            for i, s in enumerate(seqs):
                if fed[i] >= len(s):
                    continue
                take = min(len(s) - fed[i], 8 - runner.fast.seen(slots[i]) % 8, (5, 3, 8, 1)[(step + i) % 4])
                rows.append((slots[i], s[fed[i]:fed[i] + take]))
                owners.append((i, fed[i] + take - 1))
                fed[i] += take
            for (i, pos), row in zip(owners, runner.step(rows)):
                got[i].append((pos, row.float()))
            step += 1
        _quantized_oracle(oracle)
        for i, s in enumerate(seqs):
            pos = [p for p, _ in got[i]]
            want, _ = _o32(oracle)(s[None])
            ref16, _ = _o16(oracle)(s[None])
            _no_worse_than_reference_bf16(torch.stack([r for _, r in got[i]])[None], want[:, pos].float(),
                                          ref16[:, pos].float(), f"mxfp4 sequence {i}")


def test_8_bit_activations_are_the_values_of_their_rows(monkeypatch):
    """Few rows: products of MX8 rows are exact, so a step equals one whose norms and SwiGLU hand over their rows'
    values in bf16, bit for bit."""

    _, ours = _tiny(chunk=8)
    prompts = [torch.arange(3, 14, device=DEV), torch.tensor([1, 5, 17, 33, 2], device=DEV)]
    logits = []
    norm, silu = ops.rmsnorm_mx8, ops.silu_mul_mx8
    for unpacked in (False, True):
        if unpacked:
            monkeypatch.setattr(ops, "rmsnorm_mx8", lambda *a, **k: ops.mx8_unpack(norm(*a, **k)))
            monkeypatch.setattr(ops, "silu_mul_mx8", lambda *a, **k: ops.mx8_unpack(silu(*a, **k)))
        runner = LastKVServingModel(ours, max_batch=2, max_tokens_per_slot=64, num_splits=1, weights="mxfp4", activations="mxfp8")
        slots = [runner.add_sequence() for _ in prompts]
        with torch.inference_mode():
            out = [_prefill(runner, slots, prompts, 8).float()]
            for i in range(6):
                out.append(runner.step([(s, torch.tensor([7 + i], device=DEV)) for s in slots]))
        logits.append(out)
    for a, b in zip(*logits):
        assert torch.equal(a, b)


@pytest.mark.parametrize("contract", ["hf", "vllm"])
@pytest.mark.parametrize("activations", ["bf16", "mxfp8"])
def test_graph_replays_equal_eager_steps(activations, contract):
    _, ours = _tiny(chunk=8)
    make = lambda: LastKVServingModel(ours, max_batch=3, max_tokens_per_slot=96, num_splits=2, weights="mxfp4",
                                      activations=activations, contract=contract)
    eager, graphed = make(), make()
    prompts = [torch.arange(3, 14, device=DEV), torch.tensor([1, 5, 17, 33, 2], device=DEV), torch.arange(40, 61, device=DEV)]
    se, sg = [eager.add_sequence() for _ in prompts], [graphed.add_sequence() for _ in prompts]
    with torch.inference_mode():
        te, tg = _prefill(eager, se, prompts, 8), _prefill(graphed, sg, prompts, 8)
        assert torch.equal(te, tg)
        graph = graphed.decode_graph(sg)
        scratch = torch.randn(256, 256, device=DEV)
        for i in range(20):
            le = eager.step([(s, te[j:j + 1]) for j, s in enumerate(se)])
            lg, ng = graph.step(tg)
            assert torch.equal(le, lg), i
            te, tg = le.argmax(-1), ng.clone()
            scratch = scratch @ scratch.T * 1e-3
            if i % 3 == 0:
                torch.cuda.synchronize()


def test_serving_options_are_checked():
    _, ours = _tiny(chunk=8)
    make = lambda **kw: LastKVServingModel(ours, max_batch=1, max_tokens_per_slot=32, **kw)
    for kw, text in ((dict(weights="int4"), "weights"), (dict(activations="fp8"), "activations"), (dict(activations="mxfp8"), "mxfp4")):
        with pytest.raises(ValueError, match=text):
            make(**kw)


def test_generate_with_4_bit_weights():
    _, ours = _tiny(chunk=8)
    prompts = [torch.arange(3, 14, device=DEV), torch.tensor([1, 5, 17], device=DEV)]
    outs = [LastKVServingModel(ours, max_batch=2, max_tokens_per_slot=64, num_splits=1, weights="mxfp4",
                               activations="mxfp8").generate(prompts, 6, prefill_chunk=n) for n in (8, 8)]
    for a, b, p in zip(*outs, prompts):
        assert torch.equal(a, b) and a.numel() == p.numel() + 6


# ------------------------------------------------------------------------------------------ native launch path
def _rows8(seed, rows, width):
    return random_mx8(torch.Generator(device=DEV).manual_seed(seed), rows, width)


def _weight(seed, n, k):
    return ops.mx4_pack(*random_mx4(torch.Generator(device=DEV).manual_seed(seed), n, k))


def _parts(r):
    return [r.data.view(torch.uint8), r.scales]


@pytest.mark.parametrize("shape", [(5, 64), (2, 3, 96), (1, 1, 2080), (1, 7, 32)])
def test_native_path_makes_the_same_calls(monkeypatch, shape):
    def norm():
        x, r, w = _randn(1, *shape), _randn(2, *shape), _randn(3, shape[-1])
        out = ops.MX8Rows.empty(shape, DEV)
        assert ops.rmsnorm_mx8(x, w, 1e-5, out=out) is out
        return [*_parts(ops.rmsnorm_mx8(x, w, 1e-5, residual=r)), r, *_parts(out)]

    def silu():
        both = _randn(4, *shape[:-1], 2 * shape[-1])
        q = ops.silu_mul_mx8(both[..., :shape[-1]], both[..., shape[-1]:])
        assert isinstance(q, ops.MX8Rows) and q.shape == shape
        return [*_parts(q), ops.mx8_unpack(q)]

    def linear():
        x, w, b = _randn(5, *shape), _weight(6, 40, shape[-1]), _randn(7, 40)
        q = ops.rmsnorm_mx8(x, _randn(3, shape[-1]), 1e-5)
        out = torch.zeros((*shape[:-1], 40), device=DEV, dtype=BF16)
        assert ops.mx4_linear(x, w, out=out) is out
        return [ops.mx4_linear(x, w, b), out, ops.mx4_linear(q, w), ops.mx4_linear(q, w, bias=b)]

    for make in (norm, silu, linear):
        _both(monkeypatch, make)


def test_native_path_leaves_other_forms_to_python(monkeypatch):
    """Rows of one dim, four dims, no rows: the Python bodies take them."""

    def make():
        x, w, n = _randn(1, 64), _weight(2, 16, 64), _randn(3, 64)
        q = ops.rmsnorm_mx8(x, n, 1e-5)
        x4 = _randn(4, 2, 1, 2, 64)
        return [*_parts(q), ops.mx4_linear(q, w), ops.mx4_linear(x, w), ops.mx4_linear(x4, w), ops.mx8_unpack(q),
                ops.mx4_linear(x4[:0], w), *_parts(ops.silu_mul_mx8(x, x)), *_parts(ops.silu_mul_mx8(x4, x4))]

    results = []
    for host in (ops._host, None):
        monkeypatch.setattr(ops, "_host", host)
        monkeypatch.setattr(ops, "_host_bound", host is not None)
        results.append(make())
    for a, b in zip(*results):
        assert a.shape == b.shape and torch.equal(a, b)


def test_refusals_on_the_gpu():
    """Shapes, types, alignment and overlaps that either launch path must refuse (nothing is launched)."""

    x, w, n = _randn(1, 4, 64), _weight(2, 16, 64), _randn(3, 64)
    q = _rows8(4, 4, 64)
    wide = _randn(5, 4, 80)
    over = ops.MX8Rows(x.view(torch.float8_e4m3fn)[:, 64:], _rows8(1, 4, 64).scales)  # x's own bytes
    mixed, resized = _rows8(4, 4, 64), _weight(2, 16, 64)  # fields assigned later
    mixed.scales, resized.out_features = mixed.scales[:, :1], 160
    cases = [
        (lambda: ops.rmsnorm_mx8(wide[:, :40], _randn(6, 40), 1e-5), "32-value"),
        (lambda: ops.rmsnorm_mx8(x, n[:32], 1e-5), "weight"),
        (lambda: ops.rmsnorm_mx8(x, n, 1e-5, residual=x[:2]), "residual"),
        (lambda: ops.rmsnorm_mx8(x, n, 1e-5, out=_rows8(1, 3, 64)), "out shape"),
        (lambda: ops.rmsnorm_mx8(x.float(), n, 1e-5), "bfloat16"),
        (lambda: ops.rmsnorm_mx8(_randn(7, 4, 128)[:, ::2], n, 1e-5), "contiguous"),
        (lambda: ops.silu_mul_mx8(x, x[:, :32]), "up shape"),
        (lambda: ops.silu_mul_mx8(x, x, out=over), "overlap"),
        (lambda: ops.rmsnorm_mx8(x, n, 1e-5, out=over), "overlap"),
        (lambda: ops.rmsnorm_mx8(x[:3], n, 1e-5, residual=x[1:]), "overlap"),
        (lambda: ops.mx8_unpack(mixed), "scales"),
        (lambda: ops.mx4_linear(mixed, w), "scales"),
        (lambda: ops.mx4_linear(x, resized), "bytes"),
        (lambda: ops.mx4_unpack(resized), "bytes"),
        (lambda: ops.MX8Rows(q.data, q.scales[:, :1]), "scales"),
        (lambda: ops.MX8Rows(q.data.view(torch.uint8), q.scales), "float8_e4m3fn"),
        (lambda: ops.MX4Weight(w.data[:-1], 16, 64), "bytes"),
        (lambda: ops.MX4Weight(w.data, 16, 40), "multiple of 32"),
        (lambda: ops.mx4_linear(wide, w), "x must be"),
        (lambda: ops.mx4_linear(x, w, bias=n[:15]), "bias"),
        (lambda: ops.mx4_linear(x, w, out=torch.zeros((4, 17), device=DEV, dtype=BF16)), "out must be"),
        (lambda: ops.mx4_linear(x, _weight(8, 64, 64), out=x), "overlap"),
        (lambda: ops.mx4_linear(wide[:, :64], _weight(8, 16, 64), out=wide[:, 64:]), "overlap"),
        (lambda: ops.mx4_quantize(x.t()), "contiguous rows"),
        (lambda: ops.mx4_quantize(x[:, :40]), "multiple of 32"),
        (lambda: ops.mx4_pack(q.scales, q.scales), "multiple of 32"),
    ]
    for call, text in cases:
        with pytest.raises(ValueError, match=text):
            call()
    from lastkv_amd import _lib
    with pytest.raises(_lib.LastKVNativeError, match="overlap"):
        ops.mx4_linear(x, w, out=torch.zeros(16, device=DEV, dtype=BF16).expand(4, 16))
    odd = torch.zeros(4 * 64 + 4, device=DEV, dtype=BF16)[4:].view(4, 64)  # 8 bytes past a 16-byte border
    for call in (lambda: ops.rmsnorm_mx8(odd, n, 1e-5), lambda: ops.silu_mul_mx8(odd, odd), lambda: ops.mx4_linear(odd, w)):
        with pytest.raises(_lib.LastKVNativeError, match="aligned"):
            call()


# ------------------------------------------------------------------------------------------ custom operators
def test_custom_operators_equal_the_plain_calls():
    x, r, n, w, b = _randn(1, 5, 64), _randn(2, 5, 64), _randn(3, 64), _weight(4, 40, 64), _randn(5, 40)
    q = ops.rmsnorm_mx8(x, n, 1e-5)
    for got, want in ((L.rmsnorm_mx8(x, n, 1e-5), q), (L.silu_mul_mx8(x, r), ops.silu_mul_mx8(x, r))):
        assert torch.equal(got[0].view(torch.uint8), want.data.view(torch.uint8)) and torch.equal(got[1], want.scales)
    r1, r2 = r.clone(), r.clone()
    got, want = L.add_rmsnorm_mx8(x, r1, n, 1e-5), ops.rmsnorm_mx8(x, n, 1e-5, residual=r2)
    assert torch.equal(r1, r2) and torch.equal(got[0].view(torch.uint8), want.data.view(torch.uint8))
    assert torch.equal(L.mx8_unpack(q.data, q.scales), ops.mx8_unpack(q))
    assert torch.equal(L.mx4_linear(x, w.data, 40, b), ops.mx4_linear(x, w, b))
    assert torch.equal(L.mx4_linear_mx8(q.data, q.scales, w.data, 40), ops.mx4_linear(q, w))
    torch.library.opcheck(L.mx4_linear, (x, w.data, 40, b))
