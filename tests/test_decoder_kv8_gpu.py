"""``QuadDecoder`` over 8-bit caches: steps, evictions, capture and scoring.

Tolerance of a step's logits against the float32 restatement (max norm, per
model): 2e-2 for the FP16 activations, as for the decoder with FP16 caches;
plus, for each of the two layers, 1/254 (a stored value is off by at most half
a step, 1/254 of its block's largest) once for the values and once for what
the keys' errors move in the weights: 2e-2 + 4/254.
"""
from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

from test_decoder_gpu import _linear_weights, _ref_step, packed  # noqa: F401  (packed is a fixture)

pytestmark = pytest.mark.gpu
TOL = 2e-2 + 4 / 254


@pytest.fixture(scope="module")
def parts(cuda, packed):  # noqa: F811
    from polar_pack_b200.decoder import DecoderExtras
    from polar_pack_b200.quadpack import QuadPackDevice, QuadPackFile
    cfg, buf, restored = packed
    cfg = dataclasses.replace(cfg, max_pos=300)
    return cfg, QuadPackDevice(QuadPackFile(buf), cuda), DecoderExtras.random(cfg, cuda, seed=1), restored


def _decoder(parts, **kw):
    from polar_pack_b200.decoder import QuadDecoder
    cfg, pk, ex, _ = parts
    return QuadDecoder(pk, cfg, ex, kv_bits=8, **kw)


def _tokens(cfg, n, seed=3):
    return np.random.default_rng(seed).integers(0, cfg.vocab, (n, 4))


def test_steps_match_float32_reference(cuda, parts):
    cfg, _, ex, restored = parts
    dec = _decoder(parts)
    k = 2
    W = {n: t.to(cuda) for n, t in _linear_weights(cfg, restored, k).items()}
    e = dict(embed=ex.embed[k].float(), in_norm=ex.in_norm[:, k].float(), post_norm=ex.post_norm[:, k].float(),
             final=ex.final_norm[k].float(), bias=ex.qkv_bias[:, k].float())
    cache = [([], []) for _ in range(cfg.layers)]
    for pos, toks in enumerate(_tokens(cfg, 140)):
        got = dec.step(toks)[k].float()
        ref = _ref_step(cfg, W, e, cache, pos, int(toks[k]))
        assert float((got - ref).abs().max() / ref.abs().max()) <= TOL, pos
    assert int(dec.status.item()) == 0


def test_all_models_match_the_fp16_caches(cuda, parts):
    from polar_pack_b200.decoder import QuadDecoder
    cfg, pk, ex, _ = parts
    a, b, c = _decoder(parts), _decoder(parts, kv_budget=200, kv_slack=50), QuadDecoder(pk, cfg, ex)
    for pos, toks in enumerate(_tokens(cfg, 150, 4)):
        x, y, z = (d.step(toks).float() for d in (a, b, c))
        worst = z.abs().amax(1)
        # both sides round their activations
        assert bool(((x - z).abs().amax(1) <= (TOL + 2e-2) * worst).all()), pos
        assert bool(((y - z).abs().amax(1) <= (TOL + 2e-2) * worst).all()), pos
    for layer in b.kv8_weights:   # 150 steps, each query head's weights sum to one
        want = 150.0 * (cfg.q_heads // cfg.kv_heads)
        assert torch.allclose(layer.sum(-1), torch.full_like(layer.sum(-1), want), rtol=1e-3)


def test_evictions_and_capture(cuda, parts):
    cfg = parts[0]
    toks = _tokens(cfg, 280, 5)
    eager = _decoder(parts, kv_budget=90, kv_slack=40, kv_recent=16, kv_sinks=3)
    got, held = [], []
    for t in toks:
        got.append(eager.step(t).clone())
        held.append(eager.n_held)
    assert max(held) == 130 and held[130] == 91 and held[170] == 91
    assert eager.held.tolist() == [held[-1]] * 4 and eager.pos.item() == 280 and int(eager.status.item()) == 0
    assert all(bool(torch.isfinite(x).all()) for x in got)
    graph = _decoder(parts, kv_budget=90, kv_slack=40, kv_recent=16, kv_sinks=3)
    for t in toks[:100]:
        graph.step(t)
    graph.capture(torch.cuda.Stream(cuda))
    assert graph.held.tolist() == [100] * 4 and graph.rot.tolist() == [100] * 4
    for t, want in zip(toks[100:], got[100:]):
        assert torch.equal(graph.step(t), want)
    graph.reset()
    assert torch.equal(graph.step(toks[0]), got[0])


def test_eviction_keeps_first_last_and_heaviest(cuda, parts):
    from polar_pack_b200.kv8 import kv8_restore
    cfg = parts[0]
    dec = _decoder(parts, kv_budget=70, kv_slack=60, kv_recent=20, kv_sinks=2)
    for t in _tokens(cfg, 120, 6):
        dec.step(t)
    before = [kv8_restore(c, dec.held, count=120) for c in dec.kv8]
    weights = [w.clone() for w in dec.kv8_weights]
    dec.evict()
    assert dec.n_held == 70 and dec.held.tolist() == [70] * 4 and dec.rot.tolist() == [120] * 4
    for c, (k0, v0), w0, w1 in zip(dec.kv8, before, weights, dec.kv8_weights):
        k1, v1 = kv8_restore(c, dec.held, count=70)
        for b in range(4):
            for h in range(cfg.kv_heads):
                mid = w0[b, h, 2:100].sort(descending=True, stable=True).indices[:48].sort().values + 2
                want = torch.cat([torch.arange(2, device=cuda), mid, torch.arange(100, 120, device=cuda)])
                assert torch.equal(w1[b, h, :70], w0[b, h, want]) and not w1[b, h, 70:].any()
                for x0, x1 in ((k0, k1), (v0, v1)):
                    x0, x1 = x0[b, want, h].float(), x1[b, :, h].float()
                    # the first block is coded again (half a step), the rest as it was, in FP16
                    step = x0[:64].abs().max() / 127
                    assert float((x0[:64] - x1[:64]).abs().max()) <= float(step) * 0.5 * 1.01 + 2 ** -11 * float(x0.abs().max())
                    assert torch.equal(x0[64:], x1[64:])


@pytest.mark.parametrize("bits", [8, 16])
def test_score_matches_step_by_step(cuda, parts, bits):
    from polar_pack_b200.decoder import QuadDecoder
    cfg, pk, ex, _ = parts
    toks = _tokens(cfg, 20, 7).T
    a = QuadDecoder(pk, cfg, ex, kv_bits=bits)
    s = a.score(toks)
    b = QuadDecoder(pk, cfg, ex, kv_bits=bits)
    for i in range(19):
        lp = torch.log_softmax(b.step(toks[:, i]).double(), -1)
        want = lp[torch.arange(4), torch.as_tensor(toks[:, i + 1], device=cuda)]
        # FP32 sums over 1000 logits: far below 1e-5 of the largest magnitude
        assert float((s[:, i].double() - want).abs().max()) <= 1e-5 * float(lp.abs().max())
        r = b.logprobs(toks[:, i + 1], top=4)
        assert torch.equal(r.logprob, s[:, i]) and torch.equal(r.top_ids.long(), b.logits.float().topk(4).indices) or \
            float((r.top_logprobs.double() - lp.topk(4).values).abs().max()) <= 1e-5 * float(lp.abs().max())


def test_refusals(cuda, parts):
    from polar_pack_b200.decoder import QuadDecoder
    cfg, pk, ex, _ = parts
    for kw in (dict(kv_bits=4), dict(kv_budget=100), dict(kv_bits=8, kv_budget=0), dict(kv_bits=8, kv_budget=64),
               dict(kv_bits=8, kv_budget=100, kv_slack=0), dict(kv_bits=8, kv_budget=100, kv_recent=-1)):
        with pytest.raises(ValueError):
            QuadDecoder(pk, cfg, ex, **kw)
    with pytest.raises(ValueError):
        QuadDecoder(pk, cfg, ex).evict()
    dec = _decoder(parts, kv_budget=80, kv_slack=10)
    with pytest.raises(ValueError):
        dec.score([1, 2, 3])
    for t in _tokens(cfg, 90, 8):
        dec.step(t)
    with pytest.raises(ValueError):
        dec.capture(torch.cuda.Stream(cuda))


def test_capture_behind_queued_steps(cuda, parts):
    """A capture directly behind steps that the GPU has not reached yet."""
    cfg = parts[0]
    a, b = (_decoder(parts, kv_budget=90, kv_slack=40, kv_recent=16, kv_sinks=3) for _ in "ab")
    toks = _tokens(cfg, 30, 10)
    for t in toks[:20]:
        a.step(t)
    weights = [w.clone() for w in a.kv8_weights]
    x = torch.randn(8192, 8192, device=cuda)
    s = torch.cuda.Stream(cuda)
    torch.cuda.synchronize()
    for _ in range(10):                      # some 100 ms
        x = torch.mm(x, x) * 1e-4
    for t in toks[:20]:
        b.step(t)
    b.capture(s)
    assert b.held.tolist() == [20] * 4 and b.rot.tolist() == [20] * 4 and b.pos.item() == 20
    for u, w in zip(weights, b.kv8_weights):
        assert torch.equal(u, w)
    for t in toks[20:]:
        assert torch.equal(a.step(t), b.step(t))
    assert int(b.status.item()) == 0


@pytest.mark.parametrize("held", [64, 128])
def test_capture_at_a_blocks_end(cuda, parts, held):
    """A capture leaves the rows of the last block, also where the step it
    warms up with would open the next one."""
    from polar_pack_b200.kv8 import kv8_restore
    cfg = parts[0]
    a, b = (_decoder(parts, kv_budget=40, kv_slack=150, kv_recent=8, kv_sinks=2) for _ in "ab")
    toks = _tokens(cfg, held + 10, 9)
    for t in toks[:held]:
        a.step(t)
        b.step(t)
    torch.cuda.synchronize()
    b.capture(torch.cuda.Stream(cuda))
    for x, y in zip(a.kv8, b.kv8):
        for u, w in zip(kv8_restore(x, a.held, count=held), kv8_restore(y, b.held, count=held)):
            assert torch.equal(u, w)
    a.evict()
    b.evict()
    for t in toks[held:]:
        assert torch.equal(a.step(t), b.step(t))
    assert int(b.status.item()) == 0


def test_launch_overlap(cuda, parts):
    """Steps, evictions, a replayed step and scores, each kernel started while
    the one before it runs: the same bits as one after another."""
    from polar_pack_b200 import _lib
    cfg = parts[0]
    toks = _tokens(cfg, 150, 11)
    runs = []
    old = _lib.set_launch_overlap(False)
    try:
        for on in (False, True):
            _lib.set_launch_overlap(on)
            dec = _decoder(parts, kv_budget=90, kv_slack=20, kv_recent=16, kv_sinks=3)
            got = []
            for t in toks[:100]:
                got.append(dec.step(t).clone())
                r = dec.logprobs(t, top=7)
                got += [r.logprob, r.entropy, r.top_ids, r.top_logprobs]
            got.append(dec.score(toks[100:].T))
            dec.capture(torch.cuda.Stream(cuda))
            got.append(dec.score(toks[100:130].T))
            got += [w.clone() for w in dec.kv8_weights]
            assert int(dec.status.item()) == 0
            runs.append(got)
    finally:
        _lib.set_launch_overlap(old)
    for a, b in zip(*runs):
        assert torch.equal(a, b)
