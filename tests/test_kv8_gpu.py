"""The 8-bit KV cache operators against the plain 64-bit restatement (kv8_ref).

Codes, scales, tails, kept positions and restored values follow from the
definition and must be equal.  Attention outputs are FP16: rounding the output
and the softmax weights costs at most 2^-11 max|v| each, so 1.5 * 2^-10 max|v|
bounds them.  Accumulated weights are FP32: a score of these inputs carries an
error below 1e-4 (128 products of size up to 30, each sum rounded at 2^-24), so
2e-4 relative and 1e-6 absolute bounds them.
"""
from __future__ import annotations

import pytest
import torch

import kv8_ref as kr

pytestmark = pytest.mark.gpu
OUT_TOL = 1.5 * 2.0 ** -10


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _rand(g, *shape, spread=0.6):
    return (torch.randn(*shape, generator=g, device=g.device) * spread).half()


def _gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _new(batch, heads, cap, hd, dev, stale=True):
    """An empty cache whose unused contents are what must never be read."""
    from polar_pack_b200.kv8 import KV8Cache
    c = KV8Cache.empty(batch, heads, cap, hd, dev)
    if stale:
        c.k_codes.fill_(255)
        c.v_codes.fill_(255)
        for t in (c.k_scales, c.v_scales):
            t.fill_(float("nan"))
        for t in (c.k_tail, c.v_tail):
            t.fill_(float("nan"))
    return c


def _fill(cache, ref, lens, g):
    from polar_pack_b200.kv8 import kv8_append
    n = max(lens)
    if n:
        k, v = (_rand(g, cache.batch, n, cache.kv_heads, cache.head_dim) for _ in "kv")
        kv8_append(cache, k, v, _ints([0] * cache.batch, cache.device), counts=_ints(lens, cache.device))
        ref.append(k, v, lens)


def _check_cache(cache, ref):
    for w, (codes, scales, tail) in enumerate(((cache.k_codes, cache.k_scales, cache.k_tail),
                                               (cache.v_codes, cache.v_scales, cache.v_tail))):
        codes, scales, tail = codes.cpu(), scales.cpu(), tail.cpu()
        for b, row in enumerate(ref.s[w]):
            for h, r in enumerate(row):
                for j, (c, s) in enumerate(zip(r.codes, r.scales)):
                    assert torch.equal(codes[b, h, 64 * j:64 * j + 64], c), (w, b, h, j)
                    assert scales[b, h, j] == s, (w, b, h, j)
                assert torch.equal(tail[b, h, :len(r.rows)].view(torch.int16), r.rows.view(torch.int16)), (w, b, h)


def _check_out(out, want, ref):
    vmax = max([float(c.values().abs().max()) for row in ref.s[1] for c in row if c.len] + [0.0])
    err = (out.cpu().double() - want).abs().max().item()
    assert torch.isfinite(out).all()
    assert err <= OUT_TOL * vmax, (err, vmax)


# ------------------------------------------------------------- writing ----
@pytest.mark.parametrize("hd,heads,pieces", [
    (128, 2, [[1], [63], [64], [65], [200]]),
    (64, 3, [[1, 62, 1, 1], [64, 64], [5, 130, 0, 61]]),
    (128, 1, [[63, 1, 1], [10, 100, 300], [0, 0, 129]]),
])
def test_append(cuda, hd, heads, pieces):
    """Tokens in pieces of any length: equal to token by token."""
    from polar_pack_b200.kv8 import kv8_append
    B, cap = len(pieces), 448
    g = _gen(cuda, hd + heads)
    cache, ref = _new(B, heads, cap, hd, cuda), kr.RefKV(B, heads, hd)
    for step in range(max(map(len, pieces))):
        counts = [p[step] if step < len(p) else 0 for p in pieces]
        n = max(counts) + 2                      # rows past the counts are not read
        # keys and values as views of one fused projection
        qkv = _rand(g, B, n, 4 + 2 * heads, hd)
        for b, c in enumerate(counts):
            qkv[b, c:] = float("nan")
        k, v = qkv[:, :, 4:4 + heads], qkv[:, :, 4 + heads:]
        kv8_append(cache, k, v, _ints(ref.lens(), cuda), counts=_ints(counts, cuda))
        ref.append(k, v, counts)
        _check_cache(cache, ref)
    assert int(cache.status) == 0


def test_append_not_finite_zero_and_unaligned(cuda):
    from polar_pack_b200.kv8 import kv8_append
    g = _gen(cuda, 5)
    k, v = (_rand(g, 1, 128, 1, 64) for _ in "kv")
    k[0, 3, 0, 5], k[0, 7, 0, 1], k[0, 9, 0, 2] = float("nan"), float("inf"), -float("inf")
    v[0, :64] = 0                                                # a block of zeros: scale 0
    k[0, 64:] *= 1e-7                                            # subnormal FP16
    cache, ref = _new(1, 1, 128, 64, cuda), kr.RefKV(1, 1, 64)
    odd = torch.zeros(128 * 64 + 3, dtype=torch.float16, device=cuda)[3:].view(1, 128, 1, 64)
    odd.copy_(v)                                                 # rows that are not 16-byte aligned
    kv8_append(cache, k, odd, _ints([0], cuda))
    ref.append(k, v, [128])
    _check_cache(cache, ref)
    assert (cache.v_codes[0, 0, :64] == 128).all() and cache.v_scales[0, 0, 0] == 0


def test_append_refused_sequences(cuda):
    """Past the capacity: status 5 and nothing written; negative position: unused."""
    from polar_pack_b200.kv8 import kv8_append
    g = _gen(cuda, 6)
    cache = _new(3, 2, 64, 128, cuda)
    before = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_tail, cache.v_tail)]
    k, v = (_rand(g, 3, 70, 2, 128) for _ in "kv")
    kv8_append(cache, k, v, _ints([-1, 0, 60], cuda), counts=_ints([5, 70, 5], cuda))
    assert int(cache.status) == 5
    for t, u in zip((cache.k_codes, cache.v_codes, cache.k_tail, cache.v_tail), before):
        assert torch.equal(t.view(torch.uint8), u.view(torch.uint8))


def test_rotation(cuda):
    """Keys rotated by append and decode, queries by attention: as rotated by hand."""
    from polar_pack_b200.kv8 import kv8_append, kv8_attention, kv8_decode
    g = _gen(cuda, 7)
    B, nkv, nq, hd, n = 2, 2, 6, 128, 5
    cos, sin = (torch.rand(200, hd, generator=g, device=cuda).half() for _ in "cs")
    at = [30, 100]
    rows = torch.tensor(at, device=cuda)[:, None] + torch.arange(n + 1, device=cuda)
    k, v, q = _rand(g, B, n + 1, nkv, hd), _rand(g, B, n + 1, nkv, hd), _rand(g, B, n + 1, nq, hd)
    c, s = cos[rows][:, :, None], sin[rows][:, :, None]
    kr_, qr = kr.rope_fp16(k, c, s), kr.rope_fp16(q, c, s)
    plain, turned = _new(B, nkv, 64, hd, cuda), _new(B, nkv, 64, hd, cuda)
    zero, lens = _ints([0, 0], cuda), _ints([n, n], cuda)
    kv8_append(plain, kr_[:, :n], v[:, :n], zero)
    kv8_append(turned, k[:, :n], v[:, :n], zero, rope=(cos, sin, _ints(at, cuda)))
    assert torch.equal(plain.k_tail[:, :, :n], turned.k_tail[:, :, :n])
    assert torch.equal(kv8_attention(qr[:, :n], plain, lens),
                       kv8_attention(q[:, :n], turned, lens, rope=(cos, sin, _ints(at, cuda))))
    last = _ints([a + n for a in at], cuda)
    assert torch.equal(kv8_decode(qr[:, n], kr_[:, n], v[:, n], plain, lens),
                       kv8_decode(q[:, n], k[:, n], v[:, n], turned, lens, rope=(cos, sin, last)))
    assert torch.equal(plain.k_tail[:, :, :n + 1], turned.k_tail[:, :, :n + 1])
    assert int(turned.status) == 0
    out = kv8_decode(q[:, n], k[:, n], v[:, n], turned, lens, rope=(cos, sin, _ints([200, 3], cuda)))
    assert int(turned.status) == 5 and not out[0].any() and out[1].any()


def test_restore(cuda):
    from polar_pack_b200.kv8 import kv8_restore
    g = _gen(cuda, 8)
    lens = [0, 1, 64, 65, 150]
    cache, ref = _new(5, 2, 192, 64, cuda), kr.RefKV(5, 2, 64)
    _fill(cache, ref, lens, g)
    start = [-3, 0, 60, 64, 149]
    k, v = kv8_restore(cache, _ints(lens, cuda), start=_ints(start, cuda), count=70)
    whole = kv8_restore(cache, _ints(lens, cuda))
    for w, got in enumerate((k.cpu(), v.cpu())):
        for b, l in enumerate(lens):
            for h in range(2):
                x = ref.s[w][b][h].restored()
                assert torch.equal(whole[w][b, :l, h].cpu(), x) and not whole[w][b, l:].any()
                for i in range(70):
                    t = start[b] + i
                    assert torch.equal(got[b, i, h], x[t] if 0 <= t < l else torch.zeros_like(got[b, i, h]))


# ----------------------------------------------------------- attention ----
HEADS = [(1, 1, 128), (7, 1, 128), (16, 2, 64), (16, 1, 128), (6, 3, 64), (18, 2, 128)]


@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("n,lens,counts", [
    (1, [1, 0, 64, 65, 300], [1, 1, 1, 1, 1]),
    (3, [3, 2, 66, 128, 191], [3, 3, 2, 0, 1]),       # row 1: its first query precedes the sequence
    (40, [40, 33, 129, 200, 0], [40, 33, 17, 40, 0]),
])
def test_attention(cuda, nq, nkv, hd, n, lens, counts):
    from polar_pack_b200.kv8 import kv8_attention
    g = _gen(cuda, nq * 100 + n)
    B = len(lens)
    cache, ref = _new(B, nkv, 320, hd, cuda), kr.RefKV(B, nkv, hd)
    _fill(cache, ref, lens, g)
    q = _rand(g, B, n, nq + 1, hd, spread=2.0)[:, :, 1:]         # a view
    for b, c in enumerate(counts):
        q[b, c:] = float("nan")                                  # rows that are not queries
    out = kv8_attention(q, cache, _ints(lens, cuda), counts=_ints(counts, cuda))
    want, _ = kr.attention(ref, torch.nan_to_num(q), counts)
    _check_out(out, want, ref)
    for b, (l, c) in enumerate(zip(lens, counts)):
        assert not out[b, c:].any() and not out[b, :max(0, c - l)].any()
    again = kv8_attention(q, cache, _ints(lens, cuda), counts=_ints(counts, cuda))
    assert torch.equal(out, again) and int(cache.status) == 0


@pytest.mark.parametrize("nq,nkv,hd,n", [(8, 1, 128, 300), (14, 2, 64, 257), (28, 4, 128, 130), (2, 2, 128, 129)])
def test_prompt(cuda, nq, nkv, hd, n):
    """Prompts of many rows, over what the cache holds already, ragged."""
    from polar_pack_b200.kv8 import kv8_attention
    g = _gen(cuda, n)
    lens, counts = [n, n + 200, 100], [n, n - 1, 100]
    cache, ref = _new(3, nkv, 512, hd, cuda), kr.RefKV(3, nkv, hd)
    _fill(cache, ref, lens, g)
    q = _rand(g, 3, n, nq, hd, spread=2.0)
    out = kv8_attention(q, cache, _ints(lens, cuda), counts=_ints(counts, cuda))
    want, _ = kr.attention(ref, q, counts)
    _check_out(out, want, ref)


@pytest.mark.parametrize("nq,nkv,hd,scale", [(8, 1, 128, None), (16, 1, 64, -0.3), (10, 2, 128, 0.0)])
def test_prompt_over_long_cache(cuda, nq, nkv, hd, scale):
    """Few rows over many positions (split along them), odd scales, rotated queries."""
    from polar_pack_b200.kv8 import kv8_attention
    g = _gen(cuda, nq)
    n, lens, counts = 20, [5000, 20, 1301, 3], [20, 20, 7, 0]
    cache, ref = _new(4, nkv, 5056, hd, cuda), kr.RefKV(4, nkv, hd)
    _fill(cache, ref, lens, g)
    q = _rand(g, 4, n, nq, hd, spread=2.0)
    cos, sin = (torch.rand(5000, hd, generator=g, device=cuda).half() for _ in "cs")
    at = [4980, 0, 9, 1]
    rows = (torch.tensor(at, device=cuda)[:, None] + torch.arange(n, device=cuda)).clamp(max=4999)
    turned = kr.rope_fp16(q, cos[rows][:, :, None], sin[rows][:, :, None])
    want, _ = kr.attention(ref, turned, counts, scale=scale)
    for _ in range(2):
        out = kv8_attention(q, cache, _ints(lens, cuda), counts=_ints(counts, cuda), scale=scale,
                            rope=(cos, sin, _ints(at, cuda)))
        _check_out(out, want, ref)
    assert int(cache.status) == 0


@pytest.mark.parametrize("nq,nkv,hd,n,lens,counts", [
    (4, 1, 128, 300, [6000, 300, 2500, 0], [300, 299, 10, 0]),      # split by the longest
    (16, 2, 64, 70, [3000, 9000], [70, 70]),
    (10, 2, 128, 60, [1, 60, 8100], [1, 60, 60]),
    (2, 2, 64, 257, [9001, 9000, 8999], [257, 256, 0]),
    (8, 1, 128, 90, [30000, 700, 2000], [0, 90, 90]),              # the longest has no queries
])
def test_split_positions(cuda, nq, nkv, hd, n, lens, counts):
    """Chunks of prompts over long caches, whose positions are split where that pays."""
    from polar_pack_b200.kv8 import kv8_attention
    g = _gen(cuda, n)
    B = len(lens)
    cap = -(-max(lens) // 64) * 64 + 64
    cache, ref = _new(B, nkv, cap, hd, cuda), kr.RefKV(B, nkv, hd)
    _fill(cache, ref, lens, g)
    q = _rand(g, B, n, nq, hd, spread=2.0)
    out = kv8_attention(q, cache, _ints(lens, cuda), counts=_ints(counts, cuda))
    want, _ = kr.attention(ref, q, counts)
    _check_out(out, want, ref)
    again = kv8_attention(q, cache, _ints(lens, cuda), counts=_ints(counts, cuda))
    assert torch.equal(out, again) and int(cache.status) == 0
    # lengths past the capacity: refused on the device, the others as before
    bad = list(lens)
    bad[0] = cap + 1
    out = kv8_attention(q, cache, _ints(bad, cuda), counts=_ints(counts, cuda))
    _check_out(out[1:], want[1:], ref)
    assert not out[0].any() and int(cache.status) == 5


@pytest.mark.parametrize("nq,nkv,hd,n", [(8, 1, 128, 3), (8, 1, 128, 17), (4, 2, 64, 100), (7, 1, 128, 36)])
def test_small_and_large_capacity(cuda, nq, nkv, hd, n):
    """17 to 256 rows per kv head: the capacity decides which kernel they run on; both are right."""
    from polar_pack_b200.kv8 import kv8_attention
    g = _gen(cuda, n)
    lens, counts = [n + 70, n, 400, 5], [n, n, min(n, 9), min(n, 5)]
    q = _rand(g, 4, n, nq, hd, spread=2.0)
    for cap in (448, 16384):
        cache, ref = _new(4, nkv, cap, hd, cuda), kr.RefKV(4, nkv, hd)
        _fill(cache, ref, lens, _gen(cuda, 50))
        out = kv8_attention(q, cache, _ints(lens, cuda), counts=_ints(counts, cuda))
        want, _ = kr.attention(ref, q, counts)
        _check_out(out, want, ref)
        assert int(cache.status) == 0


def test_prompt_rows_do_not_mix(cuda):
    """A query of NaN changes its own row only; value blocks of very different scale."""
    from polar_pack_b200.kv8 import kv8_append, kv8_attention
    g = _gen(cuda, 31)
    n, hd, nq = 200, 128, 2
    k, v, q = _rand(g, 1, n, 1, hd), _rand(g, 1, n, 1, hd), _rand(g, 1, n, nq, hd)
    v[0, :64] *= 1e-4
    v[0, 64:128] = 0
    cache, ref = _new(1, 1, 256, hd, cuda), kr.RefKV(1, 1, hd)
    kv8_append(cache, k, v, _ints([0], cuda))
    ref.append(k, v, [n])
    out = kv8_attention(q, cache, _ints([n], cuda))
    want, _ = kr.attention(ref, q, [n])
    vv = ref.s[1][0][0].values()
    # a row's weights are FP16 beside the largest scale of the block range: for the first rows, whose values
    # are 1e-4 of the last ones, their rounding is still relative (2^11 lifts them above FP16's smallest)
    for i in range(n):
        bound = OUT_TOL * float(vv[:i + 1].abs().max()) + 2.0 ** -24
        assert ((out[0, i].cpu().double() - want[0, i]).abs() <= bound).all(), i
    q[0, 77, 1] = float("nan")
    bad = kv8_attention(q, cache, _ints([n], cuda))
    same = torch.ones(n, nq, dtype=torch.bool, device=cuda)
    same[77, 1] = False
    assert torch.equal(bad[0][same], out[0][same]) and torch.isnan(bad[0, 77, 1]).all()


@pytest.mark.parametrize("nq,nkv,hd", [(16, 2, 128), (7, 1, 64), (16, 1, 128)])
def test_decode_steps(cuda, nq, nkv, hd):
    """Steps across a block's end: outputs, cache and accumulated weights."""
    from polar_pack_b200.kv8 import kv8_decode
    g = _gen(cuda, nq)
    lens = [0, 62, 126, 190]
    B = len(lens)
    cache, ref = _new(B, nkv, 256, hd, cuda), kr.RefKV(B, nkv, hd)
    _fill(cache, ref, lens, g)
    weights = cache.new_weights()
    total = torch.zeros(B, nkv, 256, dtype=torch.float64)
    for step in range(5):
        q, k, v = _rand(g, B, nq, hd, spread=2.0), _rand(g, B, nkv, hd), _rand(g, B, nkv, hd)
        out = kv8_decode(q, k, v, cache, _ints(ref.lens(), cuda), weights=weights)
        ref.append(k[:, None], v[:, None], [1] * B)
        want, probs = kr.attention(ref, q[:, None], [1] * B)
        _check_out(out, want[:, 0], ref)
        for b in range(B):
            for h in range(nkv):
                total[b, h, :len(probs[b][h])] += probs[b][h]
    _check_cache(cache, ref)
    assert ((weights.cpu().double() - total).abs() <= 2e-4 * total + 1e-6).all()
    assert int(cache.status) == 0


def test_decode_unused_and_full(cuda):
    from polar_pack_b200.kv8 import kv8_decode
    g = _gen(cuda, 11)
    cache, ref = _new(3, 1, 64, 128, cuda), kr.RefKV(3, 1, 128)
    _fill(cache, ref, [10, 10, 64], g)
    w = cache.new_weights()
    q, k, v = _rand(g, 3, 4, 128), _rand(g, 3, 1, 128), _rand(g, 3, 1, 128)
    out = kv8_decode(q, k, v, cache, _ints([-1, 10, 64], cuda), weights=w)
    assert not out[0].any() and out[1].any() and not out[2].any()
    assert int(cache.status) == 5 and not w[0].any() and not w[2].any() and w[1].any()
    ref.append(k[:, None], v[:, None], [0, 1, 0])
    _check_cache(cache, ref)


@pytest.mark.parametrize("batch,lens", [(1, [20011]), (3, [9000, 31, 4096]), (70, None)])
def test_decode_long_and_many(cuda, batch, lens):
    """Long caches and many ragged sequences (the work is split over the GPU)."""
    from polar_pack_b200.kv8 import kv8_decode
    g = _gen(cuda, batch)
    lens = lens or [(37 * b) % 190 for b in range(batch)]
    nq, nkv, hd = 7, 1, 128
    cache, ref = _new(batch, nkv, max(lens) + 1, hd, cuda), kr.RefKV(batch, nkv, hd)
    from polar_pack_b200.kv8 import kv8_append
    k, v = (_rand(g, batch, max(lens), nkv, hd) for _ in "kv")
    kv8_append(cache, k, v, _ints([0] * batch, cuda), counts=_ints(lens, cuda))
    for w, x in enumerate((k.cpu(), v.cpu())):                  # whole blocks at once: the reference goes by rows
        for b, l in enumerate(lens):
            r = ref.s[w][b][0]
            for j in range(l // 64):
                c, s = kr.quantise(x[b, 64 * j:64 * j + 64, 0])
                r.codes.append(c)
                r.scales.append(s)
            last = (l - 1) // 64 * 64 if l else 0
            r.rows, r.len = x[b, last:l, 0].clone(), l
    q, kn, vn = _rand(g, batch, nq, hd, spread=2.0), _rand(g, batch, nkv, hd), _rand(g, batch, nkv, hd)
    weights = cache.new_weights()
    out = kv8_decode(q, kn, vn, cache, _ints(lens, cuda), weights=weights)
    ref.append(kn[:, None], vn[:, None], [1] * batch)
    want, probs = kr.attention(ref, q[:, None], [1] * batch)
    _check_out(out, want[:, 0], ref)
    for b in range(batch):
        p = probs[b][0]
        assert ((weights[b, 0, :len(p)].cpu().double() - p).abs() <= 2e-4 * p + 1e-6).all()
        assert not weights[b, 0, len(p):].any()


def test_batches_share_scratch(cuda):
    """Calls of different sizes in turn on one stream, and a batch that goes in parts."""
    from polar_pack_b200.kv8 import kv8_append, kv8_decode
    g = _gen(cuda, 29)
    B, n = 1100, 70
    k, v, q = _rand(g, B, n, 1, 64), _rand(g, B, n, 1, 64), _rand(g, B, 3, 64, spread=2.0)
    cache = _new(B, 1, 128, 64, cuda)
    pos = torch.arange(B, device=cuda, dtype=torch.int32) % (n - 1)
    kv8_append(cache, k, v, pos * 0, counts=pos)
    few = _new(3, 1, 20_032, 64, cuda)
    kf, vf = _rand(g, 3, 20_000, 1, 64), _rand(g, 3, 20_000, 1, 64)
    kv8_append(few, kf, vf, _ints([0, 0, 0], cuda))
    new = k[:, n - 1], v[:, n - 1]
    a = [kv8_decode(q, *new, cache, pos)]
    b = [kv8_decode(q[:3], kf[:, 0], vf[:, 0], few, _ints([20_000] * 3, cuda))]
    a.append(kv8_decode(q, *new, cache, pos))
    b.append(kv8_decode(q[:3], kf[:, 0], vf[:, 0], few, _ints([20_000] * 3, cuda)))
    assert torch.equal(*a) and torch.equal(*b) and int(cache.status) == 0
    ref = kr.RefKV(B, 1, 64)
    for w, (x, y) in enumerate(((k, new[0]), (v, new[1]))):
        x, y = x.cpu(), y.cpu()
        for i in range(B):
            r, l = ref.s[w][i][0], i % (n - 1)
            rows = torch.cat([x[i, :l, 0], y[i]])
            if l + 1 >= 64:
                c, s = kr.quantise(rows[:64])
                r.codes.append(c)
                r.scales.append(s)
            r.rows, r.len = rows[(l // 64) * 64:], l + 1
    want, _ = kr.attention(ref, q[:, None], [1] * B)
    _check_out(a[0], want[:, 0], ref)


def test_peaked_scores_and_scale(cuda):
    """A sink that takes nearly all the weight, blocks of very different scale,
    infinite keys in one head only."""
    from polar_pack_b200.kv8 import kv8_append, kv8_attention
    g = _gen(cuda, 13)
    n, hd = 333, 128
    k, v, q = _rand(g, 1, n, 2, hd), _rand(g, 1, n, 2, hd), _rand(g, 1, 1, 4, hd, spread=1.0)
    k[0, 0, 0] = q[0, 0, 0] * 8
    v[0, 64:128] *= 1000
    v[0, 128:192] *= 1e-3
    cache, ref = _new(1, 2, 384, hd, cuda), kr.RefKV(1, 2, hd)
    kv8_append(cache, k, v, _ints([0], cuda))
    ref.append(k, v, [n])
    out = kv8_attention(q, cache, _ints([n], cuda), scale=0.7)
    want, _ = kr.attention(ref, q, [1], scale=0.7)
    for h in range(4):                     # each head within its own weighted |v|: the scales differ by 10^6
        kk, vv = ref.s[0][0][h // 2].values(), ref.s[1][0][h // 2].values()
        p = torch.softmax(kk @ q[0, 0, h].cpu().double() * 0.7, 0)
        bound = OUT_TOL * (p @ vv.abs()) + 2.0 ** -24
        assert ((out[0, 0, h].cpu().double() - want[0, 0, h]).abs() <= bound).all(), h
    cache.k_tail[0, 1, 2, 3] = float("inf")
    bad = kv8_attention(q, cache, _ints([n], cuda), scale=0.7)
    assert torch.equal(bad[0, 0, :2], out[0, 0, :2])


def test_offsets_past_32_bits(cuda):
    """The last sequence of a cache of more than 2^32 codes."""
    from polar_pack_b200.kv8 import KV8Cache, kv8_append, kv8_decode, kv8_restore
    B, heads, cap, hd = 9, 8, 1 << 16, 128
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    codes = [torch.empty(B, heads, cap, hd, dtype=torch.uint8, device=cuda) for _ in "kv"]
    scales = [torch.zeros(B, heads, cap // 64, device=cuda) for _ in "kv"]
    tails = [torch.zeros(B, heads, 64, hd, dtype=torch.float16, device=cuda) for _ in "kv"]
    cache, small = KV8Cache(*codes, *scales, *tails), _new(1, heads, 256, hd, cuda)
    g = _gen(cuda, 17)
    k, v, q = _rand(g, 1, 131, heads, hd), _rand(g, 1, 131, heads, hd), _rand(g, 1, 2 * heads, hd)
    many = lambda x: x.expand(B, *x.shape[1:])
    pos = _ints([-1] * (B - 1) + [0], cuda)
    kv8_append(cache, many(k[:, :130]), many(v[:, :130]), pos)
    kv8_append(small, k[:, :130], v[:, :130], _ints([0], cuda))
    pos = _ints([-1] * (B - 1) + [130], cuda)
    a = kv8_decode(many(q), many(k[:, 130]), many(v[:, 130]), cache, pos)
    b = kv8_decode(q, k[:, 130], v[:, 130], small, _ints([130], cuda))
    lens = _ints([0] * (B - 1) + [131], cuda)
    x, y = kv8_restore(cache, lens, count=131), kv8_restore(small, _ints([131], cuda), count=131)
    assert torch.equal(x[0][-1], y[0][0]) and torch.equal(x[1][-1], y[1][0])
    assert (a[-1].float() - b[0].float()).abs().max() <= OUT_TOL * v.abs().max().float() and not a[:-1].any()


def test_streams_and_graph(cuda):
    """On another stream, and replayed from a CUDA graph with positions on the device."""
    from polar_pack_b200.kv8 import kv8_decode
    g = _gen(cuda, 19)
    def start():
        c, r = _new(2, 2, 256, 128, cuda), kr.RefKV(2, 2, 128)
        _fill(c, r, [60, 3], _gen(cuda, 20))
        return c
    q, k, v = _rand(g, 8, 2, 14, 128), _rand(g, 8, 2, 2, 128), _rand(g, 8, 2, 2, 128)
    one, two = start(), start()
    pos = _ints([60, 3], cuda)
    w1 = one.new_weights()
    want = []
    for i in range(8):
        want.append(kv8_decode(q[i], k[i], v[i], one, pos, weights=w1))
        pos += 1
    torch.cuda.synchronize()
    s = torch.cuda.Stream(cuda)
    pos, w2 = _ints([60, 3], cuda), two.new_weights()
    qs, ks, vs = (torch.empty_like(t[0]) for t in (q, k, v))
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for t, u in ((qs, q), (ks, k), (vs, v)):
            t.copy_(u[0])
        first = kv8_decode(qs, ks, vs, two, pos, weights=w2)
    s.synchronize()
    assert torch.equal(first, want[0])
    w2.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = kv8_decode(qs, ks, vs, two, pos, weights=w2)
        pos.add_(1)
    for i in range(8):
        with torch.cuda.stream(s):
            for t, u in ((qs, q), (ks, k), (vs, v)):
                t.copy_(u[i])
            graph.replay()
        s.synchronize()
        assert torch.equal(out, want[i])
    assert torch.equal(w1, w2)


def test_workspaces(cuda):
    """A given workspace gives the same bits and is left ready for the next
    call; a graph captured without one owns its scratch, whatever the streams
    around it do."""
    from polar_pack_b200.kv8 import kv8_attention, kv8_decode
    g = _gen(cuda, 41)
    lens = [700, 64, 0, 131]
    cache, ref = _new(4, 2, 768, 128, cuda), kr.RefKV(4, 2, 128)
    _fill(cache, ref, lens, _gen(cuda, 42))
    q, k, v = _rand(g, 4, 14, 128), _rand(g, 4, 2, 128), _rand(g, 4, 2, 128)
    pos, n = _ints(lens, cuda), _ints([x + 1 for x in lens], cuda)
    want = kv8_decode(q, k, v, cache, pos)
    many = _rand(g, 4, 40, 14, 128)
    both = _ints([min(x, 40) for x in lens], cuda)
    prompt = kv8_attention(many, cache, _ints(lens, cuda), both)
    ws = cache.new_workspace(40, 14)
    step = cache.new_workspace(1, 14, True)
    w = cache.new_weights()
    for _ in range(3):      # the same token again: the cache stays the same
        assert torch.equal(kv8_decode(q, k, v, cache, pos, weights=w, workspace=step), want)
        assert torch.equal(kv8_attention(q[:, None], cache, n, workspace=step)[:, 0], want)
        assert torch.equal(kv8_attention(many, cache, _ints(lens, cuda), both, workspace=ws), prompt)
    for bad in (step[:-256], step[1:], step.view(torch.int8), step.cpu()):
        with pytest.raises(ValueError):
            kv8_decode(q, k, v, cache, pos, weights=w, workspace=bad)
    torch.cuda.synchronize()
    s, graph = torch.cuda.Stream(cuda), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        a = kv8_decode(q, k, v, cache, pos)
        b = kv8_attention(q[:, None], cache, n)[:, 0]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)


# ------------------------------------------------------------ eviction ----
@pytest.mark.parametrize("hd,keep,sinks,recent,lens", [
    (128, 100, 4, 10, [300, 100, 101, 0]),
    (64, 128, 0, 0, [129, 500, 64, 1]),
    (128, 192, 70, 122, [400, 193, 192, 257]),       # everything kept is forced: whole blocks move or stay
    (64, 1, 0, 1, [300, 1, 2, 64]),
    (128, 65, 1, 0, [448, 66, 65, 300]),
])
def test_evict(cuda, hd, keep, sinks, recent, lens):
    from polar_pack_b200.kv8 import kv8_evict
    g = _gen(cuda, keep)
    B, heads = len(lens), 2
    cache, ref = _new(B, heads, 512, hd, cuda), kr.RefKV(B, heads, hd)
    _fill(cache, ref, lens, g)
    w = torch.rand(B, heads, 512, generator=g, device=cuda)
    w[0, 0] = (w[0, 0] * 4).floor()                            # many ties
    w[:, 1, 5:90:7] = 0.0
    w[0, 1, 40:60] = float("inf")
    w[1 % B, 0, 80:84] = float("nan")
    w[2, 0] = 0.0                                              # all equal: the lowest positions stay
    into = _new(B, heads, keep + 70, hd, cuda)
    iw = torch.full((B, heads, into.capacity), 7.0, device=cuda)
    new, kept = kv8_evict(cache, into, _ints(lens, cuda), w, keep, sinks=sinks, recent=recent, into_weights=iw)
    assert new.tolist() == [min(l, keep) for l in lens] and int(into.status) == 0
    want = kr.RefKV(B, heads, hd)
    for b, l in enumerate(lens):
        for h in range(heads):
            idx = kr.evict_positions(w[b, h].cpu(), l, keep, sinks, recent)
            assert kept[b, h].tolist() == idx + [-1] * (keep - len(idx)), (b, h)
            kw = w[b, h].cpu()[idx]
            assert torch.equal(torch.nan_to_num(iw[b, h, :len(idx)].cpu(), nan=-1.0), torch.nan_to_num(kw, nan=-1.0))
            assert not iw[b, h, len(idx):].any()
            for side in (0, 1):
                want.s[side][b][h] = kr.evict_side(ref.s[side][b][h], idx)
    _check_cache(into, want)


def test_evict_long(cuda):
    """Against torch's selection at a length of many rounds, with ties throughout."""
    from polar_pack_b200.kv8 import kv8_evict, kv8_restore
    g = _gen(cuda, 23)
    L, keep = 50_001, 20_000
    cache, ref = _new(2, 1, L, 64, cuda, stale=False), kr.RefKV(2, 1, 64)
    from polar_pack_b200.kv8 import kv8_append
    k, v = (_rand(g, 2, L, 1, 64) for _ in "kv")
    kv8_append(cache, k, v, _ints([0, 0], cuda))
    w = (torch.rand(2, 1, cache.capacity, generator=g, device=cuda) * 1000).floor()
    into = _new(2, 1, keep, 64, cuda)
    lens = _ints([L, L - 7], cuda)
    new, kept = kv8_evict(cache, into, lens, w, keep, sinks=3, recent=100)
    old, got = kv8_restore(cache, lens), kv8_restore(into, new)
    for b, l in enumerate(lens.tolist()):
        key = w[b, 0].clone()
        key[:3], key[l - 100:l], key[l:] = 1e9, 1e9, -1
        idx = torch.sort(torch.sort(key, descending=True, stable=True).indices[:keep]).values
        assert torch.equal(kept[b, 0].long(), idx)
        for side in (0, 1):
            x, y = old[side][b, idx, 0].float(), got[side][b, :keep, 0].float()
            step = x.view(-1)[: keep // 64 * 64 * 64].view(-1, 64 * 64).abs().amax(1).repeat_interleave(64) / 127
            # requantised once: half a step, and FP16's rounding of both
            err = (x - y).abs().amax(1)[: keep // 64 * 64]
            assert (err <= step * 0.5 + 2e-3 * step * 127 / 2).all()


# ------------------------------------------------------------ refusals ----
def test_refusals(cuda):
    from polar_pack_b200.kv8 import KV8Cache, kv8_append, kv8_attention, kv8_decode, kv8_evict
    c = KV8Cache.empty(2, 2, 128, 128, cuda)
    z = lambda *s, t=torch.float16: torch.zeros(*s, dtype=t, device=cuda)
    pos = _ints([0, 0], cuda)
    with pytest.raises(ValueError):
        KV8Cache.empty(2, 2, 128, 96, cuda)
    with pytest.raises(ValueError):
        KV8Cache(c.k_codes[:, :, :100], c.v_codes, c.k_scales, c.v_scales, c.k_tail, c.v_tail)
    with pytest.raises(RuntimeError):
        KV8Cache.empty(1, 1, 64, 64, "cpu")
    for bad in (z(2, 3, 2, 128, t=torch.float32), z(1, 3, 2, 128), z(2, 3, 2, 64), z(2, 2, 128), z(2, 3, 2, 128).cpu()):
        with pytest.raises(ValueError):
            kv8_append(c, bad, z(2, 3, 2, 128), pos)
    for bad in (pos.long(), pos[:1], pos.cpu(), _ints([0, 0, 0, 0], cuda)[::2]):
        with pytest.raises(ValueError):
            kv8_append(c, z(2, 3, 2, 128), z(2, 3, 2, 128), bad)
        with pytest.raises(ValueError):
            kv8_attention(z(2, 3, 4, 128), c, bad)
    with pytest.raises(ValueError):
        kv8_attention(z(2, 3, 5, 128), c, pos)              # query heads not a multiple of the kv heads
    with pytest.raises(ValueError):
        kv8_attention(z(2, 1, 34, 128), c, pos)             # 17 to one
    with pytest.raises(ValueError):
        kv8_decode(z(2, 4, 128), z(2, 2, 128), z(2, 2, 128), c, pos, weights=z(2, 2, 64, t=torch.float32))
    with pytest.raises(ValueError):
        kv8_decode(z(2, 4, 128), z(2, 2, 128), z(2, 2, 128), c, pos, out=z(2, 4, 64))
    w = c.new_weights()
    for keep, sinks, recent in ((0, 0, 0), (129, 0, 0), (64, 60, 5), (64, -1, 5)):
        with pytest.raises(ValueError):
            kv8_evict(c, KV8Cache.empty(2, 2, 128, 128, cuda), pos, w, keep, sinks, recent)
    with pytest.raises(ValueError):
        kv8_evict(c, c, pos, w, 64, 0, 0)
    with pytest.raises(ValueError):
        kv8_evict(c, KV8Cache.empty(2, 1, 128, 128, cuda), pos, w, 64, 0, 0)
    assert kv8_attention(z(2, 0, 4, 128), c, pos).shape == (2, 0, 4, 128)
    kv8_append(c, z(2, 0, 2, 128), z(2, 0, 2, 128), pos)


# ----------------------------------------------- what a call must accept ----
def _odd_ones(x):
    """x with strides of its size-1 dimensions that mean nothing, and are odd."""
    return x.as_strided(x.shape, [s if n > 1 else 8 * s + 1 + 2 * i for i, (n, s) in enumerate(zip(x.shape, x.stride()))])


def test_strides_of_single_rows(cuda):
    """The stride of a dimension of one is nobody's business: batch 1, one token, one head."""
    from polar_pack_b200.kv8 import kv8_append, kv8_attention, kv8_decode
    g = _gen(cuda, 61)
    k, v, q = _rand(g, 1, 3, 1, 64), _rand(g, 1, 3, 1, 64), _rand(g, 1, 1, 2, 64)
    pos = _ints([0], cuda)
    got = []
    for odd in (lambda x: x, _odd_ones):
        c = _new(1, 1, 64, 64, cuda)
        kv8_append(c, odd(k[:, :2]), odd(v[:, :2]), pos)
        kv8_append(c, odd(k[:, 2:]), odd(v[:, 2:]), pos + 2)
        out = torch.zeros_like(q)
        res = [kv8_attention(odd(q), c, pos + 3, out=odd(out)), kv8_attention(odd(q), c, pos + 3)]
        out = torch.zeros_like(q[:, 0])
        res += [kv8_decode(odd(q[:, 0]), odd(k[:, 0]), odd(v[:, 0]), c, pos + 3, out=odd(out)), out]
        got.append(res + [c.k_tail[:, :, :4], c.v_tail[:, :, :4]])
        assert int(c.status) == 0
    for a, b in zip(*got):
        assert a.any() and torch.equal(a, b)


def test_status_is_checked(cuda):
    """The status word is written by the device: another place or type is refused."""
    from polar_pack_b200.kv8 import KV8Cache
    KV8Cache.empty(1, 1, 64, 64, cuda, status=torch.zeros(1, dtype=torch.int32, device=cuda))
    for bad in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, device=cuda),
                torch.zeros(1, dtype=torch.int64, device=cuda), torch.zeros(0, dtype=torch.int32, device=cuda)):
        with pytest.raises((ValueError, RuntimeError)):
            KV8Cache.empty(1, 1, 64, 64, cuda, status=bad)


def test_positions_at_the_end_of_the_type(cuda):
    """A position of 2^31 - 1 is past every capacity, not an unused sequence."""
    from polar_pack_b200.kv8 import kv8_append, kv8_decode
    g = _gen(cuda, 62)
    q, k, v = _rand(g, 2, 4, 128), _rand(g, 2, 1, 128), _rand(g, 2, 1, 128)
    pos = _ints([2 ** 31 - 1, 3], cuda)
    c = _new(2, 1, 64, 128, cuda, stale=False)
    w = c.new_weights()
    out = kv8_decode(q, k, v, c, pos, weights=w)
    assert int(c.status) == 5 and not out[0].any() and out[1].any() and not w[0].any() and w[1].any()
    c.status.zero_()
    kv8_append(c, k[:, None], v[:, None], pos)
    assert int(c.status) == 5


@pytest.mark.parametrize("nq,nkv,hd,n,lens,counts", [
    (4, 2, 64, 4, [40, 2, 70], [4, 4, 1]),          # one tile of rows
    (16, 2, 128, 10, [30, 90, 128], [10, 7, 9]),     # 80 rows to a kv head
    (2, 1, 128, 200, [250, 200, 60], [200, 199, 60]),   # more than 256
    (14, 2, 64, 60, [100, 4100, 0], [60, 60, 0]),    # positions split
])
def test_values_that_are_not_numbers(cuda, nq, nkv, hd, n, lens, counts):
    """Values of NaN and infinity in the open block: rows that attend them get
    what the formula gives, all others are as if they were not there."""
    from polar_pack_b200.kv8 import kv8_append, kv8_attention
    g = _gen(cuda, 63 + n)
    B = len(lens)
    cap = -(-max(lens) // 64) * 64 + 64
    k, v = (_rand(g, B, max(lens), nkv, hd) for _ in "kv")
    q = _rand(g, B, n, nq, hd, spread=2.0)
    bad = v.clone()
    late = [max(l - max(c // 2, 1), 0) for l, c in zip(lens, counts)]      # the first position that is not finite
    late = [max(t, (l - 1) // 64 * 64) for t, l in zip(late, lens)]
    for b, (t, l) in enumerate(zip(late, lens)):
        if l:
            bad[b, t, :, 3], bad[b, t, 0, 9], bad[b, l - 1, :, 3], bad[b, l - 1, 0, 20] = (
                float("inf"), float("nan"), -float("inf"), -float("inf"))
    outs, want = [], None
    for x in (v, bad):
        cache = _new(B, nkv, cap, hd, cuda)
        kv8_append(cache, k, x, _ints([0] * B, cuda), counts=_ints(lens, cuda))
        outs.append(kv8_attention(q, cache, _ints(lens, cuda), counts=_ints(counts, cuda)))
        assert int(cache.status) == 0
    ref = kr.RefKV(B, nkv, hd)
    ref.append(k, bad, lens)
    want, _ = kr.attention(ref, q, counts)
    plain, out = outs
    vmax = float(v.abs().max())
    for b, (l, c) in enumerate(zip(lens, counts)):
        for i in range(n):
            if i >= c or l - c + i < late[b]:
                assert torch.equal(out[b, i], plain[b, i]), (b, i)
                assert not (i >= c or l - c + i < 0) or not out[b, i].any()
                continue
            x, y = out[b, i].cpu().double(), want[b, i]
            same = (x == y) | (x.isnan() & y.isnan())
            assert (same | ((x - y).abs() <= OUT_TOL * vmax)).all(), (b, i)
            assert not torch.isfinite(x[:, 3]).any()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size,tail", [(1.0, 1.0), (1e-2, 1e-2), (1e-3, 1e-3), (1e-4, 1e-4), (1e-3, 30.0), (1.0, 1e-3),
                                       (100.0, 100.0)])
def test_small_values_beside_a_sink(cuda, hd, size, tail):
    """Values of any size, where a first position takes most of the weight and
    the rest of it is spread over all the others; positions not split."""
    from polar_pack_b200.kv8 import kv8_append, kv8_attention
    g = _gen(cuda, hd)
    heads, n, L = 90, 270, 3000
    last = (L - 1) // 64 * 64
    for gap in (8.0, 11.0, 13.0):
        q = torch.zeros(1, n, heads, hd, device=cuda)
        q[..., 0] = 8
        k = torch.zeros(1, L, heads, hd, device=cuda)
        k[:, 0, :, 0] = gap / 8 * hd ** 0.5
        v = 1 + 0.1 * torch.rand(1, L, heads, hd, generator=g, device=cuda)
        v[:, 0] *= -1
        v[:, :last] *= size
        v[:, last:] *= tail
        k, v, q = k.half(), v.half(), q.half()
        cache = _new(1, heads, 3008, hd, cuda, stale=False)
        kv8_append(cache, k, v, _ints([0], cuda))
        out = kv8_attention(q, cache, _ints([L], cuda))
        x = []
        for codes, scales, rows in ((cache.k_codes, cache.k_scales, cache.k_tail),
                                    (cache.v_codes, cache.v_scales, cache.v_tail)):
            y = (codes[0].double() - 128) * scales[0].double().repeat_interleave(64, 1)[..., None]
            x.append(torch.cat([y[:, :last], rows[0, :, :L - last].double()], 1))
        for i in (n - 1, n // 2, 0):
            end = L - n + i + 1
            p = torch.softmax((x[0][:, :end] @ q[0, i, :, :, None].double())[..., 0] / hd ** 0.5, -1)
            want = (p[:, None] @ x[1][:, :end])[:, 0]
            bound = OUT_TOL * x[1][:, :end].abs().amax((1, 2))[:, None] + 2.0 ** -24
            assert ((out[0, i].double() - want).abs() <= bound).all(), (gap, i)
        assert int(cache.status) == 0


def test_launch_overlap(cuda):
    """Each kernel started while the one before it runs: the same bits as one after another."""
    from polar_pack_b200 import _lib
    from polar_pack_b200.kv8 import kv8_append, kv8_attention, kv8_decode, kv8_evict, kv8_restore
    runs = []
    old = _lib.set_launch_overlap(False)
    try:
        for on in (False, True):
            _lib.set_launch_overlap(on)
            g = _gen(cuda, 71)
            got = []
            for nq, nkv, hd, n, lens in ((16, 2, 128, 150, [4000, 150, 0]), (6, 3, 64, 5, [700, 64, 5]),
                                         (7, 1, 128, 1, [63, 1, 2000])):
                counts = [min(n, l) for l in lens]
                k, v = (_rand(g, 3, max(lens), nkv, hd) for _ in "kv")
                q, q1 = _rand(g, 3, n, nq, hd, spread=2.0), _rand(g, 4, 3, nq, hd, spread=2.0)
                k1, v1 = (_rand(g, 4, 3, nkv, hd) for _ in "kv")
                a, b = (_new(3, nkv, 4100, hd, cuda, stale=False) for _ in "ab")
                pos, new, w = _ints(lens, cuda), _ints([l + 4 for l in lens], cuda), a.new_weights()
                steps = [pos + i for i in range(4)]
                for _ in range(3):           # the caches are written again while they may still be read
                    kv8_append(a, k, v, pos * 0, counts=pos)
                    got.append(kv8_attention(q, a, pos, counts=_ints(counts, cuda)))
                    for i in range(4):
                        got.append(kv8_decode(q1[i], k1[i], v1[i], a, steps[i], weights=w))
                    got += kv8_evict(a, b, new, w, 100, sinks=2, recent=30)
                    got += kv8_restore(b, got[-2], count=100)
                    got.append(kv8_attention(q, b, got[-4], counts=_ints(counts, cuda).clamp(max=100)))
                got.append(w)
                assert int(a.status) == 0 and int(b.status) == 0
            runs.append(got)
    finally:
        _lib.set_launch_overlap(old)
    for x, y in zip(*runs):
        assert torch.equal(x, y)
