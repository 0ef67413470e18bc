"""The operators around the 8-bit KV cache, as cases that can be measured: decode and prompt attention over
the cache, its writer, eviction by accumulated attention weight, and the log probabilities of given tokens.

Cache of one layer: positions 0, 1, 2, ... of a sequence in blocks of 64.  A stored key or value is
``(code - 128) * scale``, uint8 codes ``[B][kv heads][capacity][head dim]`` with one float32 scale per block
and head, ``[B][kv heads][capacity / 64]``: ``scale = max|x| / 127``, ``code = 128 + round(x / scale)``
(ties to even; all codes 128 where the scale is 0).  The block that holds a sequence's last token is read from
its FP16 rows ``[B][kv heads][64][head dim]`` (the tail); its codes are written when it is complete.
"""
import math
import random

import torch

own = False
BLOCK = 64
DEV = "cuda"


# ---------------------------------------------------------------- cases ----
def listed():
    return [
        # one decode step of the four models of the 3B-class pack at its context of 1024: latency counts
        dict(name="decode 3B ctx 1024", kind="decode", batch=4, q_heads=16, kv_heads=2, head_dim=128, length=1023,
             ragged=False, weights=False),
        # one decode step of the four 7B-class models at context 2048, with the attention weights that the
        # eviction goes by accumulated
        dict(name="decode 7B ctx 2048 weights", kind="decode", batch=4, q_heads=28, kv_heads=4, head_dim=128,
             length=2047, ragged=False, weights=True),
        # batched serving: 16 requests to each of the four 7B-class models, of all lengths (empty slots too)
        dict(name="decode 7B batch 64 ragged", kind="decode", batch=64, q_heads=28, kv_heads=4, head_dim=128,
             length=8190, ragged=True, weights=False),
        # a chunk of a long prompt over what the cache holds of it already (3B-class, ragged)
        dict(name="prompt 3B chunk 509 of 4001", kind="prompt", batch=4, q_heads=16, kv_heads=2, head_dim=128,
             tokens=509, length=4001, ragged=True),
        # whole prompts of the four 7B-class models at context 2048
        dict(name="prompt 7B 2048", kind="prompt", batch=4, q_heads=28, kv_heads=4, head_dim=128, tokens=2048,
             length=2048, ragged=False),
        # a few tokens behind what is there (a turn of a dialogue), blocks left open at both ends; read back
        dict(name="append 3B 17 tokens", kind="append", batch=4, kv_heads=2, head_dim=128, tokens=17, length=1021,
             ragged=True),
        # prompts of many requests into their caches; read back
        dict(name="append 7B batch 16 x 2048", kind="append", batch=16, kv_heads=4, head_dim=128, tokens=2048,
             length=2500, ragged=True),
        # the four 3B-class models at a full context of 1024, half of it evicted
        dict(name="evict 3B 1024 to 512", kind="evict", batch=4, kv_heads=2, head_dim=128, length=1024, keep=512,
             sinks=4, recent=64, ragged=False),
        # long caches of several requests down to a common budget
        dict(name="evict 7B 16384 to 4000", kind="evict", batch=8, kv_heads=4, head_dim=128, length=16384, keep=4000,
             sinks=4, recent=250, ragged=True),
        # the logits of one decode step: four models, their tokens and the 20 likeliest others
        dict(name="score 4 rows top 20", kind="score", rows=4, vocab=151936, top=20, dtype="float16"),
        # a prompt scored under the four models (perplexity), with the 5 likeliest tokens at each place
        dict(name="score 2048 rows top 5", kind="score", rows=2048, vocab=151936, top=5, dtype="float16"),
        # float32 logits over a small odd vocabulary, token scores only
        dict(name="score fp32 odd vocab", kind="score", rows=301, vocab=32003, top=0, dtype="float32"),
    ]


HEADS = ((16, 2, 128), (28, 4, 128), (8, 8, 128), (14, 2, 64), (16, 1, 128), (6, 3, 64))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("decode", "decode", "prompt", "prompt", "append", "evict", "score", "score"))
    nq, nkv, hd = rng.choice(HEADS)
    if kind == "score":
        vocab = rng.choice((151936, 152064, _log(rng, 1000, 200000) | 1))
        dtype = rng.choice(("float16", "bfloat16", "float32"))
        rows = _log(rng, 1, max(1, 600_000_000 // (vocab * (4 if dtype == "float32" else 2))))
        return dict(kind=kind, rows=rows, vocab=vocab, top=rng.choice((0, 1, 5, 20, 32)), dtype=dtype)
    batch, ragged = _log(rng, 1, 64), rng.random() < 0.5
    room = 64 * 4 * 8192 * 128 // (batch * nkv * hd)          # positions that the largest listed cache has
    if kind == "decode":
        return dict(kind=kind, batch=batch, q_heads=nq, kv_heads=nkv, head_dim=hd,
                    length=_log(rng, 1, min(100_000, room)) - 1, ragged=ragged, weights=rng.random() < 0.4)
    if kind == "prompt":
        batch = _log(rng, 1, 16)
        tokens = _log(rng, 2, 2048)
        pairs = 4 * 28 * 2048 * 2048 // (batch * nq)          # query-position pairs that the largest listed case has
        return dict(kind=kind, batch=batch, q_heads=nq, kv_heads=nkv, head_dim=hd, tokens=tokens,
                    length=tokens + _log(rng, 1, max(1, min(30_000, pairs // tokens - tokens))) - 1, ragged=ragged)
    if kind == "append":
        batch = _log(rng, 1, 16)
        tokens = _log(rng, 1, 2048)
        return dict(kind=kind, batch=batch, kv_heads=nkv, head_dim=hd, tokens=tokens,
                    length=tokens + _log(rng, 1, 1000) - 1, ragged=ragged)
    batch = _log(rng, 1, 8)
    length = _log(rng, 100, 16384)
    keep = max(2, int(length * rng.uniform(0.1, 0.9)))
    recent = rng.randrange(0, keep // 2 + 1)
    return dict(kind=kind, batch=batch, kv_heads=nkv, head_dim=hd, length=length, keep=keep,
                sinks=min(4, keep - recent), recent=recent, ragged=ragged)


def _lens(case):
    """Tokens of each sequence after the call (decode: before it); ragged batches hold short and empty ones."""
    n, top = case["batch"], case["length"]
    if not case["ragged"]:
        return [top] * n
    r = random.Random(top * 1009 + n)
    lens = [r.randrange(0, top + 1) for _ in range(n)]
    lens[r.randrange(n)] = top
    if n > 2:
        lens[(lens.index(top) + 1) % n] = 0
    return lens


def _counts(case):
    """New tokens of each sequence, at most what its length allows."""
    return [min(case["tokens"], l) for l in _lens(case)]


def _capacity(case):
    return -(-(case["length"] + 1) // BLOCK) * BLOCK


# --------------------------------------------------------------- inputs ----
def _rows(g, *shape):
    """Keys or values: per-channel spread as in trained models, FP16."""
    x = torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)
    spread = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=DEV))
    return (x * spread * 0.4).half()


def _cache(case, lens, g):
    """A filled cache: codes, scales and tails of `lens` tokens."""
    b, nkv, hd, cap = case["batch"], case["kv_heads"], case["head_dim"], _capacity(case)
    last = (torch.tensor(lens, device=DEV).clamp(min=1) - 1) // BLOCK
    s = {}
    for n in "kv":
        x = _rows(g, b, nkv, cap, hd).view(b, nkv, cap // BLOCK, BLOCK, hd)
        s[n + "_tail"] = x[torch.arange(b, device=DEV), :, last].contiguous()
        codes, scales = _quantise(x)
        s[n + "_codes"], s[n + "_scales"] = codes.view(b, nkv, cap, hd), scales
    return s


def _handle(s):
    from polar_pack_b200.kv8 import KV8Cache
    return KV8Cache(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"], s["k_tail"], s["v_tail"])


def _int(v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": case, "kind": case["kind"]}
    if case["kind"] == "score":
        dt = getattr(torch, case["dtype"])
        s["logits"] = (torch.randn(case["rows"], case["vocab"], generator=g, device=DEV, dtype=torch.float32)
                       * 2.5).to(dt)
        # most tokens that a model is asked about are likely ones
        s["logits"][:, : case["vocab"] // 500 + 1] += 6
        s["tokens"] = torch.randint(0, case["vocab"] // 300 + 1, (case["rows"],), generator=g, device=DEV,
                                    dtype=torch.int32)
        return s
    lens, b, nkv, hd = _lens(case), case["batch"], case["kv_heads"], case["head_dim"]
    before = [l - c for l, c in zip(lens, _counts(case))] if case["kind"] == "append" else lens
    s.update(_cache(case, before, g))
    s["lens"] = _int(lens)
    if case["kind"] == "decode":
        s["q"] = _rows(g, b, case["q_heads"], hd) * 2
        s["k"], s["v"] = _rows(g, b, nkv, hd), _rows(g, b, nkv, hd)
        if case["weights"]:
            live = torch.arange(_capacity(case), device=DEV) < s["lens"][:, None, None]
            s["weights"] = torch.rand(b, nkv, _capacity(case), generator=g, device=DEV) * live
    elif case["kind"] == "prompt":
        s["q"] = _rows(g, b, case["tokens"], case["q_heads"], hd) * 2
        s["counts"] = _int(_counts(case))
    elif case["kind"] == "append":
        s["pos"], s["counts"] = _int(before), _int(_counts(case))
        s["k"], s["v"] = (_rows(g, b, case["tokens"], nkv, hd) for _ in "kv")
    else:
        live = torch.arange(_capacity(case), device=DEV) < s["lens"][:, None, None]
        s["weights"] = torch.rand(b, nkv, _capacity(case), generator=g, device=DEV).pow(4) * live
        cap = -(-case["keep"] // BLOCK) * BLOCK
        s["into"] = {n + "_codes": torch.zeros(b, nkv, cap, hd, device=DEV, dtype=torch.uint8) for n in "kv"}
        s["into"].update({n + "_scales": torch.zeros(b, nkv, cap // BLOCK, device=DEV) for n in "kv"})
        s["into"].update({n + "_tail": torch.zeros(b, nkv, BLOCK, hd, device=DEV, dtype=torch.float16) for n in "kv"})
        s["into_weights"] = torch.zeros(b, nkv, cap, device=DEV)
    if own:
        s["cache"] = _handle(s)
        if "into" in s:
            s["into_cache"] = _handle(s["into"])
    return s


# ------------------------------------------------------------------ run ----
def run(s):
    return (_own if own else _plain)[s["kind"]](s)


def _own_decode(s):
    from polar_pack_b200.kv8 import kv8_decode
    out = kv8_decode(s["q"], s["k"], s["v"], s["cache"], s["lens"], weights=s.get("weights"))
    return {"out": out, **_state(s)}


def _own_prompt(s):
    from polar_pack_b200.kv8 import kv8_attention
    return {"out": kv8_attention(s["q"], s["cache"], s["lens"], counts=s["counts"])}


def _own_append(s):
    from polar_pack_b200.kv8 import kv8_append, kv8_restore
    kv8_append(s["cache"], s["k"], s["v"], s["pos"], counts=s["counts"])
    k, v = kv8_restore(s["cache"], s["lens"], start=s["pos"], count=s["k"].shape[1])
    return {"k": k, "v": v, **_state(s)}


def _own_evict(s):
    from polar_pack_b200.kv8 import kv8_evict, kv8_restore
    c = s["case"]
    lens, kept = kv8_evict(s["cache"], s["into_cache"], s["lens"], s["weights"], c["keep"], sinks=c["sinks"],
                           recent=c["recent"], into_weights=s["into_weights"])
    k, v = kv8_restore(s["into_cache"], lens, count=c["keep"])
    return {"lens": lens, "kept": kept, "k": k, "v": v, "weights": s["into_weights"],
            "k_scales": s["into"]["k_scales"], "v_scales": s["into"]["v_scales"]}


def _own_score(s):
    from polar_pack_b200.scoring import token_logprobs
    r = token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    return {"logprob": r.logprob, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}


_own = {"decode": _own_decode, "prompt": _own_prompt, "append": _own_append, "evict": _own_evict, "score": _own_score}


def _state(s):
    """The updated state beside the codes (the codes that a call writes are read back in the append cases)."""
    names = ("k_tail", "v_tail", "k_scales", "v_scales") + (("weights",) if "weights" in s else ())
    return {n: s[n] for n in names}


# ---------------------------------------------------------- plain forms ----
def _quantise(x):
    """Codes and scales of blocks [..., BLOCK, hd] (FP16 or float32 values)."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=65504.0, neginf=-65504.0)
    scale = x.abs().amax(dim=(-2, -1)) / torch.full((), 127.0, device=x.device)
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = torch.round(x / safe[..., None, None]) + 128
    return codes.to(torch.uint8), scale


def _values(s, n, lens):
    """Float32 keys (n = "k") or values of every position, zero past each sequence's length."""
    codes, scales, tail = s[n + "_codes"], s[n + "_scales"], s[n + "_tail"]
    b, nkv, cap, hd = codes.shape
    x = (codes.view(b, nkv, cap // BLOCK, BLOCK, hd).float() - 128) * scales[..., None, None]
    last = ((lens.clamp(min=1) - 1) // BLOCK).long()
    x[torch.arange(b, device=x.device), :, last] = tail.float()
    live = torch.arange(cap, device=x.device) < lens[:, None]
    return x.view(b, nkv, cap, hd).masked_fill(~live[:, None, :, None], 0.0)


def _softmax(scores, seen):
    """Probabilities over the last axis where `seen`; a row that sees nothing is all zeros."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _plain_append_rows(s, k, v, pos, counts):
    """Rows i < counts[b] of k, v [B][n][kv heads][hd] to positions pos[b] + i of the cache."""
    b, n, nkv, hd = k.shape
    cap = s["k_codes"].shape[2]
    bi = torch.arange(b, device=k.device)
    step = torch.arange(cap, device=k.device)
    lens = pos + counts
    src = step[None, :] - pos[:, None]
    new = (src >= 0) & (src < counts[:, None])
    old = (pos.clamp(min=1) - 1) // BLOCK
    last = ((lens.clamp(min=1) - 1) // BLOCK).long()
    first = pos // BLOCK                                             # the block that the first new token falls in
    for name, x in (("k", k), ("v", v)):
        full = torch.zeros(b, nkv, cap // BLOCK, BLOCK, hd, device=k.device, dtype=torch.float16)
        full[bi, :, old.long()] = s[name + "_tail"]                     # what the tail held
        rows = x.transpose(1, 2)[bi[:, None], :, src.clamp(0, n - 1).long()]      # [B][cap][nkv][hd]
        full = full.view(b, nkv, cap, hd)
        full = torch.where(new[:, None, :, None], rows.transpose(1, 2), full).view(b, nkv, cap // BLOCK, BLOCK, hd)
        codes, scales = _quantise(full)
        block = step[: cap // BLOCK][None, :]
        done = ((block >= first[:, None]) & ((block + 1) * BLOCK <= lens[:, None]) & (counts > 0)[:, None])[:, None]
        s[name + "_codes"].copy_(torch.where(done[..., None, None], codes, s[name + "_codes"].view_as(codes))
                                 .view_as(s[name + "_codes"]))
        s[name + "_scales"].copy_(torch.where(done, scales, s[name + "_scales"]))
        slot = step[:BLOCK]
        at = last[:, None] * BLOCK + slot[None, :]
        fresh = (at >= pos[:, None]) & (at < lens[:, None])
        s[name + "_tail"].copy_(torch.where(fresh[:, None, :, None], full[bi, :, last], s[name + "_tail"]))


def _plain_token(s):
    """One token's rows s["k"], s["v"] [B][kv heads][hd] to position s["lens"][b]."""
    pos = s["lens"].long()
    bi, block, done = torch.arange(len(pos), device=pos.device), pos // BLOCK, (pos % BLOCK == BLOCK - 1)[:, None]
    for n in "kv":
        s[n + "_tail"][bi, :, pos % BLOCK] = s[n]
        codes, scales = _quantise(s[n + "_tail"])
        blocks = s[n + "_codes"].view(*s[n + "_scales"].shape, BLOCK, -1)
        blocks[bi, :, block] = torch.where(done[..., None, None], codes, blocks[bi, :, block])
        s[n + "_scales"][bi, :, block] = torch.where(done, scales, s[n + "_scales"][bi, :, block])


def _plain_decode(s):
    lens = s["lens"] + 1
    _plain_token(s)
    k, v, q = _values(s, "k", lens), _values(s, "v", lens), s["q"].float()
    b, nkv, cap, hd = k.shape
    scores = (q.view(b, nkv, -1, hd) @ k.transpose(2, 3)) * (1 / math.sqrt(hd))
    p = _softmax(scores, (torch.arange(cap, device=k.device) < lens[:, None])[:, None, None])
    if "weights" in s:
        s["weights"] += p.sum(2)
    return {"out": (p @ v).view(b, -1, hd).half(), **_state(s)}


def _plain_prompt(s):
    lens, counts, q = s["lens"], s["counts"], s["q"].float()
    k, v = _values(s, "k", lens), _values(s, "v", lens)
    b, n, nq, hd = q.shape
    nkv, cap = k.shape[1], k.shape[2]
    i = torch.arange(n, device=q.device)
    at = lens[:, None] - counts[:, None] + i
    seen = (torch.arange(cap, device=q.device) <= at[..., None]) & (i < counts[:, None])[..., None]
    q = q.view(b, n, nkv, nq // nkv, hd).permute(0, 2, 3, 1, 4).reshape(b, nkv, -1, hd)
    scores = ((q @ k.transpose(2, 3)) * (1 / math.sqrt(hd))).view(b, nkv, nq // nkv, n, cap)
    p = _softmax(scores, seen[:, None, None])
    out = (p.view(b, nkv, -1, cap) @ v).view(b, nkv, nq // nkv, n, hd)
    return {"out": out.permute(0, 3, 1, 2, 4).reshape(b, n, nq, hd).half()}


def _plain_restore(s, lens, start, count):
    """FP16 keys and values of positions start[b] .. start[b] + count - 1, zero past the length."""
    out = []
    at = start[:, None] + torch.arange(count, device=lens.device)
    for n in "kv":
        x = _values(s, n, lens).half()
        rows = x.transpose(1, 2)[torch.arange(len(lens), device=lens.device)[:, None], at.clamp(max=x.shape[2] - 1).long()]
        out.append(rows.masked_fill((at >= lens[:, None])[..., None, None], 0))
    return out


def _plain_append(s):
    _plain_append_rows(s, s["k"], s["v"], s["pos"], s["counts"])
    k, v = _plain_restore(s, s["lens"], s["pos"], s["k"].shape[1])
    return {"k": k, "v": v, **_state(s)}


def _plain_evict(s):
    c, lens, into = s["case"], s["lens"], s["into"]
    keep, cap = c["keep"], s["k_codes"].shape[2]
    b, nkv = s["weights"].shape[:2]
    at = torch.arange(cap, device=lens.device)
    forced = (at < c["sinks"]) | (at >= lens[:, None] - c["recent"])
    key = torch.where(forced[:, None], math.inf, s["weights"])
    key = torch.where((at < lens[:, None])[:, None], key, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.sort(torch.where(order < lens[:, None, None], order, cap), dim=-1).values
    alive = kept < cap
    new = torch.minimum(lens, torch.full_like(lens, keep))
    rows = -(-keep // BLOCK) * BLOCK
    pick = torch.nn.functional.pad(torch.where(alive, kept, 0), (0, rows - keep))
    there = torch.nn.functional.pad(alive, (0, rows - keep))
    first = pick[..., ::BLOCK]
    # a new block that is one whole coded block stays as it is
    whole = (first % BLOCK == 0) & (pick[..., BLOCK - 1::BLOCK] - first == BLOCK - 1) & there[..., BLOCK - 1::BLOCK]
    whole &= first // BLOCK != ((lens.clamp(min=1) - 1) // BLOCK)[:, None, None]
    full = there[..., BLOCK - 1::BLOCK]
    last = ((new.clamp(min=1) - 1) // BLOCK).long()
    bi = torch.arange(b, device=lens.device)
    slot = torch.arange(BLOCK, device=lens.device)
    fresh = last[:, None] * BLOCK + slot < new[:, None]
    for n in "kv":
        x = _values(s, n, lens).half()
        hd = x.shape[-1]
        x = torch.gather(x, 2, pick[..., None].expand(-1, -1, -1, hd)).masked_fill(~there[..., None], 0)
        x = x.view(b, nkv, rows // BLOCK, BLOCK, hd)
        codes, scales = _quantise(x)
        src = (first // BLOCK).clamp(max=cap // BLOCK - 1)
        blocks = s[n + "_codes"].view(b, nkv, cap // BLOCK, BLOCK, hd)
        same = torch.gather(blocks, 2, src[..., None, None].expand(-1, -1, -1, BLOCK, hd))
        codes = torch.where(whole[..., None, None], same, codes)
        scales = torch.where(whole, torch.gather(s[n + "_scales"], 2, src), scales)
        into[n + "_codes"].copy_(torch.where(full[..., None, None], codes, into[n + "_codes"].view_as(codes))
                                 .view_as(into[n + "_codes"]))
        into[n + "_scales"].copy_(torch.where(full, scales, into[n + "_scales"]))
        into[n + "_tail"].copy_(torch.where(fresh[:, None, :, None], x[bi, :, last], into[n + "_tail"]))
    w = torch.gather(s["weights"], 2, pick).masked_fill(~there, 0.0)
    s["into_weights"].copy_(w)
    k, v = _plain_restore(into, new, torch.zeros_like(new), keep)
    return {"lens": new, "kept": torch.where(alive, kept, -1).int(), "k": k, "v": v, "weights": s["into_weights"],
            "k_scales": into["k_scales"], "v_scales": into["v_scales"]}


def _plain_score(s):
    x, top = s["logits"].float(), s["case"]["top"]
    rows, vocab = x.shape
    peak = x.amax(-1, keepdim=True)
    z = torch.exp(x - peak)
    total = z.sum(-1)
    lse = peak[:, 0] + torch.log(total)
    token = x.gather(1, s["tokens"].long()[:, None])[:, 0]
    entropy = torch.log(total) - (z * (x - peak)).sum(-1) / total
    # value, then the lowest index, as one whole number each
    bits = (x + 0.0).view(torch.int32)                                # -0 is 0
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = order * (1 << 32) + (vocab - 1 - torch.arange(vocab, device=x.device))
    ids = vocab - 1 - (torch.topk(key, top, dim=-1).values & 0xFFFFFFFF) if top else order[:, :0]
    return {"logprob": token - lse, "entropy": entropy, "top_ids": ids.int(),
            "top_logprobs": x.gather(1, ids) - lse[:, None]}


_plain = {"decode": _plain_decode, "prompt": _plain_prompt, "append": _plain_append, "evict": _plain_evict,
          "score": _plain_score}


# ----------------------------------------------------------------- work ----
def work(case):
    kind = case["kind"]
    if kind == "score":
        size = {"float16": 2, "bfloat16": 2, "float32": 4}[case["dtype"]]
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}
    lens, b, nkv, hd = _lens(case), case["batch"], case["kv_heads"], case["head_dim"]
    coded = lambda l: max(0, l - 1) // BLOCK * BLOCK                 # positions read as codes, the others as FP16
    held = lambda l: nkv * (coded(l) * (2 * hd + 8 / BLOCK) + (l - coded(l)) * 4 * hd)
    if kind == "decode":
        nq = case["q_heads"]
        lens = [l + 1 for l in lens]
        byte = sum(held(l) for l in lens) + b * 4 * nq * hd + b * 8 * nkv * hd
        if case["weights"]:
            byte += 8 * nkv * sum(lens)
        return {"bytes": byte, "flops": 4 * hd * nq * sum(lens)}
    if kind == "prompt":
        nq, counts = case["q_heads"], _counts(case)
        pairs = sum(c * l - c * (c - 1) // 2 for c, l in zip(counts, lens))
        return {"bytes": sum(held(l) for l in lens if l) + 2 * b * case["tokens"] * nq * hd * 2,
                "flops": 4 * hd * nq * pairs}
    if kind == "append":
        n, rows = sum(_counts(case)), b * case["tokens"]
        return {"bytes": nkv * hd * (n * 4 + n * 2 + rows * 4), "flops": 4 * n * nkv * hd}
    keep = [min(l, case["keep"]) for l in lens]
    return {"bytes": nkv * sum(4 * l for l in lens) + sum(2 * held(k) for k in keep)
            + nkv * b * case["keep"] * (hd * 4 + 8), "flops": 4 * sum(keep) * nkv * hd}


# ---------------------------------------------------------------- exact ----
def _exact_rows(s, n, b, length):
    """One sequence's keys or values [nkv][length][hd] in 64 bits."""
    done = max(0, length - 1) // BLOCK * BLOCK
    step = s[n + "_scales"][b, :, : done // BLOCK].double().repeat_interleave(BLOCK, dim=1)
    coded = (s[n + "_codes"][b, :, :done].double() - 128.0) * step[..., None]
    return torch.cat([coded, s[n + "_tail"][b, :, : length - done].double()], dim=1)


def exact(case, seed):
    """What run() returns, from the definitions in 64 bits, one sequence after another."""
    s = prepare(case, seed)
    if case["kind"] == "score":
        parts = {"logprob": [], "entropy": [], "top_ids": [], "top_logprobs": []}
        few = max(1, 40_000_000 // case["vocab"])
        for r in range(0, case["rows"], few):
            lp = torch.log_softmax(s["logits"][r:r + few].double(), 1)
            parts["logprob"].append(lp.gather(1, s["tokens"][r:r + few].long()[:, None])[:, 0])
            parts["entropy"].append(-(lp.exp() * lp).sum(1))
            got = torch.sort(lp, dim=1, descending=True, stable=True)
            parts["top_ids"].append(got.indices[:, : case["top"]].int())
            parts["top_logprobs"].append(got.values[:, : case["top"]])
        return {n: torch.cat(v) for n, v in parts.items()}
    lens, hd = _lens(case), case["head_dim"]
    if case["kind"] in ("decode", "prompt"):
        nq, nkv = case["q_heads"], case["kv_heads"]
        q = s["q"].double() if case["kind"] == "prompt" else s["q"].double()[:, None]
        out = torch.zeros(q.shape, device=DEV, dtype=torch.float64)
        weights = s["weights"].double() if "weights" in s else None
        counts = _counts(case) if case["kind"] == "prompt" else [1] * len(lens)
        for b, (l, c) in enumerate(zip(lens, counts)):
            if not c:
                continue
            k, v = (_exact_rows(s, n, b, l) for n in "kv")
            if case["kind"] == "decode":
                # the token itself; a block that it does not open is still in the tail, the block before in codes
                if l and l % BLOCK == 0:
                    k, v = (torch.cat([x[:, : l - BLOCK], (s[n + "_codes"][b, :, l - BLOCK:l].double() - 128.0)
                                       * s[n + "_scales"][b, :, l // BLOCK - 1, None, None].double()], dim=1)
                            for x, n in ((k, "k"), (v, "v")))
                k, v = (torch.cat([x, s[n][b, :, None].double()], dim=1) for x, n in ((k, "k"), (v, "v")))
            total = k.shape[1]
            late = torch.arange(total, device=DEV)[None] > torch.arange(total - c, total, device=DEV)[:, None]
            for h in range(nq):
                g = h // (nq // nkv)
                p = torch.softmax((q[b, :c, h] @ k[g].T / math.sqrt(hd)).masked_fill(late, -math.inf), -1)
                out[b, :c, h] = p @ v[g]
                if weights is not None:
                    weights[b, g, :total] += p[0]
        if case["kind"] == "prompt":
            return {"out": out}
        return {"out": out[:, 0], "k_tail": None, "v_tail": None, "k_scales": None, "v_scales": None,
                "weights": weights}
    if case["kind"] == "append":
        shape = s["k"].shape
        got = {"k": torch.zeros(shape, device=DEV, dtype=torch.float64),
               "v": torch.zeros(shape, device=DEV, dtype=torch.float64)}
        for n in "kv":
            for b, (l, c) in enumerate(zip(lens, _counts(case))):
                x = s[n][b, :c].double()
                held = (l - c) % BLOCK
                x = torch.cat([s[n + "_tail"][b, :, :held].double().transpose(0, 1), x])
                for at in range(0, max(0, len(x) - 1) // BLOCK * BLOCK, BLOCK):
                    step = x[at:at + BLOCK].abs().amax((0, 2), keepdim=True) / 127.0
                    x[at:at + BLOCK] = torch.round(x[at:at + BLOCK] / step) * step
                got[n][b, :c] = x[held:]
        return {**got, "k_tail": None, "v_tail": None, "k_scales": None, "v_scales": None}
    # eviction: the kept tokens' values, block by block
    keep, nkv = case["keep"], case["kv_heads"]
    got = {n: torch.zeros(case["batch"], keep, nkv, hd, device=DEV, dtype=torch.float64) for n in "kv"}
    weights = torch.zeros(s["into_weights"].shape, device=DEV, dtype=torch.float64)
    for b, l in enumerate(lens):
        rows = {n: _exact_rows(s, n, b, l).half().double() for n in "kv"}    # the new cache is made of FP16 values
        m = min(l, keep)
        for h in range(nkv):
            w = s["weights"][b, h, :l].double()
            if m < l:
                w[: case["sinks"]] = math.inf
                w[l - case["recent"]:] = math.inf
                left = torch.sort(torch.sort(w, descending=True, stable=True).indices[:m]).values
            else:
                left = torch.arange(l, device=DEV)
            weights[b, h, :m] = s["weights"][b, h, left].double()
            for n in "kv":
                x = rows[n][h][left]
                for at in range(0, max(0, m - 1) // BLOCK * BLOCK, BLOCK):
                    f, e = int(left[at]), int(left[at + BLOCK - 1])
                    if f % BLOCK == 0 and e - f == BLOCK - 1 and f // BLOCK != (l - 1) // BLOCK:
                        continue
                    step = x[at:at + BLOCK].abs().max() / 127.0
                    x[at:at + BLOCK] = torch.round(x[at:at + BLOCK] / step) * step
                got[n][b, :m, h] = x
    return {"lens": None, "kept": None, **got, "weights": weights, "k_scales": None, "v_scales": None}
