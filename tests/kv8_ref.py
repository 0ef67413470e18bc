"""Plain restatement of the 8-bit KV cache and its operators, in 64 bits on the
CPU (quantisation in float32, where the definition is: its divisions and
roundings are the IEEE ones)."""
from __future__ import annotations

import math

import torch

BLOCK = 64


def rope_fp16(x, c, s):
    half = x.shape[-1] // 2
    rot = torch.cat([-x[..., half:], x[..., :half]], dim=-1)
    return (x * c) + (rot * s)


def quantise(block):
    """[64, hd] FP16 -> (uint8 codes, float32 scale)."""
    x = torch.nan_to_num(block.float(), nan=0.0, posinf=65504.0, neginf=-65504.0)
    scale = x.abs().max() / torch.tensor(127.0)
    if scale == 0:
        return torch.full(x.shape, 128, dtype=torch.uint8), scale
    return (torch.round(x / scale) + 128).to(torch.uint8), scale


class RefCache:
    """One head's side (keys or values) of one sequence."""

    def __init__(self, hd):
        self.hd, self.codes, self.scales = hd, [], []
        self.rows = torch.zeros(0, hd, dtype=torch.float16)    # rows of the last block
        self.len = 0

    def append(self, x):
        for row in x:
            if len(self.rows) == BLOCK:
                self.rows = self.rows[:0]
            self.rows = torch.cat([self.rows, row[None]])
            self.len += 1
            if len(self.rows) == BLOCK:
                c, s = quantise(self.rows)
                self.codes.append(c)
                self.scales.append(s)

    def coded(self):
        """Whole blocks read as codes (not the last token's)."""
        return (self.len - 1) // BLOCK if self.len else 0

    def values(self):
        """[len, hd] float64."""
        done = [(c.double() - 128) * s.double() for c, s in zip(self.codes[:self.coded()], self.scales)]
        return torch.cat(done + [self.rows.double()])

    def restored(self):
        done = [((c.float() - 128) * s).half() for c, s in zip(self.codes[:self.coded()], self.scales)]
        return torch.cat(done + [self.rows])


class RefKV:
    def __init__(self, batch, heads, hd):
        self.s = [[[RefCache(hd) for _ in range(heads)] for _ in range(batch)] for _ in "kv"]

    def append(self, k, v, counts):
        for side, x in zip(self.s, (k.cpu(), v.cpu())):
            for b, c in enumerate(counts):
                for h, cache in enumerate(side[b]):
                    cache.append(x[b, :c, h])

    def lens(self):
        return [row[0].len for row in self.s[0]]


def attention(ref, q, counts, scale=None):
    """q [B, n, nq, hd] -> (out float64, probabilities of the last query [B][nkv][len])."""
    q = q.cpu().double()
    B, n, nq, hd = q.shape
    nkv = len(ref.s[0][0])
    out = torch.zeros_like(q)
    probs = []
    scale = 1 / math.sqrt(hd) if scale is None else scale
    for b in range(B):
        probs.append([])
        for g in range(nkv):
            k, v = ref.s[0][b][g].values(), ref.s[1][b][g].values()
            acc = torch.zeros(len(k), dtype=torch.float64)
            for i in range(counts[b]):
                end = len(k) - counts[b] + i + 1
                if end <= 0:
                    continue
                for h in range(g * nq // nkv, (g + 1) * nq // nkv):
                    p = torch.softmax(k[:end] @ q[b, i, h] * scale, 0)
                    out[b, i, h] = p @ v[:end]
                    if i == counts[b] - 1:
                        acc[:end] += p
            probs[-1].append(acc)
    return out, probs


def evict_positions(weights, length, keep, sinks, recent):
    """Old positions kept of one head, ascending."""
    if length <= keep:
        return list(range(length))
    forced = [t for t in range(length) if t < sinks or t >= length - recent]
    w = [math.inf if math.isnan(x) else x for x in weights[:length].tolist()]
    nan = [math.isnan(x) for x in weights[:length].tolist()]
    rest = sorted((t for t in range(length) if t not in set(forced)), key=lambda t: (not nan[t], -w[t], t))
    return sorted(forced + rest[:keep - len(forced)])


def evict_side(cache, kept):
    """The new cache of one head's side."""
    new = RefCache(cache.hd)
    x = cache.restored()
    new.append(x[torch.tensor(kept, dtype=torch.long)])
    for j in range(len(kept) // BLOCK):
        idx = kept[j * BLOCK:(j + 1) * BLOCK]
        if idx[0] % BLOCK == 0 and idx[-1] - idx[0] == BLOCK - 1 and idx[0] // BLOCK < cache.coded():
            new.codes[j], new.scales[j] = cache.codes[idx[0] // BLOCK], cache.scales[idx[0] // BLOCK]
    return new
