"""Paged caches for the tests of the device-tensor operators, and the operators' definitions in 64 bits."""
import math

import torch

F64 = torch.float64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def unit(t):
    """a rounding to type t is off by at most this, relative"""
    return torch.finfo(TYPES[t]).eps / 2


class Cache:
    """Pages in random order: a shared prefix and every sequence's own tokens; what no token owns is NaN."""

    def __init__(self, seed, n_kv, dim, page, typ, prefix, own, spare=0, device="cuda", extra=2):
        self.g = torch.Generator(device="cpu")
        self.g.manual_seed(seed)
        self.n_kv, self.dim, self.page, self.typ, self.prefix, self.own, self.device = n_kv, dim, page, typ, prefix, list(own), device
        n_prefix = -(-prefix // page)
        n_own = [-(-(o + spare) // page) for o in own]
        n = n_prefix + sum(n_own) + extra
        order = torch.randperm(n, generator=self.g).to(torch.int32)
        self.prefix_pages = order[:max(1, n_prefix)].clone().to(device)
        table = torch.full((len(own), max([1] + n_own) + 1), 10 ** 6, dtype=torch.int32)      # ids that nobody may follow
        at = n_prefix
        for s, c in enumerate(n_own):
            table[s, :c] = order[at:at + c]
            at += c
        self.pages = table.to(device)
        self.k = torch.full((n, n_kv, page, dim), math.nan, dtype=TYPES[typ])
        self.v = self.k.clone()
        for pages, count in [(order[:n_prefix], prefix)] + [(table[s], o) for s, o in enumerate(own)]:
            for j0 in range(0, count, page):
                c = min(page, count - j0)
                for pool in (self.k, self.v):
                    pool[pages[j0 // page].item(), :, :c] = torch.randn(n_kv, c, dim, generator=self.g).to(TYPES[typ])
        self.k, self.v = self.k.to(device), self.v.to(device)

    def ints(self, values):
        return torch.tensor(list(values), dtype=torch.int32, device=self.device)

    def tokens(self, pool, pages, n):
        """[kv heads, n, dim] in 64 bits"""
        c = -(-n // self.page)
        return pool[pages[:c].long()].to(F64).transpose(0, 1).reshape(self.n_kv, c * self.page, self.dim)[:, :n]


def attention_exact(cache, q, prefix, rows, scale=None):
    """out, sum of weight * |value|, largest scale * sum |q_d k_d| of a row: all [rows, heads, ...]"""
    R, H, D = q.shape
    G = H // cache.n_kv
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(R, H, D, dtype=F64, device=q.device)
    spread, reach = out.clone(), torch.zeros(R, H, dtype=F64, device=q.device)
    kp, vp = (cache.tokens(p, cache.prefix_pages, prefix) for p in (cache.k, cache.v))
    r0 = 0
    for s, (n, o) in enumerate(zip(rows, cache.own)):
        k, v = (torch.cat([a, cache.tokens(p, cache.pages[s], o)], 1) for a, p in ((kp, cache.k), (vp, cache.v)))
        for i in range(n):
            seen = prefix + max(0, o - n + i + 1)
            if seen == 0:
                continue
            x = q[r0 + i].to(F64).view(cache.n_kv, G, D)
            w = torch.softmax(x @ k[:, :seen].transpose(1, 2) * scale, -1)
            out[r0 + i] = (w @ v[:, :seen]).reshape(H, D)
            spread[r0 + i] = (w @ v[:, :seen].abs()).reshape(H, D)
            reach[r0 + i] = (x.abs() @ k[:, :seen].abs().transpose(1, 2)).amax(-1).reshape(H) * scale
        r0 += n
    return out, spread, reach


def attention_bar(typ, out, spread, reach, dim):
    """One rounding of the output, one of every probability (numerator alone), 32-bit scores: a dot product of dim terms is off by dim 2^-24 sum |q_d k_d|, the
    scaling and the difference to the maximum by 2^-23 of it, and weights change by that much relative, in numerator and denominator; 2^-18 for the
    exponential's 2^-22 and for sums over some ten partial results of up to 32 terms a lane."""
    u = unit(typ)
    return u * out.abs() + (u + 2 * (dim + 4) * 2 ** -24 * reach[..., None] + 2 ** -18) * spread + 2 ** -24


def rotated(x, positions, freqs, layout, amplitude=1.0):
    """[rows, heads, dim] in 64 bits"""
    x = x.to(F64)
    rot = 2 * len(freqs)
    angle = positions.to(F64)[:, None] * freqs.to(F64)[None]
    c, s = (amplitude * angle.cos())[:, None], (amplitude * angle.sin())[:, None]
    y = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if layout == "pairs" else (x[..., :rot // 2], x[..., rot // 2:rot])
    if layout == "pairs":
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, a * s + b * c
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, a * s + b * c
    return y


def logprobs_exact(logits, tokens, top):
    x = logits.to(F64)
    lp = x - torch.logsumexp(x, 1, keepdim=True)
    entropy = -torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(1)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return lp.gather(1, tokens.long()[:, None])[:, 0], entropy, lp.gather(1, ids), ids
