"""A paged cache in 4 bits for the tests: its definition in 64 bits, its bytes restated, and attention over it in 64 bits."""
import math

import torch

from device_ops_util import F64, TYPES, unit

GROUP = 32


def quantised(x):
    """codes [..., dim] (whole numbers 0 .. 15) and scales [..., dim / 32] (f16) of rows, by the definition in 64 bits"""
    y = x.to(F64).unflatten(-1, (-1, GROUP))
    bad = ~torch.isfinite(y).all(-1)
    y = torch.where(bad[..., None], 0.0, y)
    high, low = y.amax(-1), y.amin(-1)
    m = torch.where(high > -low, high, low)
    # (to f16 by way of 32 bits: entries have no more than those)
    s = (-m / 8).clamp(-65504.0, 65504.0).float().half()
    s = torch.where(s == 0, torch.zeros_like(s), s)               # (no negative zero)
    d = s.to(F64)[..., None]
    c = torch.where(d == 0, 8.0, (torch.round(y / torch.where(d == 0, 1.0, d)) + 8).clamp(0, 15))
    s = torch.where(bad, torch.full_like(s, 0x7fff, dtype=torch.int16).view(torch.float16), s)
    return c.flatten(-2).to(torch.uint8), s


def values(codes, scales):
    return ((codes.to(F64) - 8).unflatten(-1, (-1, GROUP)) * scales.to(F64)[..., None]).flatten(-2)


def coded(x):
    """what the cache gives back, in 64 bits"""
    return values(*quantised(x))


def places(D, keys):
    """byte of a block's codes [16, dim / 2] and 16-bit place of its scales [16, dim / 32], token by token"""
    n = D // GROUP
    t, j = torch.arange(16)[:, None], torch.arange(D // 2)[None]
    if keys:                         # four bytes a word, a row a token
        word = j // 4
        chunk = (word % 4) ^ ((t // 2) % 4 if D == 128 else (t // 4) % 2 * 2)
        codes = t * (D // 2) + 4 * (chunk * n + word // 4) + j % 4
    else:                            # two bytes a half of a word, a row two tokens
        half = j // 2
        chunk = (half % 8) ^ ((t // 2) % 4 * 2 if D == 128 else (t // 4) % 2 * 4)
        codes = t // 2 * D + 4 * (chunk * n + half // 8) + t % 2 * 2 + j % 2
    return codes, t * n + torch.arange(n)[None]


def packed(codes, scales, keys):
    """[..., 16 tokens, dim] codes and [..., 16, dim / 32] scales as blocks of 9 * dim bytes"""
    codes, scales = codes.cpu(), scales.cpu()
    D = codes.shape[-1]
    at, place = places(D, keys)
    out = torch.zeros(*codes.shape[:-2], 9 * D, dtype=torch.uint8)
    halves = torch.zeros(*codes.shape[:-2], D // 2, dtype=torch.float16)
    out[..., at] = codes[..., 0::2] + 16 * codes[..., 1::2]
    halves[..., place] = scales
    out[..., 8 * D:] = halves.view(torch.uint8)
    return out


def token_of_byte(D, keys):
    """whose token's a block's bytes are"""
    at, place = places(D, keys)
    out = torch.zeros(9 * D, dtype=torch.long)
    out[at] = torch.arange(16)[:, None].expand(at.shape)
    for b in range(2):
        out[8 * D + 2 * place + b] = torch.arange(16)[:, None].expand(place.shape)
    return out


class Cache4:
    """Pages in random order that hold `own` tokens of every sequence, `k` and `v` rows token by token; the other bytes are random or `fill`."""

    def __init__(self, seed, n_kv, dim, page, own, typ="f16", device="cuda", extra=2, spare=0, k=None, v=None, fill=None):
        self.g = torch.Generator(device="cpu")
        self.g.manual_seed(seed)
        self.n_kv, self.dim, self.page, self.own, self.device = n_kv, dim, page, list(own), device
        n_own = [-(-(o + spare) // page) for o in own]
        n = sum(n_own) + extra
        order = torch.randperm(n, generator=self.g).to(torch.int32)
        table = torch.full((len(own), max([1] + n_own) + 1), 10 ** 6, dtype=torch.int32)       # ids that nobody may follow
        at = 0
        for s, c in enumerate(n_own):
            table[s, :c] = order[at:at + c]
            at += c
        self.table = table
        self.pages = table.to(device)
        self.start = [0]
        for o in own:
            self.start.append(self.start[-1] + o)
        T = self.start[-1]
        # some entries of a head much larger than the others, as keys have them
        large = 1.0 + 6.0 * (torch.rand(n_kv, dim, generator=self.g) < 0.05)
        self.k = (torch.randn(T, n_kv, dim, generator=self.g) * large).to(TYPES[typ]) if k is None else k
        self.v = torch.randn(T, n_kv, dim, generator=self.g).to(TYPES[typ]) if v is None else v
        self.bytes_k, self.bytes_v = self.expect(n, self.k, True, fill), self.expect(n, self.v, False, fill)
        self.k_pool, self.v_pool = self.bytes_k.to(device), self.bytes_v.to(device)

    def ints(self, values):
        return torch.tensor(list(values), dtype=torch.int32, device=self.device)

    def expect(self, n_pages, rows, keys, fill=None, base=None):
        """the pool's bytes: packed rows over `base`, random bytes or `fill`"""
        D, G, page = self.dim, self.n_kv, self.page
        pool = torch.randint(0, 256, (n_pages, G, page // 16, 9 * D), dtype=torch.uint8, generator=self.g) if base is None else base.clone()
        if fill is not None:
            pool.fill_(fill)
        codes, scales = (x.cpu() for x in quantised(rows))
        first = [(s, b) for s, o in enumerate(self.own) for b in range(-(-o // 16))]
        if not first:
            return pool
        seq, block = (torch.tensor(x) for x in zip(*first))
        own, start = torch.tensor(self.own), torch.tensor(self.start)
        token = 16 * block[:, None] + torch.arange(16)                                        # [blocks, 16]
        here = token < own[seq][:, None]
        row = torch.where(here, start[seq][:, None] + token, 0)
        blocks = packed(codes[row].transpose(1, 2), scales[row].transpose(1, 2), keys)        # [blocks, kv heads, bytes]
        at = self.table[seq, 16 * block // page].long(), slice(None), block % (page // 16)
        pool[at] = torch.where(here[:, token_of_byte(D, keys)][:, None], blocks, pool[at])
        return pool

    def values(self, rows):
        return coded(rows).to(self.device)


def attention_exact(c, q, rows, scale=None, max_rows=None, k=None, v=None):
    """out; sum of weight * |value|; the same of 8 |scale of the value's group|; scale * sum over d of |q_d| 8 |scale of the key's group|, the largest of a row; sum over the keys that a row
    sees of |value| and an eighth of the head's largest scale"""
    R, H, D = q.shape
    G = H // c.n_kv
    scale = D ** -0.5 if scale is None else scale
    k, v = c.values(c.k) if k is None else k, c.values(c.v) if v is None else v
    steps, steps_v = (8 * torch.nan_to_num(quantised(x)[1].to(F64).abs()).repeat_interleave(GROUP, -1).to(c.device) for x in (c.k, c.v))
    least = torch.nan_to_num(quantised(c.v)[1].to(F64).abs()).amax(-1).to(c.device) / 8
    out = torch.zeros(R, H, D, dtype=F64, device=q.device)
    spread, offset, all_v, reach = out.clone(), out.clone(), out.clone(), torch.zeros(R, H, dtype=F64, device=q.device)
    r0 = 0
    for s, (n, o) in enumerate(zip(rows, c.own)):
        ks, vs, st, sv = (x[c.start[s]:c.start[s] + o].transpose(0, 1) for x in (k, v, steps, steps_v))
        seen = o - n + 1 + torch.arange(n, device=q.device)
        if max_rows is not None:
            seen[max_rows:] = 0
        if n and o:
            x = q[r0:r0 + n].to(F64).view(n, c.n_kv, G, D)
            mask = torch.arange(o, device=q.device) < seen[:, None]                           # [rows, tokens]
            score = (x @ ks.transpose(1, 2) * scale).masked_fill(~mask[:, None, None], -math.inf)
            w = torch.nan_to_num(torch.softmax(score, -1)) if (seen <= 0).any() else torch.softmax(score, -1)
            out[r0:r0 + n] = (w @ vs).reshape(n, H, D)
            spread[r0:r0 + n] = (w @ vs.abs()).reshape(n, H, D)
            offset[r0:r0 + n] = (w @ sv).reshape(n, H, D)
            each = vs.abs() + least[c.start[s]:c.start[s] + o].amax(0)[:, None, None]
            all_v[r0:r0 + n] = (mask.to(F64)[:, None, None] @ each).expand(n, c.n_kv, G, D).reshape(n, H, D)
            reach[r0:r0 + n] = (x.abs() @ st.transpose(1, 2)).masked_fill(~mask[:, None, None], 0.0).amax(-1).reshape(n, H) * scale
        r0 += n
    return out, spread, offset, reach, all_v


def attention_bar(typ, out, spread, offset, reach, all_v, dim, many=False):
    """One rounding of the output. Probabilities and values, or their scales, are rounded to f16, twice at most; with
    many rows of a sequence a KV head (`many`) probabilities are rounded to the queries' type and values are not. A score is a sum of dim products and of one offset a group, none
    larger together than |q| 8 |scale|, in 32 bits that a matrix instruction may cut off instead of rounding: within 2 (dim + 16) 2^-24 of it; weights change by that much relative,
    in numerator and denominator. 2^-18 for the exponential's 2^-22 and for joins. The smallest f16 numbers are 2^-24 apart: a weight, relative to one that is at least 1, may be off by half of
    that, and so may one times its value's scale where the largest scale is held to 64 or more: 8 / 64 of it an entry.
    Codes are multiplied without their offset of 8, which is taken off the sum: per 16 keys two instructions of 17 addends that may each be cut off at 2^-23 of the largest, at most 15 / 8 of
    a weight times 8 |scale|: within 2^-17 of the weighted sum of 8 |scale|."""
    u16 = unit("f16")
    return unit(typ) * out.abs() + ((unit(typ) + 2 ** -14 if many else 2 * u16) + 4 * (dim + 16) * 2 ** -24 * reach[..., None] + 2 ** -18) * spread + 2 ** -17 * offset + 2 ** -25 * all_v + 2 ** -24
