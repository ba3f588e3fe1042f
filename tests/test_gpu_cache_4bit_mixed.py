"""Attention over a paged cache in 4 bits on the GPU: calls that mix prompts with single tokens, numbers at the ends of their types, lengths past the tables."""
import math

import pytest

torch = pytest.importorskip("torch")

from cache_4bit_util import Cache4, attention_bar, attention_exact
from device_ops_util import F64, TYPES
from test_gpu_cache_4bit import attend, visible_nan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(native_lib):
    from llama_cpp import device_ops
    return device_ops


# Many units of at most 128 rows times heads of a KV head follow one another in a CTA of the kernel for many rows.
MIXED = [
    # heads, kv, dim, page, rows, tokens behind them, max_rows
    (32, 8, 128, 64, [100] + [1] * 255, [50] + [i * 7 % 40 for i in range(255)], 100),
    (32, 8, 64, 16, [1] * 200 + [100] + [1] * 55, [i * 13 % 300 for i in range(256)], 100),
    (32, 8, 128, 64, [1] * 256, [i * 11 % 90 for i in range(256)], None),             # a batched step whose max_rows is left open
    (64, 8, 64, 32, [2 + i * 5 % 15 for i in range(64)], [i * 17 % 120 for i in range(64)], 16),      # drafted tokens
    (32, 8, 128, 32, [20, 40, 1, 1, 33, 64, 2, 70, 1] * 20, [i * 19 % 150 for i in range(180)], 70),  # units of one tile and of two in turn
    (8, 1, 64, 16, [16] * 500, [i % 30 for i in range(500)], 16),                     # whole tiles of 128
]


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim,page,rows,behind,max_rows", MIXED)
def test_many_units_of_one_tile(ops, heads, kv, dim, page, rows, behind, max_rows, typ):
    """against the definition; a value or key that is no number reaches the rows that see it, in every one of these units"""
    own = [n + b for n, b in zip(rows, behind)]
    R, T = sum(rows), sum(own)
    g = torch.Generator().manual_seed(R)
    k, v = (torch.randn(T, kv, dim, generator=g).half() for _ in range(2))
    start = [sum(own[:s]) for s in range(len(own))]
    for s in range(0, len(own), 3):
        v[start[s] + own[s] // 2, s // 3 % kv, 5 * s % dim] = (math.nan, math.inf)[s & 1]
    c = Cache4(R, kv, dim, page, own, k=k, v=v, fill=0xff)
    q = torch.randn(R, heads, dim, generator=c.g).to(TYPES[typ]).cuda()
    got = attend(ops, c, q, rows, max_rows=R if max_rows is None else max_rows)
    assert ops.error(0) == 0
    want, sizes = visible_nan(c, q, rows, c.values(c.k), c.values(c.v))
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isnan(want).any()
    near = (got.to(F64) - want).abs() <= attention_bar(typ, torch.nan_to_num(want), *sizes, dim, True)
    assert (near | torch.isnan(want)).all()
    again = attend(ops, c, q, rows, max_rows=R if max_rows is None else max_rows)
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(again))


@pytest.mark.parametrize("dim", [64, 128])
def test_entries_past_f16_reach_the_rows_that_see_them(ops, dim):
    """f16 queries, more than 64 rows a KV head: a group with an entry past 65504 reads as NaN, for the rows that see its token and no others; entries of 65504 are numbers"""
    rows, heads = [60, 33, 100, 150], 16
    own = [n + 30 for n in rows]
    start = [sum(own[:s]) for s in range(len(own))]
    g = torch.Generator().manual_seed(dim)
    k, v = (torch.randn(sum(own), 2, dim, generator=g).bfloat16().float() for _ in range(2))
    v[start[1] - 1, 0, 5] = 1e5                                          # the last token of sequence 0
    v[start[1] + 40, 1, 40], v[start[1] + 40, 1, 3] = -3e38, 65504.0
    v[start[2] + 100, 0, 33:35] = 65536.0
    v[start[2] + 3, 1, 60] = 65504.0
    k[start[3] + 120, 1, 7] = 2e5
    k[start[3] + 130, 0, 7] = 65504.0
    c = Cache4(2, 2, dim, 16, own, k=k, v=v, fill=0xff)
    q = (torch.randn(sum(rows), heads, dim, generator=c.g)).half()
    q[..., 7] *= 1e-4
    q = q.cuda()
    keys, values = c.values(c.k), c.values(c.v)
    for x in (keys, values):
        groups = x.unflatten(-1, (-1, 32))
        groups[(groups.abs() > 65519.0).any(-1)] = math.nan
    got = attend(ops, c, q, rows)
    want, sizes = visible_nan(c, q, rows, keys, values)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and not torch.isinf(got).any() and torch.isnan(want).any()
    # (a row that sees a number is held to the bar of the numbers that it sees)
    seen = torch.nan_to_num(torch.stack(sizes_of_what_rows_see(c, q, rows, keys, values)))
    bar = attention_bar("f16", torch.nan_to_num(want), seen[0], seen[1], sizes[2], seen[2], dim, True)
    assert ((got.to(F64) - want).abs() <= bar)[~torch.isnan(want)].all() and ops.error(0) == 0


def sizes_of_what_rows_see(c, q, rows, k, v):
    """attention_exact's spread, offset and all_v with the groups that are no numbers left out"""
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    clean = Cache4.__new__(Cache4)
    clean.__dict__.update(c.__dict__)
    clean.k, clean.v = k.cpu().float(), v.cpu().float()
    _, spread, offset, _, all_v = attention_exact(clean, q, rows, k=k, v=v)
    return spread, offset, all_v


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,n", [(8, 1), (64, 2)])
def test_one_token_comes_back(ops, heads, n, dim, typ):
    """a row that sees one token has that token's value, scale * (code - 8) rounded once, whichever way it goes"""
    kv = 8
    c = Cache4(dim + heads, kv, dim, 16, [n] * 40)
    q = torch.randn(40 * n, heads, dim, generator=c.g).to(TYPES[typ]).cuda()
    got = attend(ops, c, q, [n] * 40, max_rows=n if n == 1 else 40 * n)
    want = c.values(c.v)[::n].float().to(TYPES[typ])                     # (15 bits: exact in 32)
    assert torch.equal(got[::n], want.repeat_interleave(heads // kv, 1))


@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_scores_of_many_rows_are_exact_products(ops, typ):
    """keys whose scales have all their 11 bits, queries of one entry: scores are scale * (code - 8) * query to the bits of 32, weights what they say"""
    rows, heads, dim = [40, 30], 8, 64
    own = [n + 60 for n in rows]
    T = sum(own)
    s = 1 + (33 + 2 * (torch.arange(T) % 16)).float() / 1024             # 11 bits, the last one set
    k = torch.zeros(T, 2, dim)
    k[:, :, 3], k[:, :, 5] = -8 * s[:, None], 7 * s[:, None]             # codes 0 and 15
    c = Cache4(12, 2, dim, 16, own, k=k)
    q = torch.zeros(sum(rows), heads, dim)
    q[..., 5] = 1.0 + torch.arange(heads) / 8
    q = q.to(TYPES[typ]).cuda()
    got = attend(ops, c, q, rows, scale=64.0)
    want, spread, offset, reach, all_v = attention_exact(c, q, rows, scale=64.0)
    # one product and one sum in 32 bits, both exact, the difference to the row's largest times the scale: 2^-22 of it
    reach = 7 * 2 * 64.0 * 2 * torch.ones_like(reach) * 2 ** -22 / (4 * (dim + 16) * 2 ** -24)
    assert ((got.to(F64) - want).abs() <= attention_bar(typ, want, spread, offset, reach, all_v, dim, True)).all()


@pytest.mark.parametrize("at", [0, 99980])
def test_many_small_weights(ops, at):
    """one key has the row's largest score by far, 100000 others share what is left: 2^-25.02 of its weight each, 0.3 % together. A weight may be off by 2^-31 of the largest one's and by a
    rounding of itself, all of them together by 2^-14. As many sequences as a CTA needs to have most of one's keys, all with the same pages."""
    n, kv, seqs = 100000, 8, 20
    k, v = torch.zeros(n, kv, 64), torch.ones(n, kv, 64)
    k[at, :, 0], v[at] = 17.34375, 0.0                                   # 25.02 ln 2
    c = Cache4(13, kv, 64, 64, [n], k=k, v=v)
    one, many = c.pages, c.pages.expand(seqs, -1).contiguous()
    q = torch.zeros(9, 8 * kv, 64)
    q[..., 0] = 1.0
    for rows in (1, 9):
        x = q[:rows].cuda()
        c.pages = one
        want, spread, *_ = attention_exact(c, x, [rows], scale=1.0)
        assert (want / (n * math.exp(-17.34375)) - 1).abs().max() < 0.01
        c.pages = many
        for typ in ("f16", "bf16"):
            got = attend(ops, c, x.to(TYPES[typ]).repeat(seqs, 1, 1), [rows] * seqs, scale=1.0, own=[n] * seqs)
            # (sums and scores in 32 bits: 2^-14 as elsewhere)
            unit = torch.finfo(TYPES[typ]).eps / 2
            off = (got.view(seqs, *x.shape).to(F64) - want).abs()
            assert (off <= unit * want + (unit + 2 ** -14) * spread + (2 ** -14 if typ == "f16" else 0)).all(), (rows, typ, float(got.min()), float(want.min()))


@pytest.mark.parametrize("heads,rows", [(4, [1]), (32, [1]), (16, [9])])
@pytest.mark.parametrize("first,second", [(5, 2985), (2985, 5), (1000, 1040), (700, 2000), (40, 200)])
@pytest.mark.parametrize("of", [0, 3, 5])
def test_large_scores_in_different_partial_results(ops, heads, rows, first, second, of):
    """two keys with scores of 2^22 and more, one apart, wherever partial results of the keys are cut: weights of 1 and e"""
    n = sum(rows)
    own, dim = [3000 + n], 64
    k, v = torch.zeros(own[0], 2, dim), torch.zeros(own[0], 2, dim)
    k[[first, second], :, 0] = 2048.0
    k[second, :, 40] = 1.0
    v[first], v[second] = 1.0, -1.0
    c = Cache4(14, 2, dim, 64, own, k=k, v=v)
    q = torch.zeros(n, heads, dim)
    q[..., 0], q[..., 40] = 2048.0 * (1 + of / 8), 1.0
    q = q.half().cuda()
    got = attend(ops, c, q, rows, scale=1.0)
    want = (1 - math.e) / (1 + math.e)
    assert ((got.to(F64) - want).abs() <= 2 ** -9).all(), float(got[0, 0, 0])


@pytest.mark.parametrize("heads,rows", [(4, [1, 1]), (16, [9, 12])])
def test_large_queries_and_scale(ops, heads, rows):
    """queries of 2^100 and a scale of 2^20, scores that 32 bits hold: all weight on the largest"""
    own = [200 + n for n in rows]
    T = sum(own)
    k = torch.zeros(T, 2, 64)
    k[:, :, 9] = 8.0
    k[:, :, 3] = (torch.arange(T) % 15 - 7).float()[:, None]             # codes 1 .. 15
    c = Cache4(15, 2, 64, 16, own, k=k)
    q = torch.zeros(sum(rows), heads, 64)
    q[..., 3] = 2.0 ** 100
    q = q.bfloat16().cuda()
    got = attend(ops, c, q, rows, scale=2.0 ** 20)
    want, *_ = attention_exact(c, q, rows, scale=2.0 ** 20)
    _, spread, *_ = attention_exact(c, q, rows, scale=2.0 ** 20)
    assert ((got.to(F64) - want).abs() <= 2 ** -9 * want.abs() + (2 ** -9 + 2 ** -10) * spread + 2 ** -20).all()


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("heads,rows", [(4, [1, 1, 1]), (16, [2, 9, 5]), (16, [60, 33, 100])])
def test_lengths_past_the_tables(ops, heads, rows, typ):
    """lengths past the table mean all that it holds, to the bit and by the definition"""
    full = [208] * 3
    c = Cache4(16, 2, 64, 16, full, "bf16")
    c.pages = c.pages[:, :13].contiguous()
    q = torch.randn(sum(rows), heads, 64, generator=c.g).to(TYPES[typ]).cuda()
    held = attend(ops, c, q, rows)
    assert torch.isfinite(held).all()
    want, *sizes = attention_exact(c, q, rows)
    assert ((held.to(F64) - want).abs() <= attention_bar(typ, want, *sizes, 64, max(rows) * heads // 2 > 64)).all()
    for lengths in ([2 ** 31 - 1, 209, 10 ** 9], [224, 2 ** 31 - 1, 208]):
        assert torch.equal(attend(ops, c, q, rows, own=lengths), held)


@pytest.mark.parametrize("heads,rows", [(4, [1, 1, 1]), (16, [2, 9, 5]), (16, [60, 33, 100])])
def test_page_ids_outside_the_pool(ops, heads, rows):
    """they are held inside it: the first page and the last, to the bit and by the definition"""
    own = [n + 20 for n in rows]
    c = Cache4(17, 2, 64, 16, own, fill=0)
    q = torch.randn(sum(rows), heads, 64, generator=c.g).half().cuda()
    held = c.pages.clone()
    held[0, 0], held[1, 0], held[2, 0] = 0, len(c.bytes_k) - 1, 0
    c.pages = held
    inside = attend(ops, c, q, rows)
    assert torch.isfinite(inside).all() and inside.abs().sum() > 0
    c.pages = held.clone()
    c.pages[0, 0], c.pages[1, 0], c.pages[2, 0] = -5, 2 ** 31 - 1, -2 ** 31
    assert torch.equal(attend(ops, c, q, rows), inside)


@pytest.mark.parametrize("seqs", [1, 40])
def test_queries_of_rows_far_ahead_of_their_tokens(ops, seqs):
    """rows without a place are rotated by their position all the same, whatever the length: one below -2^31 does not wrap"""
    c = Cache4(18, 2, 64, 16, [16] * seqs)
    n = 5
    x = torch.randn(n * seqs, 2, 64, generator=c.g).cuda()
    freqs = (2.0 ** (-28 - torch.arange(32) / 8)).float().cuda()
    pos = (torch.arange(n) - n - 2 ** 31).repeat(seqs).cuda()
    outs = []
    for first in (0, 2 ** 33):
        q_out = torch.zeros(n * seqs, 2, 64, dtype=torch.float16, device="cuda")
        ops.kv_append_4bit(x, x, c.k_pool, c.v_pool, c.pages, c.ints(range(0, n * seqs + 1, n)), c.ints([-2 ** 31] * seqs), q=x, q_out=q_out, freqs=freqs, first_pos=first)
        angle = (pos + first).to(F64)[:, None] * freqs.to(F64)
        cos, sin = angle.cos()[:, None], angle.sin()[:, None]
        a, b = x[..., 0::2].to(F64), x[..., 1::2].to(F64)
        want = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        assert ((q_out.to(F64) - want).abs() <= 2 ** -11 * want.abs() + 2 ** -20).all()
        outs.append(q_out)
    assert torch.equal(c.k_pool.cpu(), c.bytes_k) and not torch.equal(*outs)
