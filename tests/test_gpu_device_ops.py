"""The operators over device tensors against their definitions in 64 bits: paged appends with rotation, attention over a shared prefix, log probabilities."""
import math

import pytest

torch = pytest.importorskip("torch")

from device_ops_util import F64, TYPES, Cache, attention_bar, attention_exact, logprobs_exact, rotated, unit

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(native_lib):
    from llama_cpp import device_ops
    return device_ops


def starts(rows):
    out = [0]
    for r in rows:
        out.append(out[-1] + r)
    return out


# ------------------------------------------------------------------------------------------------------------------ append
def append_bar(typ, want, x, freqs, layout, amplitude=1.0):
    """One rounding to the cache's type (half the smallest f16 step at the bottom); before it an angle rounded to 32 bits of a half turn and sine and cosine to 2 of
    their units (4e-7 together), two products and a sum (3 roundings of 2^-24): within 1e-6 of |a| + |b|."""
    x = x.to(F64).abs()
    rot = 2 * len(freqs)
    size = x.clone()
    if layout == "pairs":
        both = x[..., 0:rot:2] + x[..., 1:rot:2]
        size[..., 0:rot:2], size[..., 1:rot:2] = both, both
    else:
        both = x[..., :rot // 2] + x[..., rot // 2:rot]
        size[..., :rot // 2], size[..., rot // 2:rot] = both, both
    return unit(typ) * want.abs() + 1e-6 * max(1.0, amplitude) * size + (2 ** -25 if typ == "f16" else 0)


APPENDS = [
    # heads, kv, dim, page, rot, rows, tokens behind, first position, input, cache, layout, joint projection
    (32, 8, 128, 64, 128, [1] * 5, [0, 63, 64, 127, 700], 0, "f32", "f16", "pairs", False),
    (32, 4, 64, 16, 64, [3, 0, 17, 1, 40, 0], [5, 0, 15, 16, 0, 9], 1000, "bf16", "bf16", "halves", True),
    (8, 8, 128, 48, 64, [100, 1, 350], [7, 1, 47], 131071, "f16", "bf16", "halves", True),
    (12, 2, 128, 32, 96, [900], [31], 0, "f16", "f16", "pairs", True),
    (5, 5, 80, 16, 20, [2, 33], [0, 16], 3, "f32", "bf16", "pairs", False),        # two entries at a time
    (3, 1, 36, 16, 36, [4, 700], [1, 0], 77, "bf16", "f16", "halves", False),      # one entry at a time
    (4, 2, 64, 64, 0, [3, 2], [0, 5], 0, "f16", "f16", "pairs", False),            # no rotation at all
]


@pytest.mark.parametrize("heads,kv,dim,page,rot,rows,behind,first,typ,cache_typ,layout,joint", APPENDS)
def test_append(ops, heads, kv, dim, page, rot, rows, behind, first, typ, cache_typ, layout, joint):
    held = [r + b for r, b in zip(rows, behind)]
    c = Cache(len(rows) + dim, kv, dim, page, cache_typ, 0, held)
    R = sum(rows)
    x = torch.randn(R, (heads + 2 * kv) * dim, generator=c.g).to(TYPES[typ]).cuda()
    q, k, v = x[:, :heads * dim].view(R, heads, dim), x[:, heads * dim:(heads + kv) * dim].view(R, kv, dim), x[:, (heads + kv) * dim:].view(R, kv, dim)
    if not joint:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    freqs = (10000.0 ** (-torch.arange(0, rot, 2, dtype=F64) / max(rot, 1))).float().cuda()
    k0, v0 = c.k.clone(), c.v.clone()
    q_out = torch.full((R, heads, dim), math.nan, dtype=TYPES[cache_typ], device="cuda")
    ops.kv_append(k, v, c.k, c.v, c.pages, c.ints(starts(rows)), c.ints(held), q=q, q_out=q_out, freqs=freqs if rot else None, layout=layout, first_pos=first)
    torch.cuda.synchronize()
    pos = torch.cat([torch.arange(b, b + r) for r, b in zip(rows, behind)]).cuda()
    want_q, want_k = rotated(q, pos + first, freqs, layout), rotated(k, pos + first, freqs, layout)
    assert ((q_out.to(F64) - want_q).abs() <= append_bar(cache_typ, want_q, q, freqs, layout)).all()
    seq = torch.cat([torch.full((r,), s) for s, r in enumerate(rows)]).cuda()
    page_of, off = c.pages[seq, pos // page].long(), pos % page
    assert ((c.k[page_of, :, off].to(F64) - want_k).abs() <= append_bar(cache_typ, want_k, k, freqs, layout)).all()
    assert torch.equal(c.v[page_of, :, off], v.float().to(TYPES[cache_typ]))
    k0[page_of, :, off], v0[page_of, :, off] = c.k[page_of, :, off], c.v[page_of, :, off]
    for got, was in ((c.k, k0), (c.v, v0)):            # nothing else was touched
        assert torch.equal(got.view(torch.int16), was.view(torch.int16))


def test_append_far_positions_and_amplitude(ops):
    """positions past 2^24 and a rotation that also scales: the product of position and frequency is a 64-bit one"""
    c = Cache(3, 2, 64, 16, "bf16", 0, [40])
    x = torch.randn(40, 2, 64, generator=c.g).cuda()
    freqs = (500000.0 ** (-torch.arange(0, 64, 2, dtype=F64) / 64)).float().cuda()
    first = 3 * 10 ** 9
    ops.kv_append(x, x, c.k, c.v, c.pages, c.ints([0, 40]), c.ints([40]), freqs=freqs, first_pos=first, amplitude=1.25)
    want = rotated(x, torch.arange(40).cuda() + first, freqs, "pairs", 1.25)
    got = c.tokens(c.k, c.pages[0], 40).transpose(0, 1)
    # (the reference's own angle, some 3e9 radians in 64 bits, is off by 2^-22)
    assert ((got - want).abs() <= append_bar("bf16", want, x, freqs, "pairs", 1.25) + 1e-6 * x.abs().amax()).all()


def test_append_rows_without_a_place(ops):
    """rows behind the last sequence are left alone; rows whose page is not in the table or not in the pool are rotated but not stored"""
    c = Cache(4, 2, 64, 16, "f16", 0, [20, 20])
    pages = c.pages[:, :2].contiguous()
    pages[1, 1] = 10 ** 6
    lengths = c.ints([36, 20])                  # sequence 0: rows 2, 3 at 34, 35 lie past its two pages; sequence 1: tokens 16.. in a page that is not there
    x = torch.randn(10, 2, 64, generator=c.g).half().cuda()
    q_out = torch.full_like(x, 7.0)
    k0, v0 = c.k.clone(), c.v.clone()
    ops.kv_append(x, x, c.k, c.v, pages, c.ints([0, 4, 8]), lengths, q=x, q_out=q_out, freqs=torch.zeros(32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(q_out[:8], x[:8]) and (q_out[8:] == 7.0).all()
    assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16)) and torch.equal(c.v.view(torch.int16), v0.view(torch.int16))
    ops.kv_append(x, x, c.k, c.v, pages, c.ints([0, 4, 8]), c.ints([2, 3]))      # more rows than tokens: the earlier rows have no place
    torch.cuda.synchronize()
    assert torch.equal(c.k[pages[0, 0].long(), :, :2].transpose(0, 1), x[2:4]) and torch.equal(c.k[pages[1, 0].long(), :, :3].transpose(0, 1), x[5:8])


def test_append_in_place_queries_and_many_sequences(ops):
    rows = [i % 3 for i in range(2500)]
    held = [r + i % 20 for i, r in enumerate(rows)]
    for layout in ("pairs", "halves"):
        c = Cache(5, 1, 64, 16, "bf16", 0, held)
        R = sum(rows)
        q = torch.randn(R, 3, 64, generator=c.g).bfloat16().cuda()
        k = torch.randn(R, 1, 64, generator=c.g).bfloat16().cuda()
        freqs = (100.0 ** (-torch.arange(0, 64, 2, dtype=F64) / 64)).float().cuda()
        pos = torch.cat([torch.arange(o - r, o) for r, o in zip(rows, held)]).cuda()
        want = rotated(q, pos, freqs, layout)
        bar = append_bar("bf16", want, q, freqs, layout)
        ops.kv_append(k, k, c.k, c.v, c.pages, c.ints(starts(rows)), c.ints(held), q=q, q_out=q, freqs=freqs, layout=layout)
        assert ((q.to(F64) - want).abs() <= bar).all()
        got = torch.cat([c.tokens(c.v, c.pages[s], o)[:, o - r:].transpose(0, 1) for s, (r, o) in enumerate(zip(rows, held)) if r])
        assert torch.equal(got, k.to(F64))


# --------------------------------------------------------------------------------------------------------------- attention
def shared(ops, c, q, prefix, rows, max_rows=None, scale=None, out=None, stream=None, fill=math.nan):
    R, H, D = q.shape
    out = torch.full((R, H, D), fill, dtype=q.dtype, device="cuda") if out is None else out
    work = torch.full((ops.attention_shared_prefix_workspace(R, H, c.n_kv, D) // 4,), math.nan, device="cuda")
    ops.attention_shared_prefix(q, c.k, c.v, c.prefix_pages, prefix, c.pages, c.ints(starts(rows)), c.ints(c.own), out, work,
                                max_rows=max(rows) if max_rows is None else max_rows, scale=scale, stream=stream)
    return out


SHARED = [
    # heads, kv, dim, page, type, prefix, rows, own
    (8, 2, 128, 64, "f16", 100, [1], [1]),                              # one row of one sequence
    (8, 2, 64, 16, "bf16", 1, [1, 1], [1, 70]),                         # one token of prefix
    (4, 4, 64, 32, "f16", 0, [1, 1, 1], [1, 16, 333]),                  # no prefix; no sharing of heads
    (32, 8, 128, 64, "f16", 512, [1] * 4, [1, 17, 48, 64]),             # rows of a KV head fill one tile of 16
    (32, 8, 128, 64, "bf16", 1000, [1] * 16, list(range(1, 17))),       # a tile of 64
    (32, 8, 128, 64, "f16", 1000, [1] * 17, [40 * i + 1 for i in range(17)]),      # tensor memory, one tile
    (32, 8, 128, 64, "f16", 1000, [1] * 33, [7 * i + 1 for i in range(33)]),       # a row past a tile of 128
    (20, 5, 64, 48, "bf16", 1500, [1] * 70, [i % 9 for i in range(70)]),           # pages of 48, two tiles and a part, sequences without own tokens
    (32, 8, 128, 128, "bf16", 4100, [1] * 64, [3 * i for i in range(64)]),         # a unit over several CTAs
    (16, 1, 128, 256, "f16", 2222, [1] * 100, [5] * 100),               # pages longer than a block of keys; 16 heads a KV head
    (8, 8, 64, 16, "f16", 129, [1] * 200, [i % 40 + 1 for i in range(200)]),
    (32, 4, 64, 16, "bf16", 300, [3, 0, 17, 1, 33, 8], [3, 0, 40, 90, 33, 100]),   # several rows a sequence, one with none
    (12, 2, 128, 32, "f16", 65, [40, 1, 2], [700, 1, 2]),
    (8, 2, 128, 16, "bf16", 0, [130], [130]),                           # a prompt of its own
    (4, 2, 64, 64, "f16", 200, [5, 6], [2, 6]),                         # fewer own tokens than rows: the earlier rows see the prefix alone
    (64, 1, 128, 64, "f16", 333, [1, 2], [64, 65]),                     # 64 heads a KV head
]


@pytest.mark.parametrize("heads,kv,dim,page,typ,prefix,rows,own", SHARED)
def test_shared_prefix(ops, heads, kv, dim, page, typ, prefix, rows, own):
    c = Cache(heads + prefix, kv, dim, page, typ, prefix, own)
    q = torch.randn(sum(rows), heads, dim, generator=c.g).to(TYPES[typ]).cuda()
    got = shared(ops, c, q, prefix, rows)
    want, spread, reach = attention_exact(c, q, prefix, rows)
    err = (got.to(F64) - want).abs()
    assert (err <= attention_bar(typ, want, spread, reach, dim)).all(), float(err.max())
    assert torch.equal(got, shared(ops, c, q, prefix, rows))            # the same bits again


# single tokens behind a longer prefix: how many SMs the prefix gets goes by the mean of the own tokens, in levels that end at powers of two
SPLITS = [
    (32, 8, 128, 64, "f16", 2000, [1] * 40, [0] * 40),
    (32, 8, 128, 64, "bf16", 2000, [1] * 40, [16] * 40),
    (32, 8, 128, 64, "f16", 2000, [1] * 40, [16] * 39 + [17]),
    (32, 8, 128, 64, "f16", 3333, [1] * 24, [512] * 24),                # all at the end of a level, which is all that the table holds but a page
    (8, 1, 64, 16, "bf16", 700, [1] * 1500, [i % 5 for i in range(1500)]),         # the mean is that of every other sequence
    (8, 1, 64, 16, "f16", 130, [1] * 1500, [1 + 99 * (i & 1) for i in range(1500)]),
    (16, 4, 64, 32, "bf16", 5000, [1] * 90, [2100 if i == 7 else 3 for i in range(90)]),
    (32, 8, 128, 64, "f16", 129, [1] * 300, [2 * i for i in range(300)]),
]


@pytest.mark.parametrize("heads,kv,dim,page,typ,prefix,rows,own", SPLITS)
def test_shared_prefix_beside_own_tokens(ops, heads, kv, dim, page, typ, prefix, rows, own):
    test_shared_prefix(ops, heads, kv, dim, page, typ, prefix, rows, own)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("at,by", [([128], 20.0), ([129, 161, 193, 225], 20.0), ([159, 191, 223, 255], 17.0), ([300, 400, 500, 600, 700, 800], 16.0), ([0, 895], 40.0),
                                   ([511, 512, 544], 30.0), ([250, 600], -20.0), ([330], 130.0), ([840, 850, 870, 899], 15.0)])
def test_shared_prefix_scores_that_grow(ops, typ, dim, at, by):
    """Scores (in log2) that rise along the prefix by `by` at some keys, by a half or a quarter of it or not at all in some rows: what a CTA has summed up by
    then, in every part of a block of 128 keys, has to fall by as much. 640 blocks: a CTA has several."""
    P, S = 900, 600
    c = Cache(dim + len(at), 8, dim, 64, typ, P, [1] * S)
    q = torch.randn(S, 32, dim, generator=c.g).to(TYPES[typ]).cuda()
    q[..., 0] = torch.tensor([[0.0, 0.25, 0.5, 1.0][(r + h) % 4] for r in range(S) for h in range(32)]).view(S, 32).to(TYPES[typ]).cuda()
    step = by / math.log2(math.e) * dim ** 0.5                                          # what one step adds to q k
    for j in range(P):
        c.k[c.prefix_pages[j // 64].long(), :, j % 64, 0] = step * sum(j >= k for k in at)
    got = shared(ops, c, q, P, [1] * S)
    want, spread, reach = attention_exact(c, q, P, [1] * S)
    ratio = (got.to(F64) - want).abs() / attention_bar(typ, want, spread, reach, dim)
    assert (ratio <= 1).all(), float(ratio.max())


def test_shared_prefix_lengths_that_change_between_replays(ops):
    """Captured once: how the SMs are split goes by the lengths at the time of the replay."""
    c = Cache(5, 8, 128, 64, "f16", 2500, [400] * 48)
    q = torch.randn(48, 32, 128, generator=c.g).half().cuda()
    lengths, out = c.ints(c.own), torch.empty_like(q)
    work = torch.full((ops.attention_shared_prefix_workspace(48, 32, 8, 128) // 4,), math.nan, device="cuda")
    row_start = c.ints(range(49))
    run = lambda stream=None: ops.attention_shared_prefix(q, c.k, c.v, c.prefix_pages, 2500, c.pages, row_start, lengths, out, work, max_rows=1, stream=stream)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        run(s)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            run(s)
        for own in ([1] * 48, [400] * 48, [0] * 48, [8 * i for i in range(48)]):
            lengths.copy_(c.ints(own))
            g.replay()
            s.synchronize()
            c.own = own
            want, spread, reach = attention_exact(c, q, 2500, [1] * 48)
            assert ((out.to(F64) - want).abs() <= attention_bar("f16", want, spread, reach, 128)).all()


def test_shared_prefix_rows_without_keys_and_behind_the_last(ops):
    c = Cache(1, 2, 64, 16, "f16", 0, [0, 3, 0])
    q = torch.randn(8, 4, 64, generator=c.g).half().cuda()
    out = torch.full_like(q, 5.0)
    shared(ops, c, q, 0, [1, 4, 2], out=out)                            # row 7 belongs to nobody
    assert (out[0] == 0).all() and (out[1] == 0).all() and (out[5:7] == 0).all() and (out[7] == 5.0).all() and (out[2:5] != 0).any()


@pytest.mark.parametrize("rows", [[1] * 3, [1] * 40])
def test_shared_prefix_large_scores(ops, rows):
    """scores up to some thousands: one key takes all the weight, later blocks bring larger ones"""
    prefix, own = 700, [30 + i for i in range(len(rows))]
    c = Cache(9, 2, 128, 64, "bf16", prefix, own)
    ramp = torch.linspace(0.1, 30, prefix)
    for j in range(prefix):
        c.k[c.prefix_pages[j // 64].item(), :, j % 64] *= ramp[j].item()
    q = (20 * torch.randn(len(rows), 8, 128, generator=c.g)).bfloat16().cuda()
    got = shared(ops, c, q, prefix, rows)
    want, spread, reach = attention_exact(c, q, prefix, rows)
    assert ((got.to(F64) - want).abs() <= attention_bar("bf16", want, spread, reach, 128)).all()


def test_shared_prefix_strides_scale_and_bound_of_rows(ops):
    """queries and outputs inside wider tensors at odd places, a scale of the caller's, max_rows left open"""
    rows, own, prefix = [1] * 30, [i + 1 for i in range(30)], 200
    c = Cache(10, 4, 64, 32, "f16", prefix, own)
    wide = torch.randn(30, 16 * 64 + 7, generator=c.g).half().cuda()
    q = wide[:, 3:3 + 16 * 64].view(30, 16, 64)
    home = torch.zeros(30, 16, 65, dtype=torch.float16, device="cuda")
    want, spread, reach = attention_exact(c, q, prefix, rows, 0.03)
    for bound in (1, 7, 30):
        out = home[..., :64]
        out.zero_()
        shared(ops, c, q, prefix, rows, max_rows=bound, scale=0.03, out=out)
        assert ((out.to(F64) - want).abs() <= attention_bar("f16", want, spread, reach, 64)).all()
        assert (home[..., 64] == 0).all()


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("heads", [4, 32])
def test_shared_prefix_no_numbers_ahead(ops, typ, heads):
    """a token whose key and value are no numbers reaches the rows that see it, and no others: neither earlier rows of its sequence nor other sequences"""
    rows, own, prefix = [6, 20], [30, 20], 150
    c = Cache(11, 4, 64, 16, typ, prefix, own)
    q = torch.randn(26, heads, 64, generator=c.g).to(TYPES[typ]).cuda()
    clean = shared(ops, c, q, prefix, rows)
    page, off = c.pages[0, 27 // 16].long(), 27 % 16                    # own token 27 of sequence 0: its rows 3, 4, 5 see it
    c.k[page, :, off], c.v[page, :, off] = math.inf, math.nan
    got = shared(ops, c, q, prefix, rows)
    assert torch.isnan(got[3:6]).all()
    keep = [i for i in range(26) if not 3 <= i < 6]
    assert ((got[keep].float() - clean[keep].float()).abs() <= 4 * unit(typ) * c.v[~torch.isnan(c.v)].abs().max()).all()      # (two weights' roundings differ)


def test_shared_prefix_page_ids_outside_the_pool_are_not_followed(ops):
    c = Cache(12, 2, 64, 16, "f16", 64, [20, 5])
    q = torch.randn(2, 4, 64, generator=c.g).half().cuda()
    good = shared(ops, c, q, 64, [1, 1])
    c.pages[0, :2] = torch.tensor([-5, 2 ** 31 - 1], dtype=torch.int32)
    bad = shared(ops, c, q, 64, [1, 1])
    torch.cuda.synchronize()
    assert torch.equal(bad[1], good[1])


def test_shared_prefix_lengths_past_the_table(ops):
    """a length that the table does not hold is cut to what it holds"""
    c = Cache(13, 2, 64, 16, "f16", 40, [32])
    c.pages = c.pages[:, :2].contiguous()
    q = torch.randn(1, 4, 64, generator=c.g).half().cuda()
    good = shared(ops, c, q, 40, [1])
    c.own = [10 ** 9]
    assert torch.equal(shared(ops, c, q, 40, [1]), good)


@pytest.mark.parametrize("prefix", [0, 200])
@pytest.mark.parametrize("rows,max_rows", [([130, 5, 1], 130), ([1, 1, 1], 1), ([3, 2, 3], 3)])
def test_shared_prefix_lengths_at_the_end_of_32_bits(ops, prefix, rows, max_rows):
    """lengths below zero are no own tokens, however far below: limits of rows would wrap to the other end"""
    c = Cache(14, 4, 64, 16, "bf16", prefix, [0, 0, 0])
    q = torch.randn(sum(rows), 32, 64, generator=c.g).bfloat16().cuda()
    none = shared(ops, c, q, prefix, rows, max_rows=max_rows)
    for own in ([-2 ** 31, -2 ** 31 + 2, -1], [-2 ** 31 + 100, -2 ** 31 + 129, -2 ** 31]):
        c.own = own
        assert torch.equal(shared(ops, c, q, prefix, rows, max_rows=max_rows), none)


@pytest.mark.parametrize("prefix", [0, 200])
def test_shared_prefix_row_starts_that_are_no_numbers_of_rows(ops, prefix):
    """sequences whose rows end below zero or begin behind the last have none"""
    c = Cache(15, 4, 64, 16, "f16", prefix, [9, 9, 9, 9])
    q = torch.randn(6, 32, 64, generator=c.g).half().cuda()
    out = torch.full_like(q, 5.0)
    work = torch.empty(ops.attention_shared_prefix_workspace(6, 32, 4, 64), dtype=torch.uint8, device="cuda")
    run = lambda at: ops.attention_shared_prefix(q, c.k, c.v, c.prefix_pages, prefix, c.pages, c.ints(at), c.ints(c.own), out, work, max_rows=3)
    run([0, 3, 3, 3, 3])
    good = out.clone()
    assert (good[3:] == 5.0).all() and (good[:3] != 5.0).any()
    for at in ([0, 3, -2 ** 31, -2 ** 31, -2 ** 31], [0, 3, -1, -7, 0]):
        out.fill_(5.0)
        run(at)
        assert torch.equal(out[:3], good[:3])


# ------------------------------------------------------------------------------------------------------- log probabilities
def logprob_bar(x, lp, entropy, V):
    """S is a sum of up to V / 256 + 40 terms a chain in 32 bits, of exponentials off by 2^-21: relative, so absolute in its logarithm; the difference to the
    maximum, its scaling by log2 e and back are 4 roundings of the logarithms' size. The entropy also divides sum d 2^d, off by the same share."""
    rel = (V / 256 + 40) * 2 ** -24 + 2 ** -21
    return rel + 2 ** -22 * (lp.abs() + math.log(V)), rel * (1 + 2 * math.log(V)) + 2 ** -22 * (entropy + math.log(V))


def logprobs(ops, x, tokens, top, **kw):
    R = x.shape[0]
    lp, h = torch.full((R,), 9.0, device="cuda"), torch.full((R,), 9.0, device="cuda")
    tl, ti = torch.full((R, top), 9.0, device="cuda"), torch.full((R, top), 9, dtype=torch.int32, device="cuda")
    ops.token_logprobs(x, tokens, lp, h, tl if top else None, ti if top else None, **kw)
    return lp, h, tl, ti


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("R,V,gap,top", [(1, 32000, 0, 5), (3, 1, 0, 1), (2, 7, 1, 7), (5, 511, 3, 64), (9, 4097, 0, 20), (300, 1000, 2, 3), (33, 32003, 5, 8),
                                         (2, 128256, 0, 20), (700, 513, 0, 1), (1, 50001, 7, 64)])
def test_logprobs(ops, typ, R, V, gap, top):
    g = torch.Generator(device="cuda")
    g.manual_seed(R + V)
    wide = (3 * torch.randn(R, V + gap, device="cuda", generator=g)).to(TYPES[typ])
    x = wide[:, gap:]                                                   # rows that start off a 16-byte boundary
    tokens = torch.randint(0, V, (R,), device="cuda", generator=g, dtype=torch.int32)
    lp, h, tl, ti = logprobs(ops, x, tokens, top)
    want, entropy, top_lp, ids = logprobs_exact(x, tokens, top)
    bar, bar_h = logprob_bar(x, want, entropy, V)
    assert ((lp.to(F64) - want).abs() <= bar).all() and ((h.to(F64) - entropy).abs() <= bar_h).all()
    assert torch.equal(ti.long(), ids)
    assert ((tl.to(F64) - top_lp).abs() <= logprob_bar(x, top_lp, entropy[:, None], V)[0]).all()


@pytest.mark.parametrize("R", [1, 400])
def test_logprobs_ties_masks_and_extremes(ops, R):
    V = 5000
    x = torch.zeros(R, V, device="cuda")
    tokens = torch.arange(R, device="cuda", dtype=torch.int32)
    for value in (0.0, -3.4028234663852886e38, 3.4028234663852886e38):  # all equal, at the type's lowest and largest value too
        x.fill_(value)
        lp, h, tl, ti = logprobs(ops, x, tokens, 20)
        assert ((lp + math.log(V)).abs() < 1e-4).all() and ((h - math.log(V)).abs() < 1e-4).all()
        assert torch.equal(ti, torch.arange(20, dtype=torch.int32, device="cuda").expand(R, 20))
    x.fill_(-math.inf)                                                  # nothing left
    lp, h, tl, ti = logprobs(ops, x, tokens, 20)
    assert (lp == -math.inf).all() and (h == 0).all() and (tl == -math.inf).all()
    assert torch.equal(ti, torch.arange(20, dtype=torch.int32, device="cuda").expand(R, 20))
    x[:, 4321], x[:, 17] = 1.0, 1.0                                     # two tokens left of 5000
    lp, h, tl, ti = logprobs(ops, x, torch.full_like(tokens, 4321), 3)
    assert ((lp + math.log(2)).abs() < 1e-6).all() and ((h - math.log(2)).abs() < 1e-6).all()
    assert (ti == torch.tensor([17, 4321, 0], device="cuda")).all() and (tl[:, 2] == -math.inf).all()
    x.copy_(torch.arange(V, device="cuda").expand(R, V))                # ascending, one token far above all
    x[:, 100] = 10 ** 6
    lp, h, tl, ti = logprobs(ops, x, torch.full_like(tokens, 100), 4)
    assert (lp == 0).all() and (h == 0).all() and (ti == torch.tensor([100, V - 1, V - 2, V - 3], device="cuda")).all()


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("top", [1, 16, 17, 33, 64])
@pytest.mark.parametrize("R", [1, 9, 300, 700])
def test_logprobs_of_rows_with_thousands_of_equal_entries(ops, R, top, typ):
    """Masked but for a few (more and fewer than are asked for), the rest at the type's lowest value, ties for the first places, ties at the end of the row: the
    lowest ids come first. Values are whole, so that they tie in 16 bits too."""
    V = 20011
    g = torch.Generator(device="cuda")
    g.manual_seed(R + top)
    lowest = torch.finfo(TYPES[typ]).min
    x = torch.empty(R, V, device="cuda")
    noise = torch.randint(-30, 0, (R, V), device="cuda", generator=g).float()
    kinds = ["masked", "lowest", "ties above", "ties at the end", "steps", "few and ties"]
    for r in range(R):
        kind = kinds[r % len(kinds)]
        if kind in ("masked", "lowest"):
            x[r] = -math.inf if kind == "masked" else lowest
            few = torch.randperm(V, device="cuda", generator=g)[:[0, 3, 40, 1][r // len(kinds) % 4]]
            x[r, few] = torch.arange(few.numel(), device="cuda").float() // 2
        elif kind == "ties above":
            x[r] = torch.where(noise[r] > -10, 5.0, noise[r])
        elif kind == "ties at the end":
            x[r] = -20.0
            x[r, V - 3000:] = 2.0
            x[r, V // 2] = 3.0
        elif kind == "steps":
            x[r] = -(torch.arange(V, device="cuda") // 4000).float()
        else:
            x[r] = -50.0
            x[r, ::5] = 1.0
            x[r, 11::4001] = 9.0
    x = x.to(TYPES[typ])
    tokens = torch.randint(0, V, (R,), device="cuda", generator=g, dtype=torch.int32)
    lp, h, tl, ti = logprobs(ops, x, tokens, top)
    _, _, _, ids = logprobs_exact(x, tokens, top)
    empty = (x == -math.inf).all(1)                                     # (what such a row gives is tested above)
    # (below the maximum first: next to the lowest value of 32 bits, 3.4e38, the logarithm of a sum is lost in 64 bits too, whose unit is 3.8e22 there)
    d = x.to(F64) - x.to(F64).amax(1, keepdim=True)
    full = d - d.exp().sum(1, keepdim=True).log()
    entropy = -torch.where(full > -700.0, full.exp() * full, 0.0).sum(1)
    want, top_lp = full.gather(1, tokens.long()[:, None])[:, 0], full.gather(1, ids)
    assert torch.equal(ti.long(), ids)
    ok = lambda a, b, bar: (a.to(F64) == b) | ((a.to(F64) - b).abs() <= bar)
    bar, bar_h = logprob_bar(x, want.nan_to_num(neginf=0.0), entropy, V)
    assert (ok(lp, want, bar) | empty).all() and (ok(h, entropy, bar_h) | empty).all()
    assert (ok(tl, top_lp, logprob_bar(x, top_lp.nan_to_num(neginf=0.0), entropy[:, None], V)[0]) | empty[:, None]).all()


def test_logprobs_no_numbers(ops):
    x = torch.zeros(3, 1000, device="cuda")
    x[0, 500] = math.nan
    x[1, 3] = math.inf
    x[2, :998] = math.nan
    lp, h, tl, ti = logprobs(ops, x, torch.tensor([1, 1, 999], dtype=torch.int32, device="cuda"), 4)
    assert torch.isnan(lp).all() and torch.isnan(h).all()
    assert ti.tolist() == [[0, 1, 2, 3], [3, 0, 1, 2], [998, 999, 0, 1]]


def test_logprobs_tokens_outside_and_left_out_results(ops):
    x = torch.randn(4, 100, device="cuda")
    lp, h, tl, ti = logprobs(ops, x, torch.tensor([-1, 100, 2 ** 31 - 1, 5], dtype=torch.int32, device="cuda"), 64)
    assert (lp[:3] == -math.inf).all() and torch.isfinite(lp[3])
    short = torch.randn(2, 10, device="cuda")
    lp, h, tl, ti = logprobs(ops, short, torch.zeros(2, dtype=torch.int32, device="cuda"), 12)
    assert (ti[:, 10:] == -1).all() and (tl[:, 10:] == -math.inf).all() and torch.equal(ti[:, :10].long(), short.sort(1, descending=True).indices)
    only = torch.empty(4, device="cuda")
    ops.token_logprobs(x, entropy=only)
    full = torch.distributions.Categorical(logits=x.double()).entropy()
    assert ((only - full).abs() < 1e-5).all()


# ------------------------------------------------------------------------------------------------------------ all together
def test_streams_and_graphs(ops):
    """the calls run on the stream that they are given, and can be captured and replayed with new inputs"""
    rows, prefix = [1] * 20, 150
    c = Cache(20, 2, 64, 16, "f16", prefix, [9] * 20, spare=40)
    freqs = (100.0 ** (-torch.arange(0, 64, 2, dtype=F64) / 64)).float().cuda()
    x = torch.randn(20, 4 + 2 + 2, 64, generator=c.g).half().cuda()
    q, out, held, start = torch.zeros(20, 4, 64, dtype=torch.float16, device="cuda"), torch.zeros(20, 4, 64, dtype=torch.float16, device="cuda"), c.ints(c.own), c.ints(starts(rows))
    work = torch.empty(ops.attention_shared_prefix_workspace(20, 4, 2, 64), dtype=torch.uint8, device="cuda")
    lp, h = torch.zeros(20, device="cuda"), torch.zeros(20, device="cuda")
    head = torch.randn(256, 500, generator=c.g).half().cuda()
    tokens = torch.arange(20, dtype=torch.int32, device="cuda")
    logits = torch.zeros(20, 500, dtype=torch.float16, device="cuda")

    def step(stream):
        ops.kv_append(x[:, 4:6], x[:, 6:], c.k, c.v, c.pages, start, held, q=x[:, :4], q_out=q, freqs=freqs, first_pos=prefix, stream=stream)
        ops.attention_shared_prefix(q, c.k, c.v, c.prefix_pages, prefix, c.pages, start, held, out, work, max_rows=1, stream=stream)
        torch.matmul(out.view(20, 256), head, out=logits)
        ops.token_logprobs(logits, tokens, lp, h, stream=stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(side)
        with torch.cuda.graph(graph, stream=side):
            step(side)
    torch.cuda.synchronize()
    for n in range(3):
        x.copy_(torch.randn(20, 8, 64, generator=c.g))
        held.add_(1)
        c.own = [o + 1 for o in c.own]
        graph.replay()
        torch.cuda.synchronize()
        first = out.clone(), lp.clone(), h.clone()
        want, spread, reach = attention_exact(c, q, prefix, rows)
        assert ((out.to(F64) - want).abs() <= attention_bar("f16", want, spread, reach, 64)).all()
        step(torch.cuda.current_stream())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, (out, lp, h)))


def test_scoring_answers_to_one_prompt(ops):
    """A one-layer model scores several answers: the shared prompt once and every answer's own tokens in pages, against every answer run by itself in 64 bits."""
    D, H, G, V, page, prefix = 64, 4, 2, 321, 16, 50
    answers = [7, 1, 19, 12]
    g = torch.Generator()
    g.manual_seed(7)
    prompt, own = torch.randint(0, V, (prefix,), generator=g), [torch.randint(0, V, (n,), generator=g) for n in answers]
    table, wq, wk, wv = (torch.randn(*s, generator=g) / 4 for s in ((V, 64), (64, H * D), (64, G * D), (64, G * D)))
    head = torch.randn(H * D, V, generator=g)
    freqs = (100.0 ** (-torch.arange(0, D, 2, dtype=F64) / D)).float()
    c = Cache(8, G, D, page, "f16", prefix, answers)
    c.k.fill_(math.nan)
    c.v.fill_(math.nan)
    part = lambda t, w, n: (table[t] @ w).half().cuda().view(-1, n, D)
    f = freqs.cuda()
    ops.kv_append(part(prompt, wk, G), part(prompt, wv, G), c.k, c.v, c.prefix_pages[None], c.ints([0, prefix]), c.ints([prefix]), freqs=f)
    flat = torch.cat(own)
    start, held = c.ints(starts(answers)), c.ints(answers)
    q = part(flat, wq, H)
    ops.kv_append(part(flat, wk, G), part(flat, wv, G), c.k, c.v, c.pages, start, held, q=q, q_out=q, freqs=f, first_pos=prefix)
    out = torch.zeros_like(q)
    work = torch.empty(ops.attention_shared_prefix_workspace(len(flat), H, G, D), dtype=torch.uint8, device="cuda")
    ops.attention_shared_prefix(q, c.k, c.v, c.prefix_pages, prefix, c.pages, start, held, out, work, max_rows=max(answers))
    logits = out.view(-1, H * D).float() @ head.cuda()
    tokens = torch.randint(0, V, (len(flat),), generator=g, dtype=torch.int32).cuda()
    lp, h, tl, ti = logprobs(ops, logits, tokens, 5)
    r0 = 0
    for t in own:
        whole = torch.cat([prompt, t])
        pos = torch.arange(len(whole)).cuda()
        qq, kk = (rotated(part(whole, w, n).double(), pos, f, "pairs") for w, n in ((wq, H), (wk, G)))
        vv = part(whole, wv, G).double()
        s = torch.einsum("ighd,jgd->ghij", qq.view(-1, G, H // G, D), kk) * D ** -0.5
        s = s.masked_fill(pos[None, :] > pos[:, None], -math.inf)
        o = torch.einsum("ghij,jgd->ighd", s.softmax(-1), vv).reshape(len(whole), H * D)[prefix:]
        want = torch.log_softmax(o @ head.cuda().double(), -1)
        n = len(t)
        got = lp[r0:r0 + n].double()
        ref = want.gather(1, tokens[r0:r0 + n, None].long())[:, 0]
        # queries, keys, probabilities, outputs rounded to f16 (2^-11 each of values up to about 1) times a head row's norm of 16, twice (numerator and sum)
        assert ((got - ref).abs() <= 2 * 16 * 4 * 2 ** -11).all()
        assert (want.gather(1, ti[r0:r0 + n].long()) - tl[r0:r0 + n].double()).abs().max() <= 2 * 16 * 4 * 2 ** -11
        r0 += n


def test_no_wait_ran_out(native_lib):
    import ctypes
    code = ctypes.c_uint32(9)
    assert native_lib.b2_device_op_error(0, ctypes.byref(code)) == 0 and code.value == 0


def test_a_failed_call_is_not_reported_by_the_next_one(native_lib, ops):
    """a device that is not there: the calls behind it say how they went themselves"""
    import ctypes
    import numpy as np
    c = Cache(1, 2, 64, 16, "f16", 0, [3])
    k = torch.randn(3, 2, 64, generator=c.g).cuda()
    start, held = c.ints([0, 3]), c.ints([3])
    x, w, y = np.ones(64, np.float32), np.ones(64, np.float32), np.zeros(64, np.float32)
    ptr = lambda a: a.ctypes.data_as(ctypes.c_void_p)
    torch.cuda.synchronize()
    code = ctypes.c_uint32()
    fails = [lambda: native_lib.b2_device_op_error(99, ctypes.byref(code)), lambda: native_lib.b2_token_logprobs(99, 256, 0, 8, 1, 8, None, None, 256, 0, None, None, None)]
    for fail in fails:
        assert fail() < 0 and "invalid device" in native_lib.b2_last_error().decode()
        ops.kv_append(k, k, c.k, c.v, c.pages, start, held)
        assert fail() < 0
        assert native_lib.b2_op_rmsnorm(0, ptr(x), ptr(w), 1e-5, 64, 1, ptr(y)) == 0
    torch.cuda.synchronize()
    assert torch.equal(c.k[c.pages[0, 0], :, :3], k.half().transpose(0, 1)) and np.abs(y - 1).max() < 1e-4


@pytest.mark.parametrize("tensor_memory", [0, 1])
def test_a_wait_that_ran_out_is_reported_once(native_lib, tensor_memory):
    """also from a stream that the default one does not wait for, behind work that is still under way"""
    from llama_cpp import device_ops as ops
    assert ops.error(0) == 0
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(int(2e8))
    assert native_lib.b2_op_give_up(0, tensor_memory, 0x90001 + tensor_memory, side.cuda_stream) == 0
    assert native_lib.b2_op_give_up(0, tensor_memory, 0x77, side.cuda_stream) == 0          # (not the first)
    assert ops.error(0) == 0x90001 + tensor_memory
    assert ops.error(0) == 0
    for words in (0, 1):                                                                    # both files' words are taken at once
        assert native_lib.b2_op_give_up(0, words, 0x11 + words, None) == 0
    assert ops.error(0) == 0x11 and ops.error(0) == 0
    with pytest.raises(RuntimeError):
        ops.error(99)
    with pytest.raises(RuntimeError):
        ops.error(-1)
    assert ops.error(0) == 0
