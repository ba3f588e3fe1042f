"""The paged cache in 4 bits on the GPU against its definition in 64 bits: appends byte for byte, rows read back, attention, and the three together."""
import math

import pytest

torch = pytest.importorskip("torch")

from cache_4bit_util import GROUP, Cache4, attention_bar, attention_exact, coded, quantised, values
from device_ops_util import F64, TYPES, rotated, unit

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


def rotated_32(x, positions, freqs, layout, amplitude=1.0):
    """the rotation as it is defined for codes: angles, sines and cosines in 64 bits, rounded once, products and sums in 32 bits one by one"""
    x, rot = x.float(), 2 * len(freqs)
    angle = positions.to(F64)[:, None] * freqs.to(F64)[None]
    c, s = ((amplitude * t).float()[:, None] for t in (angle.cos(), angle.sin()))
    y = x.clone()
    if layout == "pairs":
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, a * s + b * c
    return y


# ------------------------------------------------------------------------------------------------------------------ append
APPENDS = [
    # heads, kv, dim, page, rot, rows, tokens behind, first position, input, q_out, layout, joint projection
    (32, 8, 128, 64, 128, [1] * 5, [0, 63, 64, 127, 300], 0, "f32", "f16", "pairs", False),
    (32, 4, 64, 16, 64, [3, 0, 17, 1, 40, 0], [5, 0, 15, 16, 0, 9], 1000, "bf16", "bf16", "halves", True),
    (8, 8, 128, 48, 64, [50, 1, 33], [7, 1, 47], 131071, "f16", "bf16", "halves", True),
    (12, 2, 128, 32, 96, [70], [31], 0, "f16", "f16", "pairs", True),
    (5, 5, 64, 16, 20, [2, 33], [0, 16], 3, "f32", "bf16", "pairs", False),
    (3, 1, 64, 16, 36, [4, 50], [1, 0], 77, "bf16", "f16", "halves", False),       # halves that are no whole pieces
    (4, 2, 64, 64, 0, [3, 2], [0, 5], 0, "f16", "f16", "pairs", False),            # no rotation at all
    (7, 1, 128, 16, 128, [1, 2, 1], [0, 5, 30], 3 * 10 ** 9, "f32", "f16", "halves", False),
]


@pytest.mark.parametrize("heads,kv,dim,page,rot,rows,behind,first,typ,out_typ,layout,joint", APPENDS)
def test_append(ops, heads, kv, dim, page, rot, rows, behind, first, typ, out_typ, layout, joint):
    """the pools byte for byte: the rows' codes and scales, and everything else as it was"""
    held = [r + b for r, b in zip(rows, behind)]
    c = Cache4(len(rows) + dim, kv, dim, page, held)
    R = sum(rows)
    x = torch.randn(R, (heads + 2 * kv) * dim, generator=c.g).to(TYPES[typ]).cuda()
    q, k, v = x[:, :heads * dim].view(R, heads, dim), x[:, heads * dim:(heads + kv) * dim].view(R, kv, dim), x[:, (heads + kv) * dim:].view(R, kv, dim)
    if not joint:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    freqs = (10000.0 ** (-torch.arange(0, rot, 2, dtype=F64) / max(rot, 1))).float().cuda()
    pos = torch.cat([torch.arange(b, b + r) for r, b in zip(rows, behind)]).cuda() + first
    q_out = torch.full((R, heads, dim), math.nan, dtype=TYPES[out_typ], device="cuda")
    ops.kv_append_4bit(k, v, c.k_pool, c.v_pool, c.pages, c.ints(starts(rows)), c.ints(held), q=q, q_out=q_out, freqs=freqs if rot else None, layout=layout, first_pos=first)
    new = torch.cat([torch.arange(c.start[s + 1] - r, c.start[s + 1]) for s, r in enumerate(rows)])
    for got, was, old, now in ((c.k_pool, c.bytes_k, c.k, rotated_32(k, pos, freqs, layout)), (c.v_pool, c.bytes_v, c.v, v)):
        all_rows = old.float()
        all_rows[new] = now.float().cpu()
        assert torch.equal(got.cpu(), c.expect(len(was), all_rows, got is c.k_pool, base=was))
    # queries: one rounding, before it four of 2^-24 of the two entries' sizes, and angles that are off by 2^-52 of themselves here and there (positions of 3e9: 7e-7, where equality
    # with another order of the same 64-bit products cannot be asked for)
    want, size = rotated(q, pos, freqs, layout), q.to(F64).abs().amax(-1, keepdim=True) * 2
    assert ((q_out.to(F64) - want).abs() <= unit(out_typ) * want.abs() + (2 ** -22 + 2 ** -51 * float(pos.max())) * size + (2 ** -25 if out_typ == "f16" else 0)).all()
    # and the definition: the rotation in 32 bits is within 4 roundings (2^-24 of the two entries' sizes) of the one in 64, an entry within half a step and its scale's rounding of that
    want = rotated(k, pos, freqs, layout)
    back = torch.full((R, kv, dim), math.nan, device="cuda")
    ops.kv_read_4bit(c.k_pool, c.v_pool, c.pages, c.ints(starts(rows)), c.ints(held), back, None)
    step = quantised(want)[1].to(F64).abs().repeat_interleave(GROUP, -1)
    off = (back.to(F64) - want).abs()
    assert ((off <= 0.501 * step + 1e-5) | ((back.abs() >= 6.99 * step) & (off <= 1.01 * step + 1e-5))).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("typ", ["f32", "bf16", "f16"])
def test_append_of_special_entries(ops, dim, typ):
    """zeros of both signs, groups of one entry, m and -m in a group, ties between codes, entries past the largest scale and below the smallest, infinities, NaN"""
    big = {"f32": 3e38, "bf16": 3e38, "f16": 65504.0}[typ]
    x = torch.randn(13, 2, dim).to(TYPES[typ])
    x[0] = 0.0
    x[1] = -0.0
    x[2] = 0.0
    x[2, :, 5::GROUP] = 3.0
    x[3, :, 1::GROUP], x[3, :, 9::GROUP] = 4.0, -4.0
    x[4] = torch.tensor([-8.0, 0.5, 1.5, -0.5, -1.5, 2.5, -2.5, 7.5]).repeat(dim // 8)      # scale 1: ties to even
    x[5, :, 0] = big
    x[6, :, 3] = -big
    x[7] *= 1e-7
    x[8] = 2.0 ** -24
    x[9, 0, 4] = math.inf
    x[9, 1, 40] = -math.inf
    x[10, :, 33] = math.nan
    x[11, 0] = math.nan
    x[12] = 2.0 ** -20 * torch.arange(dim)
    for seq in range(2):
        c = Cache4(seq, 2, dim, 16, [13])
        ops.kv_append_4bit(x.cuda(), x.flip(1).contiguous().cuda(), c.k_pool, c.v_pool, c.pages, c.ints([0, 13]), c.ints([13]))
        assert torch.equal(c.k_pool.cpu(), c.expect(len(c.bytes_k), x, True, base=c.bytes_k))
        assert torch.equal(c.v_pool.cpu(), c.expect(len(c.bytes_v), x.flip(1), False, base=c.bytes_v))
        back = torch.zeros(13, 2, dim, device="cuda")
        ops.kv_read_4bit(c.k_pool, c.v_pool, c.pages, c.ints([0, 13]), c.ints([13]), back, None)
        want = coded(x)
        assert torch.equal(torch.nan_to_num(back.cpu().to(F64), nan=1e9), torch.nan_to_num(want, nan=1e9))
        assert torch.isnan(want[9, 0, :32]).all() and not torch.isnan(want[9, 0, 32:]).any() and torch.isnan(want[10, :, 32:64]).all()


def test_append_rows_without_a_place(ops):
    """rows behind the last sequence are left alone; rows whose page is not in the table or not in the pool are rotated but not stored"""
    c = Cache4(4, 2, 64, 16, [20, 20])
    pages = c.pages[:, :2].contiguous()
    pages[1, 1] = 10 ** 6
    x = torch.randn(10, 2, 64, generator=c.g).half().cuda()
    q_out = torch.full_like(x, 7.0)
    ops.kv_append_4bit(x, x, c.k_pool, c.v_pool, pages, c.ints([0, 4, 8]), c.ints([36, 20]), q=x, q_out=q_out, freqs=torch.zeros(32, device="cuda"))
    assert torch.equal(q_out[:8], x[:8]) and (q_out[8:] == 7.0).all()
    assert torch.equal(c.k_pool.cpu(), c.bytes_k) and torch.equal(c.v_pool.cpu(), c.bytes_v)
    back = torch.full((10, 2, 64), 5.0, device="cuda")
    ops.kv_read_4bit(c.k_pool, c.v_pool, pages, c.ints([0, 4, 8]), c.ints([34, 18]), back, back)       # rows 2, 3 have no page in the table, 6, 7 none in the pool
    assert (back[2:4] == 5.0).all() and (back[6:] == 5.0).all() and (back[:2] != 5.0).any() and (back[4:6] != 5.0).any()
    ops.kv_append_4bit(x, x, c.k_pool, c.v_pool, pages, c.ints([0, 4, 8]), c.ints([2, 3]))              # more rows than tokens: the earlier rows have no place
    ops.kv_read_4bit(c.k_pool, c.v_pool, pages, c.ints([0, 2, 5]), c.ints([2, 3]), back, None)
    assert torch.equal(back[:5].to(F64), torch.cat([coded(x[2:4]), coded(x[5:8])]))
    for lengths in ([-5, -2 ** 31], [2 ** 31 - 1, 2 ** 31 - 1]):
        before = c.k_pool.clone()
        back.fill_(5.0)
        ops.kv_append_4bit(x, x, c.k_pool, c.v_pool, pages, c.ints([0, 4, 8]), c.ints(lengths))
        ops.kv_read_4bit(c.k_pool, c.v_pool, pages, c.ints([0, 4, 8]), c.ints(lengths), back, None)
        assert torch.equal(c.k_pool, before) and (back == 5.0).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_append_in_place_queries_and_many_sequences(ops, dim):
    rows = [i % 3 for i in range(1500)]
    held = [r + i % 20 for i, r in enumerate(rows)]
    c = Cache4(5, 1, dim, 16, held, "bf16", fill=0)
    R = sum(rows)
    pos = torch.cat([torch.arange(o - r, o) for r, o in zip(rows, held)]).cuda()
    freqs = (100.0 ** (-torch.arange(0, dim, 2, dtype=F64) / dim)).float().cuda()
    for layout in ("pairs", "halves"):
        q = torch.randn(R, 3, dim, generator=c.g).bfloat16().cuda()
        k = torch.randn(R, 1, dim, generator=c.g).bfloat16().cuda()
        want = rotated_32(q, pos, freqs, layout).bfloat16()
        ops.kv_append_4bit(k, k, c.k_pool, c.v_pool, c.pages, c.ints(starts(rows)), c.ints(held), q=q, q_out=q, freqs=freqs, layout=layout)
        assert torch.equal(q, want)
        back = torch.zeros(2, R, 1, dim, device="cuda")
        ops.kv_read_4bit(c.k_pool, c.v_pool, c.pages, c.ints(starts(rows)), c.ints(held), back[0], back[1])
        assert torch.equal(back[0].to(F64), coded(rotated_32(k, pos, freqs, layout))) and torch.equal(back[1].to(F64), coded(k))


# -------------------------------------------------------------------------------------------------------------------- read
READS = [
    # kv, dim, page, rows, tokens behind, type, gap between rows, first entry
    (8, 128, 64, [1], [0], "f16", 0, 0),
    (8, 128, 64, [100, 7], [33, 0], "bf16", 0, 0),
    (5, 64, 48, [3, 0, 50, 16], [0, 9, 13, 16], "f32", 0, 0),
    (4, 64, 16, [40, 1], [2, 70], "f16", 8, 0),
    (3, 128, 128, [31, 130], [1, 5], "bf16", 3, 1),               # rows that start anywhere
    (1, 128, 16, [17], [0], "f32", 2, 1),
    (2, 64, 32, [i % 4 for i in range(300)], [i % 9 for i in range(300)], "f16", 0, 0),
]


@pytest.mark.parametrize("kv,dim,page,rows,behind,typ,gap,at", READS)
def test_read(ops, kv, dim, page, rows, behind, typ, gap, at):
    held = [r + b for r, b in zip(rows, behind)]
    c = Cache4(dim + page, kv, dim, page, held)
    R = sum(rows)
    wide = torch.full((2, R + 2, kv, dim + gap + at), 9.0, dtype=TYPES[typ], device="cuda")
    k, v = wide[0, :, :, at:at + dim], wide[1, :, :, at:at + dim]
    pick = torch.cat([torch.arange(c.start[s + 1] - r, c.start[s + 1]) for s, r in enumerate(rows)])
    ops.kv_read_4bit(c.k_pool, c.v_pool, c.pages, c.ints(starts(rows)), c.ints(held), k, v)
    for got, rows_of in ((k, c.k), (v, c.v)):
        want = coded(rows_of[pick]).float().to(TYPES[typ])        # (exact in 32 bits, one rounding)
        assert torch.equal(got[:R].cpu(), want) and (got[R:] == 9.0).all()
    left = torch.ones(dim + gap + at, dtype=torch.bool)
    left[at:at + dim] = False
    assert (wide[..., left.cuda()] == 9.0).all()
    both = k.clone(), v.clone()
    for one, name in ((k, "k"), (v, "v")):                        # one of them alone
        wide.fill_(9.0)
        ops.kv_read_4bit(c.k_pool, c.v_pool, c.pages, c.ints(starts(rows)), c.ints(held), k if name == "k" else None, v if name == "v" else None)
        assert torch.equal(one[:R], both[name == "v"][:R]) and ((v if name == "k" else k) == 9.0).all()


# --------------------------------------------------------------------------------------------------------------- attention
def attend(ops, c, q, rows, max_rows=None, scale=None, out=None, stream=None, fill=math.nan, own=None):
    R, H, D = q.shape
    out = torch.full((R, H, D), fill, dtype=q.dtype, device="cuda") if out is None else out
    work = torch.full((ops.attention_4bit_workspace(R, H, c.n_kv, D) // 4,), math.nan, device="cuda")
    ops.attention_4bit(q, c.k_pool, c.v_pool, c.pages, c.ints(starts(rows)), c.ints(c.own if own is None else own), out, work,
                       max_rows=max([1] + rows) if max_rows is None else max_rows, scale=scale, stream=stream)
    return out


ATTENTIONS = [
    # heads, kv, dim, page, type, rows, tokens
    (8, 2, 128, 64, "f16", [1], [1]),
    (8, 2, 64, 16, "bf16", [1, 1], [1, 70]),
    (4, 4, 64, 32, "f16", [1, 1, 1], [31, 32, 33]),                     # ends of steps
    (8, 1, 128, 16, "f16", [1, 1], [16, 17]),                           # eight heads a KV head: a tile of eight rows
    (9, 1, 128, 16, "bf16", [1], [1500]),                               # nine: one of sixteen
    (16, 1, 64, 256, "f16", [1] * 3, [5, 300, 0]),                      # a sequence without tokens
    (17, 1, 64, 16, "bf16", [1] * 2, [64, 65]),                         # more than one tile a token
    (64, 1, 128, 64, "f16", [1, 2], [64, 65]),
    (32, 8, 128, 64, "f16", [1], [3000]),                               # a long one: many warps a segment
    (32, 8, 128, 64, "bf16", [1], [2999]),
    (32, 8, 128, 48, "f16", [1] * 32, [37 * i + 1 for i in range(32)]),
    (32, 4, 64, 16, "bf16", [1] * 65, [(i * 31) % 200 for i in range(65)]),
    (8, 8, 64, 128, "f16", [1] * 700, [i % 40 for i in range(700)]),    # short ones, several a warp
    (20, 5, 128, 32, "bf16", [2, 0, 3, 1], [700, 5, 90, 1]),            # several rows, none
    (32, 4, 64, 16, "bf16", [3, 0, 17, 1, 33, 8], [3, 0, 40, 90, 33, 100]),
    (12, 2, 128, 32, "f16", [40, 1, 2], [400, 1, 2]),
    (8, 2, 128, 16, "bf16", [130], [130]),                              # a prompt
    (32, 8, 128, 64, "f16", [150], [407]),
    (4, 2, 64, 64, "f16", [5, 6], [2, 6]),                              # fewer tokens than rows: the earlier rows see nothing
    (32, 8, 64, 64, "bf16", [70, 3, 200], [70, 500, 333]),
]


@pytest.mark.parametrize("heads,kv,dim,page,typ,rows,own", ATTENTIONS)
def test_attention(ops, heads, kv, dim, page, typ, rows, own):
    c = Cache4(heads + sum(own), kv, dim, page, own)
    q = torch.randn(sum(rows), heads, dim, generator=c.g).to(TYPES[typ]).cuda()
    got = attend(ops, c, q, rows)
    want, *sizes = attention_exact(c, q, rows)
    err = (got.to(F64) - want).abs()
    assert (err <= attention_bar(typ, want, *sizes, dim, max(rows) * heads // kv > 64)).all(), float(err.max())
    assert torch.equal(got, attend(ops, c, q, rows))                    # the same bits again
    assert ops.error(0) == 0


# more than 64 rows of a KV head of a sequence go another way than fewer; more than 8 and up to 8 too
WAYS = [(4, [1, 1, 1]), (8, [3, 1, 4]), (16, [2, 9, 5]), (16, [60, 33, 100])]


def visible_nan(c, q, rows, k, v):
    """attention over values some of which are no numbers, by the definition: a row's dims are NaN where a value that it sees is, all of them where a key is"""
    R, H, D = q.shape
    G = H // c.n_kv
    clean_k, clean_v = torch.nan_to_num(k, nan=0.0), torch.nan_to_num(v, nan=0.0)
    out, *sizes = attention_exact(c, q, rows, k=clean_k, v=clean_v)
    r0 = 0
    for s, (n, o) in enumerate(zip(rows, c.own)):
        for i in range(n):
            seen = slice(c.start[s], c.start[s] + max(0, o - n + i + 1))
            bad_v = torch.isnan(v[seen]).any(0)                          # [kv heads, dim]
            bad_k = torch.isnan(k[seen]).any(0).any(-1, keepdim=True)
            out[r0 + i][(bad_v | bad_k).repeat_interleave(G, 0)] = math.nan
        r0 += n
    return out, sizes


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,rows", WAYS)
def test_attention_numbers_that_are_none(ops, heads, rows, dim, typ):
    """a NaN or an infinity in a value reaches the dims of its group, in rows that see its key, and no others; in a key it reaches those rows alone; what lies behind the last token
    (NaN everywhere) reaches nobody"""
    own = [n + 37 + 50 * s for s, n in enumerate(rows)]
    rows_k, rows_v = (torch.randn(sum(own), 2, dim).half() for _ in range(2))
    start = [sum(own[:s]) for s in range(len(own))]
    rows_v[start[1] - 1, 0, 5] = math.nan                                # the last token of sequence 0: its last row alone
    rows_v[start[0] + 3, 1, 40] = math.inf                               # a token that all rows see
    rows_v[start[2] - 2, 1, 33] = -math.inf                              # the last but one of sequence 1
    rows_k[start[2] + own[2] - 1, 1, 7] = math.nan                       # a key, sequence 2
    c = Cache4(1, 2, dim, 16, own, k=rows_k, v=rows_v, fill=0xff)
    q = torch.randn(sum(rows), heads, dim, generator=c.g).to(TYPES[typ]).cuda()
    got = attend(ops, c, q, rows)
    want, sizes = visible_nan(c, q, rows, c.values(c.k), c.values(c.v))
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isnan(want).any() and not torch.isnan(want).all()
    fine = ~torch.isnan(want)
    bar = attention_bar(typ, torch.nan_to_num(want), *sizes, dim, max(rows) * heads // 2 > 64)
    assert ((got.to(F64) - want).abs() <= bar)[fine].all()


@pytest.mark.parametrize("heads,rows", WAYS)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_sizes_of_values(ops, heads, rows, dim):
    """values and keys far apart in size from head to head, group to group and token to token: near the smallest f16 numbers, past the largest"""
    own = [n + 70 + 30 * s for s, n in enumerate(rows)]
    c0 = Cache4(2, 4, dim, 16, own, "bf16")
    k, v = c0.k.float(), c0.v.float()
    v[:, 0] *= 2.0 ** -17                                                # scales that f16 holds with few bits
    v[:, 1] *= 3e4                                                       # past f16's largest number
    v[:, 2] *= (10.0 ** torch.arange(-3, 4).float())[torch.arange(len(v)) % 7][:, None]
    v[:, 3, :32] = 0.0
    k[:, 1] *= 1e-4
    k[:, 2] *= 2e4
    c = Cache4(2, 4, dim, 16, own, k=k.bfloat16(), v=v.bfloat16())
    q = torch.randn(sum(rows), heads, dim, generator=c.g)
    q[:, heads // 2:heads // 4 * 3] *= 1e-4                              # (of the large keys)
    q = q.bfloat16().cuda()
    got = attend(ops, c, q, rows)
    want, *sizes = attention_exact(c, q, rows)
    assert torch.isfinite(got).all()
    assert ((got.to(F64) - want).abs() <= attention_bar("bf16", want, *sizes, dim, max(rows) * heads // 4 > 64)).all()


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("heads,rows", WAYS)
def test_attention_ends_of_the_scale(ops, heads, rows, typ):
    """the smallest and the largest scale: even weights, and all weight on the largest score; queries of zero: even weights whatever the scale"""
    own = [n + 40 for n in rows]
    c = Cache4(10, 2, 64, 16, own)
    q = torch.randn(sum(rows), heads, 64, generator=c.g).to(TYPES[typ]).cuda()
    q[::2, ::3] = 0.0
    for scale in (2.0 ** -40, 2.0 ** 40):
        got = attend(ops, c, q, rows, scale=scale)
        want, *sizes = attention_exact(c, q, rows, scale=scale)
        assert torch.isfinite(got).all()
        near = (got.to(F64) - want).abs() <= attention_bar(typ, want, *sizes, 64, max(rows) * heads // 2 > 64)
        assert near.all()
        if scale > 1:
            # scores of 2^40 and more, whose two largest are apart by more than their errors: the largest one's value
            k, v = c.values(c.k), c.values(c.v)
            r0 = 0
            for s, n in enumerate(rows):
                for i in range(n):
                    at = slice(c.start[s], c.start[s] + own[s] - n + i + 1)
                    for h in range(heads):
                        top = (k[at, h // (heads // 2)] @ q[r0 + i, h].to(F64)).topk(2)
                        if top.values[0] - top.values[1] > 2 ** -6 * top.values[0].abs():
                            one = v[at, h // (heads // 2)][top.indices[0]]
                            assert ((got[r0 + i, h].to(F64) - one).abs() <= 2 ** -7 * one.abs() + 2 ** -20).all()
                r0 += n


@pytest.mark.parametrize("heads,rows", WAYS)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_largest_f16_entries(ops, heads, rows, dim):
    """keys and values up to f16's largest number, in f16"""
    own = [n + 50 for n in rows]
    c0 = Cache4(11, 2, dim, 16, own)
    k, v = c0.k.float(), c0.v.float()
    k[:, 1] = (k[:, 1] * 2e4).clamp(-65504, 65504)
    v[::3, 0, :32] = (v[::3, 0, :32] * 3e4).clamp(-65504, 65504)
    v[5::7, 1] = 65504.0
    k[7::9, 0, 32:] *= 3e3
    c = Cache4(11, 2, dim, 16, own, k=k.half(), v=v.half())
    q = torch.randn(sum(rows), heads, dim, generator=c.g)
    q[:, heads // 2:] *= 1e-4
    q[:, :heads // 2, 32:] *= 1e-3
    q = q.half().cuda()
    got = attend(ops, c, q, rows)
    want, sizes = visible_nan(c, q, rows, c.values(c.k), c.values(c.v))      # (one of the keys is past it)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and not torch.isinf(got).any()
    near = (got.to(F64) - want).abs() <= attention_bar("f16", torch.nan_to_num(want), *sizes, dim, max(rows) * heads // 2 > 64)
    assert (near | torch.isnan(want)).all()


@pytest.mark.parametrize("heads,kv,dim,page,rows,own", [
    (16, 8, 64, 64, [1] * 64, [1500 + 20 * i for i in range(64)]),                  # long runs: warps that have more of it than others
    (8, 2, 128, 64, [1 + i % 3 for i in range(300)], [i * 7 % 150 for i in range(300)]),      # many sequences; rows that see nothing
    (32, 8, 128, 32, [300, 0, 1, 40, 700], [3000, 0, 1, 1700, 700]),                # units over several CTAs, several units a CTA
    (32, 2, 64, 16, [1 + i % 37 for i in range(70)], [1 + i % 37 + 11 * i % 90 for i in range(70)]),      # many short prompts
    (64, 1, 64, 16, [1100], [1500]),                                                # units of four rows
    (8, 2, 64, 16, [1] * 1030, [1 + i * 7 % 50 for i in range(1030)]),              # more sequences than a CTA keeps
])
def test_attention_many(ops, heads, kv, dim, page, rows, own):
    c = Cache4(sum(own), kv, dim, page, own)
    q = torch.randn(sum(rows), heads, dim, generator=c.g).half().cuda()
    got = attend(ops, c, q, rows)
    want, *sizes = attention_exact(c, q, rows)
    assert ((got.to(F64) - want).abs() <= attention_bar("f16", want, *sizes, dim, max(rows) * heads // kv > 64)).all()
    assert torch.equal(got, attend(ops, c, q, rows)) and ops.error(0) == 0


@pytest.mark.parametrize("heads,rows", WAYS)
@pytest.mark.parametrize("at,by", [([0], 30.0), ([40], 20.0), ([33, 66, 99, 130], 15.0), ([131, 132], 40.0), ([64], -20.0)])
def test_attention_scores_that_grow(ops, heads, rows, at, by):
    """scores that rise by `by` (in log2) at some keys, by a half of it or not at all in some rows: what has been summed up by then falls by as much"""
    own = [180 + n for n in rows]
    c0 = Cache4(3, 2, 64, 16, own)
    k = c0.k.float() * 0.3
    k[:, :, 0] = 0.0
    for a in at:
        for s in range(len(own)):
            k[c0.start[s] + a:c0.start[s + 1], :, 0] += 8.0
    c = Cache4(3, 2, 64, 16, own, k=k.half(), v=c0.v)
    q = torch.randn(sum(rows), heads, 64, generator=c.g)
    q[..., 0] = torch.tensor([[0.0, 0.5, 1.0, 1.0][(r + h) % 4] * by / 8 / math.log2(math.e) * 8 for r in range(sum(rows)) for h in range(heads)]).view(sum(rows), heads)
    q = q.half().cuda()
    got = attend(ops, c, q, rows)
    want, *sizes = attention_exact(c, q, rows)
    assert ((got.to(F64) - want).abs() <= attention_bar("f16", want, *sizes, 64, max(rows) * heads // 2 > 64)).all()


@pytest.mark.parametrize("heads,rows", WAYS)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_strides_alignment_and_scale(ops, heads, rows, dim):
    """rows and heads apart from each other, queries and outputs that start anywhere, another scale; what lies between the outputs, and behind the last sequence, stays"""
    own = [n + 20 for n in rows]
    c = Cache4(4, 4, dim, 48, own)
    R = sum(rows)
    wide = torch.randn(R + 3, heads + 1, dim + 7, generator=c.g).bfloat16().cuda()
    q = wide[:, :heads, 3:3 + dim]
    out_wide = torch.full((R + 3, heads, dim + 5), 9.0, dtype=torch.bfloat16, device="cuda")
    out = out_wide[:, :, 1:1 + dim]
    attend(ops, c, q, rows, scale=0.03, out=out)
    want, *sizes = attention_exact(c, q[:R], rows, scale=0.03)
    assert ((out[:R].to(F64) - want).abs() <= attention_bar("bf16", want, *sizes, dim, max(rows) * heads // 4 > 64)).all()
    assert (out[R:] == 9.0).all() and (out_wide[..., 0] == 9.0).all() and (out_wide[..., 1 + dim:] == 9.0).all()
    again = torch.full((R, heads, dim), 5.0, dtype=torch.bfloat16, device="cuda")
    attend(ops, c, q[:R].contiguous(), rows, scale=0.03, out=again)
    assert torch.equal(again, out[:R])


@pytest.mark.parametrize("heads,rows", WAYS)
def test_attention_rows_past_max_rows_and_what_lengths_say(ops, heads, rows):
    """rows past max_rows stay; lengths below zero are no tokens, past the table all that it holds; page ids outside the pool are held inside it; rows of nobody stay"""
    own = [n + 20 for n in rows]
    c = Cache4(5, 2, 64, 16, own)
    R, most = sum(rows), max(rows) - 1
    q = torch.randn(R, heads, 64, generator=c.g).half().cuda()
    whole = attend(ops, c, q, rows)
    if most:
        # the same way with fewer rows (more than 64 of a KV head, or not): rows that are computed are the same to rounding, those past it stay
        got = attend(ops, c, q, rows, max_rows=most, fill=7.0)
        want, *sizes = attention_exact(c, q, rows, max_rows=most)
        r0 = 0
        for n in rows:
            assert (got[r0 + min(n, most):r0 + n] == 7.0).all()
            here = slice(r0, r0 + min(n, most))
            bar = attention_bar("f16", want, *sizes, 64, most * heads // 2 > 64)
            assert ((got[here].to(F64) - want[here]).abs() <= bar[here]).all()
            r0 += n
    for lengths in ([-1, -2 ** 31, -7], [0, 0, 0]):
        assert (attend(ops, c, q, rows, own=lengths) == 0).all()
    full = c.pages.shape[1] * 16
    c.pages = torch.randint(0, len(c.bytes_k), c.pages.shape, dtype=torch.int32, device="cuda")
    all_held = attend(ops, c, q, rows, own=[full] * 3)
    assert torch.equal(attend(ops, c, q, rows, own=[2 ** 31 - 1, full + 1, 10 ** 9]), all_held) or torch.isnan(all_held).any()
    c.pages[0, 0], c.pages[1, 0] = -5, 2 ** 31 - 1
    held = c.pages.clone()
    held[0, 0], held[1, 0] = 0, len(c.bytes_k) - 1
    a = attend(ops, c, q, rows)
    c.pages = held
    assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(attend(ops, c, q, rows)))
    out = torch.full_like(q, 3.0)
    work = torch.empty(ops.attention_4bit_workspace(R, heads, 2, 64), dtype=torch.uint8, device="cuda")
    for at in ([0, 0, 0, 0], [0, -5, -2 ** 31, -1], [R, R, R + 5, 2 ** 31 - 1]):
        ops.attention_4bit(q, c.k_pool, c.v_pool, c.pages, c.ints(at), c.ints(own), out, work, max_rows=max(rows))
        assert (out == 3.0).all()
    assert whole.shape == out.shape and ops.error(0) == 0


@pytest.mark.parametrize("rows", [[1, 1], [90, 70]])
def test_attention_table_that_could_hold_more_than_32_bits_of_work(ops, rows):
    """the same result whatever the table could hold"""
    c = Cache4(6, 8, 64, 64, [300, 77])
    q = torch.randn(sum(rows), 8, 64, generator=c.g).half().cuda()
    small = attend(ops, c, q, rows)
    wide = torch.full((2, 2 ** 25 - 100), -1, dtype=torch.int32, device="cuda")
    wide[:, :c.pages.shape[1]] = c.pages
    c.pages = wide
    assert torch.equal(attend(ops, c, q, rows), small)


def test_pools_past_32_bits(ops):
    """pages whose bytes begin past 2^31: appended to, read, attended to as others are"""
    n_kv, dim, n_pages = 8, 128, 70000
    own = [200, 64]
    c = Cache4(7, n_kv, dim, 64, own)
    far = [torch.empty(n_pages, n_kv, 4, 9 * dim, dtype=torch.uint8, device="cuda") for _ in range(2)]
    assert far[0].numel() > 2 ** 31
    table = c.pages.clone()
    table[table < len(c.bytes_k)] += n_pages - len(c.bytes_k)
    ops.kv_append_4bit(c.k.cuda(), c.v.cuda(), far[0], far[1], table, c.ints(starts(own)), c.ints(own))
    back = torch.zeros(sum(own), n_kv, dim, device="cuda")
    ops.kv_read_4bit(far[0], far[1], table, c.ints(starts(own)), c.ints(own), back, None)
    assert torch.equal(back.to(F64), c.values(c.k))
    for rows in ([1, 1], [3, 2], [100, 20]):
        q = torch.randn(sum(rows), 16, dim, generator=c.g).half().cuda()
        near = attend(ops, c, q, rows)
        out = torch.zeros_like(q)
        work = torch.empty(ops.attention_4bit_workspace(sum(rows), 16, n_kv, dim), dtype=torch.uint8, device="cuda")
        ops.attention_4bit(q, far[0], far[1], table, c.ints(starts(rows)), c.ints(own), out, work, max_rows=max(rows))
        assert torch.equal(out, near)


# -------------------------------------------------------------------------------------------------------------- the three together
class Session:
    """Chats over a cache in 4 bits: prompts, then tokens one by one; what the definition says beside it."""

    def __init__(self, ops, heads, n_kv, dim, page, n_seqs, most, typ, layout, seed=0):
        self.ops, self.heads, self.n_kv, self.dim, self.layout, self.typ = ops, heads, n_kv, dim, layout, typ
        self.g = torch.Generator(device="cpu")
        self.g.manual_seed(seed)
        per = -(-most // page)
        self.k_pool, self.v_pool = (torch.randint(0, 256, (n_seqs * per + 1, n_kv, page // 16, 9 * dim), dtype=torch.uint8, generator=self.g).cuda() for _ in range(2))
        self.pages = torch.randperm(n_seqs * per + 1, generator=self.g)[:n_seqs * per].to(torch.int32).view(n_seqs, per).cuda()
        self.freqs = (10000.0 ** (-torch.arange(0, dim, 2, dtype=F64) / dim)).float().cuda()
        self.held = [0] * n_seqs
        self.k_rows, self.v_rows = [[] for _ in range(n_seqs)], [[] for _ in range(n_seqs)]

    def ints(self, values):
        return torch.tensor(list(values), dtype=torch.int32, device="cuda")

    def inputs(self, rows):
        x = torch.randn(sum(rows), (self.heads + 2 * self.n_kv) * self.dim, generator=self.g).to(TYPES[self.typ]).cuda()
        H, G, D = self.heads, self.n_kv, self.dim
        return x[:, :H * D].view(-1, H, D), x[:, H * D:(H + G) * D].view(-1, G, D), x[:, (H + G) * D:].view(-1, G, D)

    def call(self, q, k, v, rows, start, held, q_out, out, work, stream=None):
        self.ops.kv_append_4bit(k, v, self.k_pool, self.v_pool, self.pages, start, held, freqs=self.freqs, layout=self.layout, q=q, q_out=q_out, stream=stream)
        self.ops.attention_4bit(q_out, self.k_pool, self.v_pool, self.pages, start, held, out, work, max_rows=max(rows), stream=stream)

    def note(self, k, v, rows):
        r0 = 0
        for s, n in enumerate(rows):
            pos = torch.arange(self.held[s], self.held[s] + n, device="cuda")
            self.k_rows[s].append(coded(rotated_32(k[r0:r0 + n], pos, self.freqs, self.layout)))
            self.v_rows[s].append(coded(v[r0:r0 + n].float()))
            self.held[s] += n
            r0 += n

    def check(self, q, rows, out):
        """against the definition over what the cache has been given: the output's rounding and 2^-9 of the size of what is summed up (bf16: 2^-6): three times what the roundings come to"""
        r0 = 0
        for s, n in enumerate(rows):
            if n == 0:
                continue
            pos = torch.arange(self.held[s] - n, self.held[s], device="cuda")
            x = rotated_32(q[r0:r0 + n], pos, self.freqs, self.layout).to(TYPES[self.typ]).to(F64)
            k, v = torch.cat(self.k_rows[s]).transpose(0, 1), torch.cat(self.v_rows[s]).transpose(0, 1)
            mask = torch.arange(k.shape[1], device="cuda") > pos[:, None]
            for h in range(self.heads):
                g = h // (self.heads // self.n_kv)
                w = torch.softmax((x[:, h] @ k[g].T * self.dim ** -0.5).masked_fill(mask, -math.inf), -1)
                bar = {"f16": 2 ** -9, "bf16": 2 ** -6}[self.typ] * (w @ v[g].abs())
                assert ((out[r0:r0 + n, h].to(F64) - w @ v[g]).abs() <= bar).all()
            r0 += n

    def step(self, rows, stream=None):
        q, k, v = self.inputs(rows)
        q_out, out = (torch.full((sum(rows), self.heads, self.dim), math.nan, dtype=TYPES[self.typ], device="cuda") for _ in range(2))
        work = torch.empty(self.ops.attention_4bit_workspace(sum(rows), self.heads, self.n_kv, self.dim), dtype=torch.uint8, device="cuda")
        held = [h + n for h, n in zip(self.held, rows)]
        self.call(q, k, v, rows, self.ints(starts(rows)), self.ints(held), q_out, out, work, stream)
        self.note(k, v, rows)
        self.check(q, rows, out)


@pytest.mark.parametrize("typ,layout,dim,page", [("f16", "pairs", 128, 64), ("bf16", "halves", 64, 16), ("f16", "halves", 64, 48)])
def test_chats_over_the_cache(ops, typ, layout, dim, page):
    """prompts of several lengths in one call, a second part of one of them, drafted tokens, single tokens; the whole cache read back in the end"""
    s = Session(ops, 8, 2, dim, page, 4, 400, typ, layout)
    for rows in ([130, 3, 40, 1], [0, 200, 0, 0], [1, 1, 1, 1], [4, 0, 2, 4], [1, 1, 1, 1], [1, 0, 1, 1]):
        s.step(rows)
    R = sum(s.held)
    k, v = (torch.zeros(R, 2, dim, device="cuda") for _ in range(2))
    ops.kv_read_4bit(s.k_pool, s.v_pool, s.pages, s.ints(starts(s.held)), s.ints(s.held), k, v)
    assert torch.equal(k.to(F64), torch.cat([torch.cat(x) for x in s.k_rows])) and torch.equal(v.to(F64), torch.cat([torch.cat(x) for x in s.v_rows]))
    assert ops.error(0) == 0


@pytest.mark.parametrize("rows", [[1, 1, 1], [40, 17, 60]])
def test_captured_steps(ops, rows):
    """an append and attention in one graph, replayed with other rows and lengths in the same memory; two graphs with the same workspace, one after the other"""
    s = Session(ops, 8, 2, 128, 64, 3, 500, "f16", "pairs", seed=1)
    s.step([70, 5, 33])
    q, k, v = (x.contiguous() for x in s.inputs(rows))
    start, held = s.ints(starts(rows)), s.ints(s.held)
    work = torch.empty(ops.attention_4bit_workspace(sum(rows), 8, 2, 128), dtype=torch.uint8, device="cuda")
    graphs, outs = [], []
    stream = torch.cuda.Stream()
    q_out = torch.zeros_like(q)
    s.call(q, k, v, rows, start, s.ints([h + n for h, n in zip(s.held, rows)]), q_out, torch.zeros_like(q), work)      # (attributes are set outside of a capture; what this stores is stored again)
    torch.cuda.synchronize()
    for _ in range(2):
        out = torch.zeros_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            s.call(q, k, v, rows, start, held, q_out, out, work, stream=torch.cuda.current_stream())
        graphs.append(g)
        outs.append(out)
    for i in range(4):
        for old, new in zip((q, k, v), s.inputs(rows)):
            old.copy_(new)
        held.copy_(s.ints([h + n for h, n in zip(s.held, rows)]))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        s.note(k, v, rows)
        s.check(q, rows, outs[i % 2])


def test_two_streams_at_once(ops):
    """calls with workspaces of their own on two streams give what they give one after the other"""
    c = Cache4(8, 4, 128, 32, [3000, 700, 64, 1500])
    cases = [([1, 1, 1, 1], 16), ([300, 2, 64, 120], 16), ([1, 2, 3, 4], 32), ([1, 1, 1, 1], 4)]
    qs = [torch.randn(sum(rows), heads, 128, generator=c.g).bfloat16().cuda() for rows, heads in cases]
    want = [attend(ops, c, q, rows) for (rows, _), q in zip(cases, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    works = [[torch.empty(ops.attention_4bit_workspace(len(q), q.shape[1], 4, 128), dtype=torch.uint8, device="cuda") for q in qs] for _ in streams]
    outs = [[torch.zeros_like(q) for q in qs] for _ in range(12)]
    ints = [c.ints(starts(rows)) for rows, _ in cases]
    own = c.ints(c.own)
    torch.cuda.synchronize()
    for i in range(12):
        for j, (rows, _) in enumerate(cases):
            ops.attention_4bit(qs[j], c.k_pool, c.v_pool, c.pages, ints[j], own, outs[i][j], works[i % 2][j], max_rows=max(rows), stream=streams[i % 2])
    torch.cuda.synchronize()
    for got in outs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("words", [2, 3])
def test_a_wait_that_ran_out_is_reported_once(ops, native_lib, words):
    side = torch.cuda.Stream()
    assert ops.error(0) == 0
    assert native_lib.b2_op_give_up(0, words, 0xb0001, side.cuda_stream) == 0 and native_lib.b2_op_give_up(0, words, 0x77, side.cuda_stream) == 0
    assert ops.error(0) == 0xb0001 and ops.error(0) == 0
    for other in (0, 1, 2, 3):                                          # all files' words are taken at once
        assert native_lib.b2_op_give_up(0, other, 0x11 + other, None) == 0
    assert ops.error(0) == 0x11 and ops.error(0) == 0


def test_empty_calls(ops):
    c = Cache4(9, 2, 64, 16, [5])
    none = torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda")
    kv = torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda")
    work = torch.zeros(16, dtype=torch.uint8, device="cuda")
    ops.attention_4bit(none, c.k_pool, c.v_pool, c.pages, c.ints([0, 0]), c.ints([5]), none, work)
    ops.kv_append_4bit(kv, kv, c.k_pool, c.v_pool, c.pages, c.ints([0, 0]), c.ints([5]), q=none, q_out=none)
    ops.kv_read_4bit(c.k_pool, c.v_pool, c.pages, c.ints([0, 0]), c.ints([5]), kv, kv)
    assert ops.attention_4bit_workspace(0, 4, 2, 64) == 0
    torch.cuda.synchronize()
    assert torch.equal(c.k_pool.cpu(), c.bytes_k)
