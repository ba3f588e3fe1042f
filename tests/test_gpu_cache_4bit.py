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
