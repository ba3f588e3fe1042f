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
