"""The paged cache in 4 bits without a GPU: its block's layout, what the entry points refuse before anything reaches a device."""
import ctypes
import os

import pytest

torch = pytest.importorskip("torch")

from cache_4bit_util import Cache4, coded, packed, quantised
from conftest import PKG
from test_device_ops_host import OnGpu, append_args, native_calls, tensors


@pytest.fixture(scope="module")
def host(native_lib):
    lib = ctypes.CDLL(os.path.join(PKG, "lib", "libb200_hosttest.so"))
    return lib


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("keys", [True, False])
def test_block_layout(host, dim, keys):
    """every piece and scale of a block has a place of its own, all of them fill it, and it is the tests' own"""
    codes, scales = torch.zeros(16, dim, dtype=torch.uint8), torch.zeros(16, dim // 32, dtype=torch.float16)
    used = [0] * (9 * dim)
    size = 4 if keys else 2          # bytes of a piece
    place = host.b2_host_q4_key if keys else host.b2_host_q4_value
    for t in range(16):
        for w in range(dim // 2 // size):
            at = place(dim, t, w)
            assert at % size == 0
            for b in range(size):
                used[at + b] += 1
            one = codes.clone()
            one[t, 2 * size * w:2 * size * (w + 1)] = torch.arange(1, 2 * size + 1)
            assert packed(one, scales, keys)[at:at + size].tolist() == [0x21, 0x43, 0x65, 0x87][:size]
        for g in range(dim // 32):
            at = host.b2_host_q4_scale(dim, t, g)
            used[at] += 1
            used[at + 1] += 1
            one = scales.clone()
            one[t, g] = 1.0
            assert packed(codes, one, keys)[at + 1].item() == 0x3c
    assert used == [1] * (9 * dim)
    # the words that a lane takes at once, one of every group, are neighbours, 16 (8) bytes aligned; no two of a quarter (half) warp's chunks share a bank
    n, chunk = dim // 32, dim // 8
    for t in range(16):
        for w in range(4 if keys else 8):
            first = place(dim, t & ~1 if not keys else t, w)
            assert first % chunk == 0 and [place(dim, t & ~1 if not keys else t, w + (4 if keys else 8) * g) for g in range(n)] == [first + 4 * g for g in range(n)]
    for lanes in range(0, 32, 128 // chunk):
        where = [place(dim, lane >> 2, lane & 3) if keys else place(dim, 2 * (lane & 3), lane >> 2) for lane in range(lanes, lanes + 128 // chunk)]
        assert len({at // chunk % (128 // chunk) for at in where}) == len(where)


def test_definition():
    """the largest entry comes back but for its scale's rounding, the others within half a step, those near its negative within one"""
    x = torch.randn(50, 128, dtype=torch.float64)
    y = coded(x)
    g, back = x.unflatten(-1, (-1, 32)), y.unflatten(-1, (-1, 32))
    step = quantised(x)[1].double().abs()[..., None]
    assert ((back - g).abs() <= step * (1 + 16 * 2 ** -11)).all()
    assert (((back - g).abs() <= step * (0.5 + 8 * 2 ** -11)) | (back.abs() >= 6.99 * step)).all()
    m = g.abs().argmax(-1, keepdim=True)
    assert ((back.gather(-1, m) / g.gather(-1, m) - 1).abs() <= 2 ** -11).all()


def test_a_cache_holds_its_rows(host):
    c = Cache4(1, 2, 64, 48, [5, 0, 50], device="cpu", fill=0)
    for pool, rows, place, n in ((c.bytes_k, c.k, host.b2_host_q4_key, 8), (c.bytes_v, c.v, host.b2_host_q4_value, 4)):
        codes, scales = quantised(rows)
        for s, t in ((0, 0), (0, 4), (2, 0), (2, 33), (2, 49)):
            block, at = pool[c.table[s, t // 48].item(), 1, t % 48 // 16], c.start[s] + t
            for w in range(64 // n):
                b = place(64, t % 16, w)
                assert block[b:b + n // 2].tolist() == [int(codes[at, 1, n * w + e] + 16 * codes[at, 1, n * w + e + 1]) for e in range(0, n, 2)]
            for g in range(2):
                b = host.b2_host_q4_scale(64, t % 16, g)
                assert block[b:b + 2].view(torch.float16).item() == scales[at, 1, g].item()
        last = pool[c.table[0, 0].item(), :, 0]                  # five tokens of 16
        assert (last != 0).sum() <= 2 * 5 * (32 + 4) and (pool[c.table[0, 0].item(), :, 1:] == 0).all()


def read_args(**over):
    from llama_cpp import _cabi
    where = _cabi.B2RaggedPages(64, 64, 64, 4, 10, 4, 2, 5, 16)
    args = _cabi.B2KvRead4Bit(64, 64, 64, 64, 128, 64, 128, 64, 2, 64, _cabi.B2_TYPE_F16)
    for k, v in over.items():
        setattr(where if hasattr(where, k) else args, k, v)
    return where, args


def attention_args(**over):
    from llama_cpp import _cabi
    where = _cabi.B2RaggedPages(64, 64, 64, 4, 10, 4, 2, 5, 16)
    args = _cabi.B2Attention4Bit(64, 64, 64, 64, 64, 1 << 30, 256, 64, 256, 64, 1, 4, 2, 64, _cabi.B2_TYPE_F16, 0.125)
    for k, v in over.items():
        setattr(where if hasattr(where, k) else args, k, v)
    return where, args


WHERE_REFUSALS = [(dict(n_rows=-1), "negative"), (dict(n_seqs=70000), "65535"), (dict(block_tokens=24), "block_tokens"), (dict(max_pages=0), "max_pages"), (dict(n_pages=0), "n_pages"),
                  (dict(max_pages=2 ** 28, block_tokens=32), "32 bits"), (dict(table_stride=3), "table_stride"), (dict(row_start=None), "null"), (dict(pages=66), "aligned")]
APPEND_REFUSALS = WHERE_REFUSALS + [
    (dict(in_type=2), "f32, f16 or bf16"), (dict(cache_type=0), "q_out must be f16 or bf16"), (dict(n_kv=0), "n_kv"), (dict(head_dim=96, rot_dims=0), "64 or 128"),
    (dict(head_dim=256), "64 or 128"), (dict(rot_dims=66), "rot_dims"), (dict(rot_dims=3), "rot_dims"), (dict(layout=2), "layout"), (dict(amplitude=float("nan")), "amplitude"),
    (dict(first_pos=-1), "first_pos"), (dict(n_head=0), "n_head"), (dict(n_head=2 ** 26), "32 bits"), (dict(k=None), "null"), (dict(q_out=None), "null"), (dict(freqs=None), "null"), (dict(v=62), "aligned"),
    (dict(k_pool=72), "16-byte"), (dict(v_pool=66), "16-byte")]
READ_REFUSALS = WHERE_REFUSALS + [(dict(out_type=2), "f32, f16 or bf16"), (dict(head_dim=96), "64 or 128"), (dict(n_kv=0), "n_kv"), (dict(n_kv=2 ** 25), "32 bits"),
                                  (dict(k_pool=None), "null"), (dict(v_pool=None), "null"), (dict(k_pool=72), "16-byte"), (dict(v=65), "aligned")]
ATTENTION_REFUSALS = WHERE_REFUSALS + [
    (dict(head_dim=96), "head_dim"), (dict(n_head=5), "multiple"), (dict(n_kv=0), "multiple"), (dict(n_head=130), "64 heads"), (dict(type=0), "f16 or bf16"), (dict(max_rows=0), "max_rows"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=2.0 ** -41), "scale"), (dict(scale=1.1 * 2 ** 40), "scale"), (dict(scale=-1.0), "scale"), (dict(n_rows=2 ** 30), "32 bits"), (dict(max_rows=2 ** 30), "32 bits"), (dict(q=None), "null"),
    (dict(workspace=None), "null"), (dict(v_pool=None), "null"), (dict(k_pool=72), "16-byte"), (dict(workspace=72), "16-byte"), (dict(q=65), "aligned"), (dict(out=65), "aligned"),
    (dict(workspace_bytes=100), "workspace holds 100 bytes")]


@pytest.mark.parametrize("name,make,refusals", [("b2_kv_append_4bit", append_args, APPEND_REFUSALS), ("b2_kv_read_4bit", read_args, READ_REFUSALS),
                                                ("b2_attention_4bit", attention_args, ATTENTION_REFUSALS)])
def test_refusals(native_lib, name, make, refusals):
    for over, why in refusals:
        where, args = make(**over)
        assert getattr(native_lib, name)(0, ctypes.byref(where), ctypes.byref(args), None) < 0, over
        text = native_lib.b2_last_error().decode()
        assert why in text and name in text, (over, text)
    assert getattr(native_lib, name)(0, None, None, None) < 0


def test_nothing_to_do_is_no_error(native_lib):
    for over in (dict(n_rows=0), dict(n_seqs=0)):
        for name, make in (("b2_kv_append_4bit", append_args), ("b2_kv_read_4bit", read_args), ("b2_attention_4bit", attention_args)):
            where, args = make(row_start=None, lengths=None, pages=None, k_pool=None, **over)
            assert getattr(native_lib, name)(0, ctypes.byref(where), ctypes.byref(args), None) == 0
    where, args = read_args(k=None, v=None)
    assert native_lib.b2_kv_read_4bit(0, ctypes.byref(where), ctypes.byref(args), None) == 0


def test_workspace(native_lib):
    from llama_cpp.device_ops import attention_4bit_workspace as need
    assert need(0, 8, 8, 64) == 0 and need(1, 32, 8, 128) > 0
    for rows, heads, kv, dim in [(1, 8, 8, 64), (17, 32, 8, 128), (256, 32, 8, 128), (5000, 8, 8, 128), (2 ** 26 - 1, 32, 8, 128)]:
        assert need(rows, heads, kv, dim) >= need(1, heads, kv, dim)
    for bad in [(4, 8, 3, 64), (4, 8, 8, 96), (2 ** 30, 32, 8, 128)]:
        with pytest.raises(RuntimeError):
            need(*bad)
    with pytest.raises(ValueError):
        need(2 ** 31, 8, 8, 64)


def good_cache(f, i):
    return dict(k_pool=f(9, 2, 1, 576, dtype=torch.uint8), v_pool=f(9, 2, 1, 576, dtype=torch.uint8), pages=i(3, 4), row_start=i(4), lengths=i(3))


CACHE_REFUSALS = [("v_pool", lambda f, i: f(9, 2, 2, 576, dtype=torch.uint8), "shape"), ("k_pool", lambda f, i: f(9, 2, 1, 576), "dtype"),
                  ("pages", lambda f, i: i(2, 4), "shape"), ("lengths", lambda f, i: i(3, 1), "dimension"), ("row_start", lambda f, i: i(3), "shape"),
                  ("pages", lambda f, i: f(3, 4, dtype=torch.int64), "dtype"), ("v_pool", lambda f, i: f(9, 2, 1, 576, dtype=torch.uint8, device=1), "device 1")]


def test_python_refusals_of_append(native_lib):
    from llama_cpp.device_ops import kv_append_4bit
    f, i = tensors()
    good = dict(k=f(5, 2, 64), v=f(5, 2, 64), **good_cache(f, i), q=f(5, 4, 64), q_out=f(5, 4, 64), freqs=f(32, dtype=torch.float32))
    for over, why in [({n: make(f, i)}, why) for n, make, why in CACHE_REFUSALS] + [
            (dict(k=f(5, 128)), "shape"), (dict(k=f(5, 2, 64, dtype=torch.uint8)), "dtype"), (dict(v=f(5, 2, 64, dtype=torch.bfloat16)), "dtype"), (dict(k=f(5, 3, 64)), "go together"),
            (dict(k_pool=f(9, 2, 1, 500, dtype=torch.uint8), v_pool=f(9, 2, 1, 500, dtype=torch.uint8)), "9 \\* 64"), (dict(layout="other"), "layout"), (dict(q_out=None), "go together"),
            (dict(q=f(5, 4, 32)), "go together"), (dict(q_out=f(5, 4, 64, dtype=torch.float32)), "dtype"), (dict(q_out=f(5, 4, 64, dtype=torch.uint8)), "dtype"),
            (dict(k=torch.zeros(5, 2, 64).half()), "not on a CUDA device"), (dict(v=OnGpu(torch.zeros(5, 2, 128).half()[..., ::2])), "contiguous"), (dict(freqs=f(32)), "dtype")]:
        with pytest.raises(ValueError, match=why):
            kv_append_4bit(**{**good, **over})
    with pytest.raises(RuntimeError, match="rot_dims"):
        kv_append_4bit(**{**good, "freqs": f(40, dtype=torch.float32)})


def test_python_refusals_of_read(native_lib):
    from llama_cpp.device_ops import kv_read_4bit
    f, i = tensors()
    good = dict(**good_cache(f, i), k=f(5, 2, 64), v=f(5, 2, 64))
    for over, why in [({n: make(f, i)}, why) for n, make, why in CACHE_REFUSALS] + [
            (dict(k=None, v=None), "one of k and v"), (dict(v=f(5, 2, 64, dtype=torch.float32)), "dtype"), (dict(v=f(6, 2, 64)), "shape"), (dict(k=f(5, 3, 64)), "go together"),
            (dict(k=f(5, 2, 64, dtype=torch.uint8)), "dtype"), (dict(k=None, v=f(5, 2, 128)), "go together")]:
        with pytest.raises(ValueError, match=why):
            kv_read_4bit(**{**good, **over})


def test_python_refusals_of_attention(native_lib):
    from llama_cpp.device_ops import attention_4bit
    f, i = tensors()
    good = dict(q=f(5, 4, 64), **good_cache(f, i), out=f(5, 4, 64), workspace=f(10, dtype=torch.uint8))
    for over, why in [({n: make(f, i)}, why) for n, make, why in CACHE_REFUSALS] + [
            (dict(q=f(5, 4, 64, dtype=torch.float32)), "dtype"), (dict(q=f(5, 3, 64)), "go together"), (dict(out=f(5, 4, 32)), "shape"), (dict(out=f(5, 4, 64, dtype=torch.bfloat16)), "dtype"),
            (dict(workspace=None), "workspace"), (dict(workspace=f(10, device=1)), "workspace"),
            (dict(k_pool=f(9, 0, 1, 576, dtype=torch.uint8), v_pool=f(9, 0, 1, 576, dtype=torch.uint8)), "go together")]:
        with pytest.raises(ValueError, match=why):
            attention_4bit(**{**good, **over})
    with pytest.raises(RuntimeError, match="workspace holds 10 bytes"):
        attention_4bit(**good)
    with pytest.raises(RuntimeError, match="max_rows"):
        attention_4bit(**good, max_rows=0)


def test_native_calls_pass_what_the_python_ones_pass(native_lib, monkeypatch):
    """every argument reaches the entry points alike, whether the call is made in native code or in Python"""
    import struct
    from llama_cpp import _cabi, device_ops as ops
    calls = native_calls()
    seen = []
    where, *kinds = (struct.Struct("@" + "".join({ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_float: "f"}[t] for _, t in k._fields_))
                     for k in (_cabi.B2RaggedPages, _cabi.B2KvAppend, _cabi.B2KvRead4Bit, _cabi.B2Attention4Bit))

    def entry(kind):
        def f(device, w, args, stream):
            seen.append((device, where.unpack(ctypes.string_at(w, where.size)), kind.unpack(ctypes.string_at(args, kind.size)), stream))
            return 0
        return ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p)(f)

    names = ("kv_append_4bit", "kv_read_4bit", "attention_4bit")
    Lib = type("Lib", (), {"b2_" + n: staticmethod(entry(k)) for n, k in zip(names, kinds)})
    f, i = tensors()
    g = lambda *s, dtype=torch.float16: f(*s, dtype=dtype, device=3)
    j = lambda *s: g(*s, dtype=torch.int32)
    wide = OnGpu(torch.zeros(5, 9, 64).half(), 3)
    part = lambda a, b: OnGpu(wide.t[:, a:b], 3)
    cache = dict(k_pool=g(9, 2, 3, 576, dtype=torch.uint8), v_pool=g(9, 2, 3, 576, dtype=torch.uint8), pages=j(3, 4), row_start=j(4), lengths=j(3))
    out, work = g(5, 4, 64), g(1000)
    freqs, q_out, k32 = g(20, dtype=torch.float32), g(5, 5, 64), g(5, 2, 64, dtype=torch.float32)
    jobs = [lambda: ops.kv_append_4bit(part(0, 2), part(2, 4), **cache, freqs=freqs, layout="halves", first_pos=77, amplitude=1.5, q=part(4, 9), q_out=q_out, stream=1234),
            lambda: ops.kv_append_4bit(k32, k32, **{**cache, "pages": OnGpu(cache["pages"].t[:, :2], 3)}),
            lambda: ops.kv_read_4bit(**cache, k=part(0, 2), v=part(2, 4), stream=7),
            lambda: ops.kv_read_4bit(**cache, k=None, v=k32),
            lambda: ops.attention_4bit(part(0, 4), *cache.values(), out, work, max_rows=2, stream=5),
            lambda: ops.attention_4bit(part(4, 8), *cache.values(), out, work, scale=0.3)]
    monkeypatch.setattr(_cabi, "load_library", lambda path=None: Lib)
    for job in jobs:
        both = []
        for native in (None, True, False):                               # (None: dtypes are met)
            monkeypatch.setattr(ops, "_entries", {n: (None, None) for n in names} if native is False else {})
            made = []
            if native:
                for n in names:
                    ops._entries[n] = ((lambda fn: lambda *a: made.append(fn(*a)) or made[-1])(getattr(calls, n)), ctypes.cast(getattr(Lib, "b2_" + n), ctypes.c_void_p).value)
            seen.clear()
            job()
            assert len(seen) == 1 and (not native or made == [0])
            both.append(seen[0])
        assert both[1] == both[2] and both[1][0] == 3
