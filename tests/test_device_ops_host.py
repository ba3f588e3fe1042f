"""What the operators over device tensors refuse, before anything reaches a device (no GPU here): the C entry points on sizes and pointers, the Python
ones on tensors."""
import ctypes
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama-fastapi-k8s-gpu_b200")


class OnGpu:
    """A CPU tensor that says it is on a CUDA device: for calls that must be refused."""

    def __init__(self, t, device=0):
        self.t, self.device_no = t, device

    def get_device(self):
        return self.device_no

    def __getattr__(self, name):
        return getattr(self.t, name)


def append_args(**over):
    from llama_cpp import _cabi
    where = _cabi.B2RaggedPages(64, 64, 64, 4, 10, 4, 2, 5, 16)
    args = _cabi.B2KvAppend(64, 64, 64, 64, 64, 64, 64, 128, 64, 128, 64, 256, 64, 256, 64, 0, _cabi.B2_TYPE_F32, _cabi.B2_TYPE_F16, 4, 2, 64, 64, 0, 1.0)
    for k, v in over.items():
        setattr(where if hasattr(where, k) else args, k, v)
    return where, args


APPEND_REFUSALS = [
    (dict(n_rows=-1), "negative"), (dict(n_seqs=70000), "65535"), (dict(block_tokens=24), "block_tokens"), (dict(block_tokens=0), "block_tokens"),
    (dict(max_pages=0), "max_pages"), (dict(n_pages=0), "n_pages"), (dict(max_pages=2 ** 28, block_tokens=32), "32 bits"), (dict(table_stride=3), "table_stride"),
    (dict(row_start=None), "null"), (dict(pages=66), "aligned"), (dict(in_type=2), "f32, f16 or bf16"), (dict(cache_type=0), "f16 or bf16"), (dict(n_kv=0), "n_kv"),
    (dict(head_dim=63, rot_dims=0), "head_dim"), (dict(head_dim=2048), "head_dim"), (dict(rot_dims=66), "rot_dims"), (dict(rot_dims=3), "rot_dims"),
    (dict(layout=2), "layout"), (dict(amplitude=float("nan")), "amplitude"), (dict(first_pos=-1), "first_pos"), (dict(n_head=0), "n_head"),
    (dict(k=None), "null"), (dict(q_out=None), "null"), (dict(freqs=None), "null"), (dict(v=62), "aligned"), (dict(k_pool=63), "aligned"),
]


@pytest.mark.parametrize("over,why", APPEND_REFUSALS)
def test_append_refusals(native_lib, over, why):
    where, args = append_args(**over)
    assert native_lib.b2_kv_append(0, ctypes.byref(where), ctypes.byref(args), None) < 0
    assert why in native_lib.b2_last_error().decode()


def test_nothing_to_do_is_no_error(native_lib):
    for over in (dict(n_rows=0), dict(n_seqs=0)):
        where, args = append_args(row_start=None, lengths=None, pages=None, k=None, v=None, **over)
        assert native_lib.b2_kv_append(0, ctypes.byref(where), ctypes.byref(args), None) == 0
        where, args = shared_args(row_start=None, lengths=None, pages=None, q=None, **over)
        assert native_lib.b2_attention_shared_prefix(0, ctypes.byref(where), ctypes.byref(args), None) == 0
    assert native_lib.b2_token_logprobs(0, None, 0, 5, 0, 5, None, None, None, 0, None, None, None) == 0
    assert native_lib.b2_kv_append(0, None, None, None) < 0 and native_lib.b2_attention_shared_prefix(0, None, None, None) < 0


def shared_args(**over):
    from llama_cpp import _cabi
    where = _cabi.B2RaggedPages(64, 64, 64, 4, 10, 4, 2, 5, 16)
    args = _cabi.B2SharedPrefix(64, 64, 64, 64, 64, 64, 1 << 30, 256, 64, 256, 64, 40, 1, 4, 2, 64, _cabi.B2_TYPE_F16, 0.125)
    for k, v in over.items():
        setattr(where if hasattr(where, k) else args, k, v)
    return where, args


SHARED_REFUSALS = [
    (dict(block_tokens=40), "block_tokens"), (dict(head_dim=96), "head_dim"), (dict(head_dim=256), "head_dim"), (dict(n_head=5), "multiple"), (dict(n_kv=0), "multiple"),
    (dict(n_head=130), "64 heads"), (dict(type=0), "f16 or bf16"), (dict(n_prefix=-1), "n_prefix"), (dict(max_rows=0), "max_rows"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(n_pages=2 ** 31 - 1), "32 bits"),
    (dict(n_rows=2 ** 30), "32 bits"), (dict(q=None), "null"), (dict(workspace=None), "null"), (dict(prefix_pages=None), "null"), (dict(k_pool=72), "16-byte"),
    (dict(workspace=72), "16-byte"), (dict(q=65), "aligned"), (dict(workspace_bytes=100), "workspace holds 100 bytes"),
]


@pytest.mark.parametrize("over,why", SHARED_REFUSALS)
def test_shared_prefix_refusals(native_lib, over, why):
    where, args = shared_args(**over)
    assert native_lib.b2_attention_shared_prefix(0, ctypes.byref(where), ctypes.byref(args), None) < 0
    assert why in native_lib.b2_last_error().decode()


def test_shared_prefix_workspace_covers_every_prefix(native_lib):
    """the partial results of any prefix length fit what the sizes alone ask for (the same cut of the work, in Python)"""
    from llama_cpp.device_ops import attention_shared_prefix_workspace as need
    for rows, heads, kv, dim in [(1, 8, 8, 64), (17, 32, 8, 128), (64, 32, 8, 128), (65, 64, 1, 64), (256, 32, 8, 128), (1000, 32, 4, 64), (5000, 8, 8, 128)]:
        group = heads // kv
        slots = need(rows, heads, kv, dim) // (rows * heads * (dim + 2) * 4)
        if rows * group <= 64:
            assert slots >= 32
            continue
        units = kv * -(-rows * group // 256)
        for blocks in list(range(1, 700)) + [8000, 100000]:
            run = -(-units * blocks // 148)
            assert max(((u + 1) * blocks - 1) // run - u * blocks // run + 1 for u in range(units)) <= slots
    assert need(0, 8, 8, 64) == 0
    with pytest.raises(RuntimeError):
        need(4, 8, 3, 64)


def own_slots(rows, heads, kv):
    """partial results of own tokens: splits of the fewest CTAs that so many rows can be"""
    tiles, n = -(-rows * (heads // kv) // 64) * kv, 1
    while 2 * n <= 8 and tiles * 2 * n <= 2 * 148:
        n *= 2
    return n


def prefix_cut(units, blocks, sms):
    """the runs of key blocks that CTAs take: (length, cut unit by unit)"""
    run = -(-units * blocks // sms)
    parts = sms // units if units <= sms else 1
    each = -(-blocks // parts)
    return (each, True) if units <= sms and each <= run + 3 else (run, False)


@pytest.mark.parametrize("rows,heads,kv,dim", [(1, 8, 8, 64), (8, 32, 8, 128), (33, 8, 8, 128), (9, 32, 8, 128), (12, 32, 8, 64), (16, 32, 8, 128), (5, 32, 4, 64), (17, 32, 8, 128),
                                               (64, 32, 8, 128), (1, 64, 1, 64), (65, 64, 1, 64), (256, 32, 8, 128), (720, 32, 4, 64), (1000, 32, 4, 64), (5000, 8, 8, 128), (40, 149, 149, 64)])
def test_prefix_results_stay_ahead_of_the_own_tokens(native_lib, rows, heads, kv, dim):
    """The prefix's partial results of every length, cut end to end or unit by unit for any number of SMs that it may get, lie in the slots ahead of the own tokens'."""
    from llama_cpp.device_ops import attention_shared_prefix_workspace as need
    one = rows * heads * (dim + 2) * 4
    total, rest = divmod(need(rows, heads, kv, dim), one)
    assert rest == 16
    prefix, group = total - own_slots(rows, heads, kv), heads // kv
    if rows * group <= 32:
        assert prefix == 32                                       # (that kernel's splits, 32 at most)
        return
    units = kv * -(-rows * group // 256)
    most = 0
    for blocks in [*range(1, 400), 1000, 8000, 100000]:
        for sms in range(148, 20, -8):
            run, per_unit = prefix_cut(units, blocks, sms)
            if per_unit:
                most = max(most, -(-blocks // run))
                assert units * -(-blocks // run) <= sms
            else:
                most = max(most, *(((u + 1) * blocks - 1) // run - u * blocks // run + 1 for u in range(units)))
    assert most <= prefix


@pytest.mark.parametrize("sizes", [(2 ** 31 - 1, 512, 512, 128), (2 ** 30, 1024, 1024, 64), (2 ** 28, 4096, 4096, 64), (2 ** 27, 64, 1, 64), (2 ** 26, 32, 8, 128), (2 ** 32 + 5, 32, 8, 128),
                                   (-1, 32, 8, 128), (5, 2 ** 32 + 32, 8, 128)])
def test_shared_prefix_workspace_refusals(native_lib, sizes):
    """Sizes that the call itself refuses have no workspace either. In a process of its own: a division by a wrapped product of the sizes ends it."""
    code = ("import sys\nsys.path.insert(0, sys.argv[1])\nfrom llama_cpp.device_ops import attention_shared_prefix_workspace as need\n"
            "try:\n    print(need(*eval(sys.argv[2])))\nexcept (RuntimeError, ValueError) as e:\n    print('refused:', e)")
    r = subprocess.run([sys.executable, "-c", code, PACKAGE, repr(sizes)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.startswith("refused:"), (r.returncode, r.stdout, r.stderr[-500:])


def test_shared_prefix_workspace_of_the_largest_sizes(native_lib):
    """the largest that a call takes, rows * heads just inside 32 bits: there are two slots of partial results at least, prefix and own tokens, and nothing wraps"""
    from llama_cpp.device_ops import attention_shared_prefix_workspace as need
    for rows, heads, kv, dim in [(2 ** 26 - 1, 32, 8, 128), (2 ** 31 - 1, 1, 1, 64), ((2 ** 31 - 1) // 65535, 65535, 65535, 64), (1, 64 * 65535, 65535, 128)]:
        assert need(rows, heads, kv, dim) >= 2 * rows * heads * (dim + 2) * 4


def test_tables_of_nearly_32_bits_of_tokens_are_refused(native_lib):
    """the kernels count on from the last token to the end of its tile"""
    for pages, ok in ((2 ** 27 - 1, False), (2 ** 27 - 256, False), (2 ** 27 - 257, True)):
        for args, call in ((append_args, native_lib.b2_kv_append), (shared_args, native_lib.b2_attention_shared_prefix)):
            where, x = args(max_pages=pages, block_tokens=16, table_stride=pages, n_rows=0)
            assert (call(0, ctypes.byref(where), ctypes.byref(x), None) == 0) == ok
            assert ok or "32 bits" in native_lib.b2_last_error().decode()


LOGPROB_REFUSALS = [
    (dict(type=2), "f32, f16 or bf16"), (dict(n_rows=-1), "n_rows"), (dict(n_vocab=0), "n_vocab"), (dict(row_stride=99), "row_stride"), (dict(n_top=65), "n_top"),
    (dict(n_top=-1), "n_top"), (dict(logits=None), "null"), (dict(tokens=None), "null"), (dict(top_id=None), "null"), (dict(logits=66), "aligned"), (dict(entropy=66), "aligned"),
]


@pytest.mark.parametrize("over,why", LOGPROB_REFUSALS)
def test_logprob_refusals(native_lib, over, why):
    a = dict(logits=64, type=0, row_stride=100, n_rows=3, n_vocab=100, tokens=64, logprob=64, entropy=64, n_top=5, top_logprob=64, top_id=64)
    a.update(over)
    assert native_lib.b2_token_logprobs(0, *a.values(), None) < 0
    assert why in native_lib.b2_last_error().decode()


# ------------------------------------------------------------------------------------------------------------ tensors
def tensors():
    f = lambda *s, dtype=torch.float16, device=0: OnGpu(torch.zeros(*s, dtype=dtype), device)
    i = lambda *s: f(*s, dtype=torch.int32)
    return f, i


def test_python_refusals_of_append(native_lib):
    from llama_cpp.device_ops import kv_append
    f, i = tensors()
    good = dict(k=f(5, 2, 64), v=f(5, 2, 64), k_pool=f(9, 2, 16, 64), v_pool=f(9, 2, 16, 64), pages=i(3, 4), row_start=i(4), lengths=i(3), q=f(5, 4, 64), q_out=f(5, 4, 64),
                freqs=f(32, dtype=torch.float32))
    for over, why in [(dict(k=f(5, 128)), "shape"), (dict(k=f(5, 2, 64, dtype=torch.int32)), "dtype"), (dict(v=f(5, 2, 64, dtype=torch.bfloat16)), "dtype"),
                      (dict(v=f(4, 2, 64)), "shape"), (dict(k=f(5, 3, 64)), "go together"), (dict(v_pool=f(9, 2, 32, 64)), "shape"),
                      (dict(k_pool=f(9, 2, 16, 64, dtype=torch.float32)), "dtype"), (dict(pages=i(2, 4)), "shape"), (dict(lengths=i(3, 1)), "dimension"),
                      (dict(row_start=i(3)), "shape"), (dict(pages=f(3, 4, dtype=torch.int64)), "dtype"), (dict(layout="other"), "layout"), (dict(q_out=None), "go together"),
                      (dict(q=f(5, 4, 32)), "go together"), (dict(q_out=f(5, 4, 64, dtype=torch.bfloat16)), "dtype"), (dict(v=f(5, 2, 64, device=1)), "device 1"),
                      (dict(k=torch.zeros(5, 2, 64).half()), "not on a CUDA device"), (dict(v=OnGpu(torch.zeros(5, 2, 128).half()[..., ::2])), "contiguous"),
                      (dict(k_pool=OnGpu(torch.zeros(9, 16, 2, 64).half().transpose(1, 2))), "contiguous"), (dict(freqs=f(32)), "dtype"),
                      (dict(freqs=f(32, 1, dtype=torch.float32)), "shape")]:
        a = {**good, **over}
        with pytest.raises(ValueError, match=why):
            kv_append(**a)
    for freqs, amplitude, why in ((f(40, dtype=torch.float32), 1.0, "rot_dims"), (None, float("inf"), "amplitude")):      # what the C side refuses comes as its own error
        with pytest.raises(RuntimeError, match=why):
            kv_append(good["k"], good["v"], good["k_pool"], good["v_pool"], good["pages"], good["row_start"], good["lengths"], freqs=freqs, amplitude=amplitude)


def test_python_refusals_of_shared_prefix(native_lib):
    from llama_cpp.device_ops import attention_shared_prefix
    f, i = tensors()
    order = ("q", "k_pool", "v_pool", "prefix_pages", "n_prefix", "pages", "row_start", "lengths", "out", "workspace")
    good = dict(q=f(5, 4, 64), k_pool=f(9, 2, 16, 64), v_pool=f(9, 2, 16, 64), prefix_pages=i(2), n_prefix=30, pages=i(3, 4), row_start=i(4), lengths=i(3), out=f(5, 4, 64),
                workspace=f(10, dtype=torch.uint8))
    for over, why in [(dict(q=f(5, 4, 64, dtype=torch.float32)), "dtype"), (dict(q=f(5, 4, 64, dtype=torch.bfloat16)), "the cache float16"), (dict(q=f(5, 3, 64)), "go together"),
                      (dict(out=f(5, 4, 32)), "shape"), (dict(n_prefix=33), "does not fit"), (dict(n_prefix=-1), "does not fit"), (dict(workspace=None), "workspace"),
                      (dict(workspace=f(10, device=1)), "workspace"), (dict(prefix_pages=i(2, 1)), "shape"), (dict(k_pool=f(9, 0, 16, 64), v_pool=f(9, 0, 16, 64)), "go together")]:
        a = {**good, **over}
        with pytest.raises(ValueError, match=why):
            attention_shared_prefix(*(a[n] for n in order))
    with pytest.raises(RuntimeError, match="workspace holds 10 bytes"):
        attention_shared_prefix(*(good[n] for n in order))
    with pytest.raises(RuntimeError, match="max_rows"):
        attention_shared_prefix(*(good[n] for n in order), max_rows=0)


def test_python_refusals_of_logprobs(native_lib):
    from llama_cpp.device_ops import token_logprobs
    f, i = tensors()
    good = dict(logits=f(5, 100), tokens=i(5), logprob=f(5, dtype=torch.float32), entropy=f(5, dtype=torch.float32), top_logprob=f(5, 3, dtype=torch.float32), top_id=i(5, 3))
    for over, why in [(dict(logits=f(500)), "shape"), (dict(logits=i(5, 100)), "dtype"), (dict(tokens=i(4)), "shape"), (dict(tokens=None), "go together"),
                      (dict(logprob=f(5)), "dtype"), (dict(entropy=f(6, dtype=torch.float32)), "shape"), (dict(top_id=None), "go together"), (dict(top_id=i(15)), "shape"),
                      (dict(top_logprob=f(5, 4, dtype=torch.float32)), "shape"), (dict(logits=OnGpu(torch.zeros(100, 5).half().t())), "contiguous")]:
        with pytest.raises(ValueError, match=why):
            token_logprobs(**{**good, **over})
    with pytest.raises(RuntimeError, match="n_top"):
        token_logprobs(**{**good, "top_logprob": f(5, 65, dtype=torch.float32), "top_id": i(5, 65)})


# ------------------------------------------------------------------------------------------------------ the native calls
def native_calls():
    from llama_cpp import _cabi
    calls = _cabi.load_calls()
    if calls is None:
        pytest.skip("the native calls are not built for this interpreter")
    return calls


def test_native_calls_pass_what_the_python_ones_pass(native_lib, monkeypatch):
    """every argument reaches the entry point alike, whether the call is made in native code or in Python"""
    import struct
    from llama_cpp import _cabi, device_ops as ops
    calls = native_calls()
    seen = []
    where, append, shared = (struct.Struct("@" + "".join({ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_float: "f"}[t] for _, t in s._fields_))
                             for s in (_cabi.B2RaggedPages, _cabi.B2KvAppend, _cabi.B2SharedPrefix))

    def entry(kind):
        def f(device, w, args, stream):
            seen.append((device, where.unpack(ctypes.string_at(w, where.size)), kind.unpack(ctypes.string_at(args, kind.size)), stream))
            return 0
        return ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p)(f)

    def flat(*a):
        seen.append(a)
        return 0

    class Lib:
        b2_kv_append, b2_attention_shared_prefix = entry(append), entry(shared)
        b2_token_logprobs = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p,
                                             ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p)(flat)

    f, i = tensors()
    wide = OnGpu(torch.zeros(5, 9, 64).half(), 3)
    part = lambda a, b: OnGpu(wide.t[:, a:b], 3)
    g = lambda *s, dtype=torch.float16: f(*s, dtype=dtype, device=3)
    j = lambda *s: g(*s, dtype=torch.int32)
    pools = dict(k_pool=g(9, 2, 16, 64), v_pool=g(9, 2, 16, 64), pages=j(3, 4), row_start=j(4), lengths=j(3))
    jobs = [lambda: ops.kv_append(part(0, 2), part(2, 4), **pools, freqs=g(20, dtype=torch.float32), layout="halves", first_pos=77, amplitude=1.5, q=part(4, 9), q_out=g(5, 5, 64), stream=1234),
            lambda: ops.kv_append(part(0, 2), part(2, 4), **{**pools, "pages": OnGpu(pools["pages"].t[:, :2], 3)}),
            lambda: ops.attention_shared_prefix(part(0, 4), pools["k_pool"], pools["v_pool"], j(2), 30, pools["pages"], pools["row_start"], pools["lengths"], g(5, 4, 64), g(1000), max_rows=2, stream=5),
            lambda: ops.attention_shared_prefix(part(0, 4), pools["k_pool"], pools["v_pool"], None, 0, pools["pages"], pools["row_start"], pools["lengths"], g(5, 4, 64), None, scale=0.3),
            lambda: ops.token_logprobs(OnGpu(torch.zeros(5, 20)[:, :18], 3), j(5), g(5, dtype=torch.float32), g(5, dtype=torch.float32), g(5, 3, dtype=torch.float32), j(5, 3), stream=9),
            lambda: ops.token_logprobs(g(1, 20), entropy=g(1, dtype=torch.float32))]
    held = []
    real = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, **k: held.append(real(*a, **k)) or held[-1])      # (addresses stay taken, so that they can be compared)
    monkeypatch.setattr(_cabi, "load_library", lambda path=None: Lib)
    for job in jobs:
        monkeypatch.setattr(ops, "_entries", {})
        job()                                                           # (dtypes are met)
        for native in (True, False):
            monkeypatch.setattr(ops, "_entries", {} if native else {n: (None, None) for n in ("kv_append", "attention_shared_prefix", "token_logprobs")})
            seen.clear()
            made = []
            if native:
                for name in ("kv_append", "attention_shared_prefix", "token_logprobs"):
                    fn = getattr(calls, name)
                    ops._entries[name] = ((lambda fn: lambda *a: made.append(fn(*a)) or made[-1])(fn), ctypes.cast(getattr(Lib, "b2_" + name), ctypes.c_void_p).value)
            start = len(held)
            job()
            new = {t.data_ptr(): n for n, t in enumerate(held[start:])}     # a call's own tensors by their order
            call = [tuple(tuple(new.get(v, v) for v in part) if isinstance(part, tuple) else new.get(part, part) for part in one) for one in seen]
            assert len(call) == 1 and (not native or made == [0])
            if native:
                want = call
            else:
                assert call == want
