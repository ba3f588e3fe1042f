"""The device operators on the engines' own paths: log probabilities of sampled tokens (single, batched and ragged steps), scoring, and batched decoding over
pages that sequences share, each against the oracle or the logits that the engine hands out."""
import math
import os
import threading

import numpy as np
import pytest

import zogurax_util as zu

pytestmark = pytest.mark.gpu

LOGIT_TOL = 1e-2          # the bar of the other engine tests against the oracle
N_TOP = 6


def _model(tmp_models, arch, ftype, seed):
    from llama_cpp import synth
    path = os.path.join(tmp_models, f"{arch}_{ftype}_{seed}.gguf")
    if not os.path.exists(path):
        synth.write_synthetic_model(path, arch, ftype, seed=seed, output_std=0.1)
    return path


def _engine(path, flags=0, max_seqs=4, n_ctx=256, bt=16):
    from llama_cpp.engine import Engine
    from llama_cpp.gguf_file import GGUFFile
    return Engine(GGUFFile(path), n_ctx=n_ctx, max_seqs=max_seqs, kv_block_tokens=bt, flags=flags)


def _greedy(**kw):
    from llama_cpp.engine import SamplingSettings
    return SamplingSettings(**dict(dict(temperature=0.0, repeat_penalty=1.0), **kw))


def prompt_of(n, seed):
    return [int(t) for t in np.random.default_rng(seed).integers(3, 700, size=n)]


def check_logprobs(got, logits, token):
    """The sums have at most V / 256 + 40 terms a chain in 32 bits of exponentials off by 2^-21, the logarithms four roundings of their own size; the entropy
    divides by the same sums."""
    x = logits.astype(np.float64)
    V = len(x)
    lp = x - x.max() - math.log(np.exp(x - x.max()).sum())
    rel = (V / 256 + 40) * 2 ** -24 + 2 ** -21
    bar = lambda v: rel + 2 ** -22 * (abs(v) + math.log(V))
    assert abs(got.logprob - lp[token]) <= bar(lp[token])
    h = -(np.exp(lp) * lp).sum()
    assert abs(got.entropy - h) <= rel * (1 + 2 * math.log(V)) + 2 ** -22 * (h + math.log(V))
    order = np.argsort(-logits, kind="stable")[:len(got.top)]
    assert [t for t, _ in got.top] == order.tolist()
    assert all(abs(v - lp[t]) <= bar(lp[t]) for t, v in got.top)


@pytest.mark.parametrize("flags", [0, 1])
def test_single_sequence(native_lib, tmp_models, flags):
    """Sampled and penalised as the reference's app does: the tokens are the ones of a run that keeps nothing, the log probabilities those of the logits ahead of
    the penalties, which the same steps give when the tokens are set."""
    from llama_cpp._cabi import B2Error
    from llama_cpp.engine import SamplingSettings
    st = SamplingSettings(temperature=1.2, top_p=0.9, frequency_penalty=0.7, presence_penalty=0.8)
    u = np.random.default_rng(4).random(64)
    eng = _engine(_model(tmp_models, "tiny", "Q4_K_M", 1), flags=flags)
    prompt = prompt_of(12, 0)
    runs = []
    for on in (False, True):
        eng.set_logprobs(N_TOP if on else None)
        eng.ensure_pages(0, 64)
        eng.seq_begin(0, 0, [], st, uniforms=u)
        eng.prefill(0, prompt)
        toks = [eng.sample(0)]
        kept = [eng.logprobs(0)] if on else []
        for _ in range(10):
            toks.append(eng.decode([0])[0])
            if on:
                kept.append(eng.logprobs(0))
        runs.append(toks)
    assert runs[0] == runs[1] and all(len(k.top) == N_TOP for k in kept)
    with pytest.raises(B2Error):
        eng.decode_n(0, 2)
    eng.set_logprobs(None)
    with pytest.raises(B2Error):
        eng.logprobs(0)
    assert len(eng.decode_n(0, 2)) == 2
    eng.ensure_pages(1, 64)
    eng.seq_begin(1, 0, [], _greedy())
    eng.prefill(1, prompt)
    for i, t in enumerate(runs[0]):
        check_logprobs(kept[i], eng.logits(1), t)
        eng.set_token(1, t)
        eng.forward_pending(1)
    for n in (-2, 65):
        with pytest.raises(B2Error):
            eng.set_logprobs(n)
    eng.close()


@pytest.mark.parametrize("slots", [[0, 1, 2, 3], [6, 2, 4], [5, 0, 7, 3, 1]])
def test_batched(native_lib, tmp_models, monkeypatch, slots):
    """Results are kept by slot: those of a slot that takes no part stay."""
    monkeypatch.setenv("B2_BATCH_MIN", "3")
    path = _model(tmp_models, "tiny128", "Q8_0", 6)
    prompts = [prompt_of(n, n) for n in (5, 9, 17, 30, 12, 3, 8, 40)]
    penal, plain = _greedy(frequency_penalty=0.7, presence_penalty=0.8), _greedy()
    eng = _engine(path, max_seqs=8)
    eng.set_logprobs(N_TOP)

    def begin(settings):
        for s, p in enumerate(prompts):
            eng.ensure_pages(s, len(p) + 12)
            eng.seq_begin(s, 0, [], settings)
            eng.prefill(s, p)

    begin(penal)
    toks = {s: [eng.sample(s)] for s in range(8)}
    first = {s: eng.logprobs(s) for s in range(8)}
    kept = []
    for _ in range(6):
        for s, t in zip(slots, eng.decode(slots)):
            toks[s].append(t)
        kept.append({s: eng.logprobs(s) for s in slots})
        for s in range(8):
            if s not in slots:
                assert eng.logprobs(s) == first[s]
    eng.set_logprobs(None)
    begin(plain)
    for s in range(8):
        check_logprobs(first[s], eng.logits(s), toks[s][0])
    for i in range(6):
        for s in slots:
            eng.set_token(s, toks[s][i])
        eng.decode(slots)
        for s in slots:
            check_logprobs(kept[i][s], eng.logits(s), toks[s][i + 1])
    eng.close()


SHARED = [("tiny", "Q4_K_M", 1, 16, 140, 3), ("tiny128", "Q8_0", 6, 16, 128, 5), ("tiny128", "Q8_0", 6, 64, 200, 8), ("tiny", "Q4_K_M", 1, 16, 520, 17),
          ("tiny", "Q4_K_M", 1, 16, 980, 17), ("tiny128", "Q8_0", 6, 32, 900, 33), ("tiny", "Q4_K_M", 1, 64, 300, 66)]


@pytest.mark.parametrize("arch,ftype,seed,bt,common,n", SHARED)
def test_batched_decoding_over_shared_pages(native_lib, tmp_models, monkeypatch, arch, ftype, seed, bt, common, n):
    """Sequences that begin alike, the first one's whole pages of it in all tables: logits of every step against the oracle, which runs each sequence by itself
    (three of them), and against the same steps over pages of their own (all).

    The bar against the oracle counts two parts: |step over the engine's cache - oracle| <= |step - exact step over that cache| + |exact step over that cache -
    oracle|. Each is at most LOGIT_TOL where it stands alone: the second where a prompt's cache (f16 products) is followed by single steps in 32 bits, the first
    where a batched step (f16 products) follows such single steps. Here both meet, so 2 * LOGIT_TOL; steps over pages of their own are off by up to 0.0145."""
    from oracle.llama_ref import RefModel
    monkeypatch.setenv("B2_BATCH_MIN", "3")
    path = _model(tmp_models, arch, ftype, seed)
    head = prompt_of(common, 1)
    rest = [prompt_of(1 + (5 * i) % 23, 100 + i) for i in range(n)]
    forced = [prompt_of(4, 500 + i) for i in range(n)]
    whole = common // bt * bt
    out, launches = {}, {}
    for share in (False, True):
        eng = _engine(path, max_seqs=n, n_ctx=1024, bt=bt)
        for s in range(n):
            begin = eng.share_pages(s, 0, common) if share and s else 0
            assert begin == (whole if share and s else 0)
            prompt = head + rest[s]
            eng.ensure_pages(s, len(prompt) + 8)
            eng.seq_begin(s, begin, prompt[:begin], _greedy())
            eng.prefill(s, prompt[begin:])
        if share:
            tables = [eng.pages.table(s) for s in range(n)]
            assert all(t[:whole // bt] == tables[0][:whole // bt] for t in tables) and len({p for t in tables for p in t[whole // bt:]}) == sum(len(t) - whole // bt for t in tables)
        got = []
        for i in range(4):
            for s in range(n):
                eng.set_token(s, forced[s][i])
            before = eng.launch_count()
            eng.decode(list(range(n)))
            launches[share] = eng.launch_count() - before
            got.append(np.stack([eng.logits(s).copy() for s in range(max(0, n - 64) if n > 64 else 0, n)]))      # (of more than 64 the last step's rows)
        out[share] = got
        eng.close()
    group = {"tiny": 4, "tiny128": 2}[arch]
    more = [0 if k * group > 16 and k * whole < 16384 else 1 if k * group <= 16 else 2 for k in ([n] if n <= 64 else [64, n - 64])]      # kernels a layer
    assert launches[True] - launches[False] == 2 * sum(more)
    worst = max(np.abs(a - b).max() for a, b in zip(out[False], out[True]))
    assert worst <= LOGIT_TOL, worst
    ref = RefModel(path)
    rows = out[True][0].shape[0]
    for s in {n - 1, n - rows, n - rows // 2 - 1}:
        ref.reset()
        prompt = head + rest[s]
        want = ref.forward(prompt + forced[s])[len(prompt):]
        if n > 64 and s < 64:
            continue
        for i in range(4):
            assert np.abs(out[True][i][s - (n - rows)] - want[i]).max() <= 2 * LOGIT_TOL, (s, i)


@pytest.mark.parametrize("arch,ftype,seed,bt,groups,wanted", [
    ("tiny128", "Q8_0", 6, 16, [(40, 900), (9, 0)], (40, 896)),                 # one without anything in common, in between
    ("tiny", "Q4_K_M", 1, 64, [(20, 300), (36, 980)], (36, 960)),               # two groups: the larger one
    ("tiny128", "Q8_0", 6, 32, [(36, 980), (3, 900), (25, 40)], (36, 960)),     # the full step of 64
    ("tiny", "Q4_K_M", 1, 16, [(8, 200), (8, 300)], None),                      # not worth it
    ("tiny128", "Q8_0", 6, 16, [(30, 900), (1, 0)], None),                      # nor this, with another sequence beside
])
def test_batched_decoding_over_groups_of_shared_pages(native_lib, tmp_models, monkeypatch, arch, ftype, seed, bt, groups, wanted):
    """Sequences of several groups in mixed order, every group with pages of its own in common: logits against the same steps over own pages, tokens in the
    callers' order."""
    monkeypatch.setenv("B2_BATCH_MIN", "3")
    path = _model(tmp_models, arch, ftype, seed)
    kinds = [g for g, (n, _) in enumerate(groups) for _ in range(n)]
    np.random.default_rng(1).shuffle(kinds)
    n = len(kinds)
    heads = [prompt_of(common, 10 + g) for g, (_, common) in enumerate(groups)]
    rest = [prompt_of(1 + (7 * i) % 29, 100 + i) for i in range(n)]
    forced = [prompt_of(3, 500 + i) for i in range(n)]
    order = [int(i) for i in np.random.default_rng(2).permutation(n)]
    out, launches = {}, {}
    for share in (False, True):
        eng = _engine(path, max_seqs=n, n_ctx=1024, bt=bt)
        eng.set_logprobs(2)
        first = {}
        for s in range(n):
            g = kinds[s]
            prompt = heads[g] + rest[s]
            begin = eng.share_pages(s, first[g], groups[g][1]) if share and g in first else 0
            first.setdefault(g, s)
            eng.ensure_pages(s, len(prompt) + 8)
            eng.seq_begin(s, begin, prompt[:begin], _greedy())
            eng.prefill(s, prompt[begin:])
        got = []
        for i in range(3):
            for s in range(n):
                eng.set_token(s, forced[s][i])
            before = eng.launch_count()
            toks = eng.decode(order)
            launches[share] = eng.launch_count() - before
            rows = np.stack([eng.logits(s).copy() for s in range(n)])
            for s, t in zip(order, toks):
                assert t == int(rows[s].argmax())
                check_logprobs(eng.logprobs(s), rows[s], t)
            got.append(rows)
        out[share] = np.stack(got)
        eng.close()
    group = {"tiny": 4, "tiny128": 2}[arch]
    assert launches[True] - launches[False] == (0 if wanted is None else 2 * (1 + (1 if wanted[0] * group <= 16 else 2)))
    assert wanted is None or wanted == max(((k, common // bt * bt) for k, common in groups), key=lambda g: g[0] * g[1])
    assert np.abs(out[True] - out[False]).max() <= LOGIT_TOL


@pytest.mark.parametrize("arch,ftype,seed,bt,first,groups", [
    ("tiny", "Q4_K_M", 1, 16, 64, [(36, 960), (20, 64)]),                       # a group, and sequences that share its first pages alone
    ("tiny128", "Q8_0", 6, 16, 16, [(38, 896), (1, 16)]),                       # one such sequence, one page
    ("tiny", "Q4_K_M", 1, 64, 128, [(36, 960), (26, 704)]),                     # two groups behind a common head
])
def test_batched_decoding_over_groups_with_a_common_head(native_lib, tmp_models, monkeypatch, arch, ftype, seed, bt, first, groups):
    """Every sequence begins with the same `first` tokens in the same pages, and those of a group share more: the larger group reads all that it shares once. Logits
    against the same steps over own pages."""
    monkeypatch.setenv("B2_BATCH_MIN", "3")
    path = _model(tmp_models, arch, ftype, seed)
    kinds = [g for g, (n, _) in enumerate(groups) for _ in range(n)]
    np.random.default_rng(3).shuffle(kinds)
    n = len(kinds)
    head = prompt_of(first, 9)
    heads = [head + prompt_of(common - first, 10 + g) for g, (_, common) in enumerate(groups)]
    rest = [prompt_of(1 + (7 * i) % 29, 100 + i) for i in range(n)]
    forced = [prompt_of(2, 500 + i) for i in range(n)]
    out, launches = {}, {}
    for share in (False, True):
        eng = _engine(path, max_seqs=n, n_ctx=1024, bt=bt)
        owner = {}
        for s in range(n):
            g, prompt = kinds[s], heads[kinds[s]] + rest[s]
            begin = 0
            if share and s:
                begin = eng.share_pages(s, owner.get(g, 0), groups[g][1] if g in owner else first)
            owner.setdefault(g, s)
            eng.ensure_pages(s, len(prompt) + 8)
            eng.seq_begin(s, begin, prompt[:begin], _greedy())
            eng.prefill(s, prompt[begin:])
        if share:
            assert len({tuple(eng.pages.table(s)[:first // bt]) for s in range(n)}) == 1
            assert len({tuple(eng.pages.table(s)[:groups[0][1] // bt]) for s in range(n) if kinds[s] == 0}) == 1
        got = []
        for i in range(2):
            for s in range(n):
                eng.set_token(s, forced[s][i])
            before = eng.launch_count()
            eng.decode(list(range(n)))
            launches[share] = eng.launch_count() - before
            got.append(np.stack([eng.logits(s).copy() for s in range(n)]))
        out[share] = np.stack(got)
        eng.close()
    assert launches[True] - launches[False] == 2 * 3              # two layers: prefix, own tokens and joining beside the others' attention
    assert np.abs(out[True] - out[False]).max() <= LOGIT_TOL


def test_shared_pages_are_given_up_before_they_are_written(native_lib, tmp_models, monkeypatch):
    """A slot that goes on inside pages that another one holds gets its own there; the other's tokens stay as they were."""
    monkeypatch.setenv("B2_BATCH_MIN", "2")
    path = _model(tmp_models, "tiny", "Q4_K_M", 1)
    eng = _engine(path, max_seqs=3)
    prompt = prompt_of(150, 3)
    eng.ensure_pages(0, 200)
    eng.seq_begin(0, 0, [], _greedy())
    eng.prefill(0, prompt)
    n = eng.share_pages(1, 0, 150)
    assert n == 144
    eng.ensure_pages(1, 200)
    eng.seq_begin(1, n, prompt[:n], _greedy())
    eng.prefill(1, prompt[n:])
    assert np.abs(eng.logits(0) - eng.logits(1)).max() <= LOGIT_TOL
    before = eng.logits(0).copy()
    kept = eng.own_pages(0, 100)
    assert kept == 96
    eng.ensure_pages(0, 200)
    eng.seq_begin(0, kept, prompt[:kept], _greedy())
    eng.prefill(0, prompt_of(40, 9))                    # other tokens at the positions that slot 1 still reads
    eng.own_pages(1, 149)
    eng.ensure_pages(1, 200)
    eng.seq_begin(1, 149, prompt[:149], _greedy())
    eng.prefill(1, prompt[149:])
    assert np.abs(eng.logits(1) - before).max() <= LOGIT_TOL
    with pytest.raises(ValueError):
        eng.share_pages(1, 1, 100)
    eng.close()


@pytest.fixture(scope="module")
def layered(native_lib, tmp_path_factory):
    from llama_cpp import models
    cfg = zu.config([zu.biased(mlp=zu.moe()), zu.conved()], vocab=1031)
    path = zu.write_model(str(tmp_path_factory.mktemp("lp_layered")), cfg, zu.random_weights(cfg, seed=5))
    eng = models.open_engine(models.open_model(path), n_ctx=512, max_seqs=5, dtype="float32")
    yield eng
    eng.close()


def test_ragged_steps(layered):
    """Sampled rows beside wanted ones; a second run of the same steps (captured by then) wants the sampled rows' logits."""
    from llama_cpp.kv_pages import SequenceSlots
    eng = layered
    toks = [[int(t) for t in np.random.default_rng(i).integers(0, 1031, size=40)] for i in range(4)]
    eng.set_logprobs(N_TOP)
    runs = []
    for _ in range(3):
        seqs = SequenceSlots(eng)
        for k in range(4):
            seqs.open(k)
        steps = [{0: toks[0][:9], 2: toks[2][:1], 3: toks[3][:5]}, {2: toks[2][1:3], 1: toks[1][:2], 0: toks[0][9:10]}, {k: toks[k][20:21] for k in range(4)}, {k: toks[k][21:22] for k in range(4)}]
        run = []
        for e in steps:
            keys = list(e)
            entries = [(seqs.extend(k, len(e[k])), e[k]) for k in keys]
            logits, sampled = eng.step(entries, want=[[len(e[k]) - 1] for k in keys], sample=[True] * len(keys))
            got = [eng.logprobs(slot) for slot, _ in entries]
            for g, row, t in zip(got, logits, sampled):
                check_logprobs(g, row, t)
            run.append((sampled, [(g.logprob, g.top) for g in got]))
            _, only = eng.step([(seqs.extend(k, 1), [toks[k][30]]) for k in keys], sample=[i == 0 for i in range(len(keys))])
            run.append((only, eng.logprobs(entries[0][0]).logprob))
            assert [(eng.logprobs(slot).logprob, eng.logprobs(slot).top) for slot, _ in entries[1:]] == run[-2][1][1:]
        for k in range(4):
            seqs.close(k)
        runs.append(run)
    assert runs[0] == runs[1] == runs[2]
    eng.set_logprobs(None)


@pytest.mark.parametrize("n_top", [0, 5, 64])
def test_scores(layered, n_top):
    """Scores of a prompt's tokens, up to more rows than are worked out at once, against the logits of the same step; they leave sampled tokens' log
    probabilities and captured steps alone."""
    from llama_cpp.kv_pages import SequenceSlots
    eng = layered
    toks = [int(t) for t in np.random.default_rng(1).integers(0, 1031, size=400)]
    seqs = SequenceSlots(eng)
    eng.set_logprobs(3)
    for k in ("a", "b", "s"):
        seqs.open(k)
    _, sampled = eng.step([(seqs.extend("s", 3), toks[:3])], sample=[True])
    sampled_lp = eng.logprobs(seqs.slot("s"))
    for lo, hi in ((0, 330), (330, 332), (332, 333)):
        n = hi - lo
        want = list(range(n))
        logits, _ = eng.step([(seqs.extend("a", n), toks[lo:hi])], want=[want])
        lp, h, tl, ti = eng.score([(seqs.extend("b", n), toks[lo:hi])], [want], [toks[lo + 1:hi + 1]], n_top=n_top)
        from llama_cpp.engine import TokenLogprobs
        for i in range(n):
            check_logprobs(TokenLogprobs(float(lp[i]), float(h[i]), [(int(t), float(v)) for t, v in zip(ti[i], tl[i])]), logits[i], toks[lo + 1 + i])
    assert eng.logprobs(seqs.slot("s")) == sampled_lp
    for bad in (dict(want=[[0, 1]], tokens=[[3, 3]]), dict(want=[[0]], tokens=[[]]), dict(want=[[]], tokens=[[]]), dict(want=[[0]], tokens=[[1]], n_top=65)):
        with pytest.raises(Exception) as e:
            eng.score([(seqs.slot("b"), [5])], **bad)
        assert type(e.value).__name__ in ("ValueError", "B2Error")
    eng.set_logprobs(None)
    for k in ("a", "b", "s"):
        seqs.close(k)


@pytest.mark.parametrize("share", [False, True])
def test_callers_with_one_system_prompt(native_lib, tmp_models, share):
    """Through `Llama`: concurrent chats behind one prompt with log probabilities, against single calls. A greedy token may differ only where the two most
    likely tokens are no further apart than ten times the bar (as in the other tests), and then that sequence's comparison ends."""
    from llama_cpp import Llama
    llm = Llama(model_path=_model(tmp_models, "tiny128", "Q8_0", 6), n_gpu_layers=-1, n_ctx=512, n_seq_max=4, share_prefix=share, verbose=False)
    system = prompt_of(300, 2)
    prompts = [system + prompt_of(3 + 4 * i, 40 + i) for i in range(7)]
    ask = lambda p: llm.create_completion(p, max_tokens=12, temperature=0.0, repeat_penalty=1.0, logprobs=2)["choices"][0]["logprobs"]
    single = []
    for p in prompts:
        llm.reset()
        single.append(ask(p))
    llm.reset()
    stats = dict(llm._scheduler.stats)
    out = [None] * len(prompts)
    threads = [threading.Thread(target=lambda i=i: out.__setitem__(i, ask(prompts[i]))) for i in range(len(prompts))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    for got, want in zip(out, single):
        assert got is not None
        both = [g["tokens"] + [None] * (13 - len(g["tokens"])) for g in (got, want)]          # (None: the end, which may come early)
        for i in range(12):
            if both[0][i] != both[1][i]:
                top = sorted((want if both[1][i] is not None else got)["top_logprobs"][i].values(), reverse=True)
                assert len(top) < 2 or top[0] - top[1] < 10 * LOGIT_TOL
                break
            if both[0][i] is None:
                break
            assert abs(got["token_logprobs"][i] - want["token_logprobs"][i]) <= 2 * LOGIT_TOL
    new = llm._scheduler.stats["prefill_tokens"] - stats["prefill_tokens"]
    assert new < (2 if share else 5) * 300 + sum(map(len, prompts)) - 7 * 300
    llm.close()
