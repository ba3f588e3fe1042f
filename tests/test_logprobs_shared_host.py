"""Log probabilities and shared prompt pages through `Llama` and the scheduler, without a GPU: a fake engine whose cache is a list of tokens by page, so that a
page that is written while another sequence reads it, or read where it was not written, shows."""
import threading

import numpy as np
import pytest

from fake_engine import FakeEngine


class PagedFake(FakeEngine):
    """Tokens are kept in pages; every step reads them back from there."""
    wrong = None

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.store = np.full((self.pages.num_blocks, self.block_tokens), -1)
        self.n_top, self.kept, self.shared = None, {}, 0

    def _read(self, slot, n):
        t = self.pages.table(slot)
        return [int(self.store[t[i // self.block_tokens], i % self.block_tokens]) for i in range(n)]

    def _write(self, slot, pos, token):
        page = self.pages.table(slot)[pos // self.block_tokens]
        if any(page in self.pages.table(s) for s in range(self.max_seqs) if s != slot):
            PagedFake.wrong = f"slot {slot} wrote to page {page}, which another slot holds"
        self.store[page, pos % self.block_tokens] = token

    def seq_begin(self, slot, n_past, history, sampling, uniforms=None):
        if self._read(slot, n_past) != list(history):
            PagedFake.wrong = "the cache does not hold the tokens that are to be reused"
        self.seqs[slot] = {"toks": list(history), "pending": None, "n_prompt": 0}

    def prefill(self, slot, tokens):
        n = len(self.seqs[slot]["toks"])
        super().prefill(slot, tokens)
        for i, t in enumerate(tokens):
            self._write(slot, n + i, t)

    def sample(self, slot):
        t = super().sample(slot)
        self._keep(slot, t)
        return t

    def decode(self, slots):
        for s in slots:
            self._write(s, len(self.seqs[s]["toks"]), self.seqs[s]["pending"])
            if self._read(s, len(self.seqs[s]["toks"])) != self.seqs[s]["toks"]:
                PagedFake.wrong = "a sequence's cached tokens changed"
        out = super().decode(slots)
        for s, t in zip(slots, out):
            self._keep(s, t)
        return out

    def decode_n(self, slot, n):
        assert self.n_top is None
        return super().decode_n(slot, n)

    def share_pages(self, slot, other, n_tokens):
        self.pages.release(slot)
        self.shared += 1
        return self.pages.share(slot, other, n_tokens)

    def own_pages(self, slot, n_tokens):
        return self.pages.own_from(slot, n_tokens)

    def set_logprobs(self, n_top):
        self.n_top, self.kept = n_top, {}

    def _keep(self, slot, token):
        from llama_cpp.engine import TokenLogprobs
        if self.n_top is not None:
            self.kept[slot] = TokenLogprobs(-token / 1000, 1.0, [(token + i, -(token + i) / 1000) for i in range(self.n_top)])

    def logprobs(self, slot):
        return self.kept[slot]


@pytest.fixture(scope="module")
def tiny_path(tmp_path_factory):
    from llama_cpp import synth
    p = str(tmp_path_factory.mktemp("lp") / "tiny.gguf")
    synth.write_synthetic_model(p, "tiny", "Q4_K_M", seed=1)
    return p


def make(tiny_path, monkeypatch, **kw):
    from llama_cpp import Llama
    from llama_cpp import llama as L
    monkeypatch.setattr(L, "Engine", PagedFake)
    PagedFake.delay, PagedFake.eos_after, PagedFake.fail_with, PagedFake.wrong = 0.0, None, None, None
    return Llama(model_path=tiny_path, n_gpu_layers=-1, n_ctx=256, verbose=False, **kw)


def test_logprobs_of_a_completion(tiny_path, monkeypatch):
    llm = make(tiny_path, monkeypatch)
    plain = llm.create_completion([9, 10, 11], max_tokens=12, temperature=0.0)
    assert plain["choices"][0]["logprobs"] is None and llm._engine.n_top is None
    out = llm.create_completion([9, 10, 11], max_tokens=12, temperature=0.0, logprobs=3)
    lp = out["choices"][0]["logprobs"]
    assert out["choices"][0]["text"] == plain["choices"][0]["text"] == "".join(lp["tokens"])
    assert all(len(v) == 12 for v in lp.values()) and set(lp) == {"tokens", "text_offset", "token_logprobs", "top_logprobs"}
    at = 0
    for tok, off, p, top in zip(lp["tokens"], lp["text_offset"], lp["token_logprobs"], lp["top_logprobs"]):
        assert off == at and top[tok] == p and 1 <= len(top) <= 3
        at += len(tok)
    assert llm.create_completion([9, 10, 11], max_tokens=4, temperature=0.0, logprobs=0)["choices"][0]["logprobs"]["top_logprobs"][0].keys() == {lp["tokens"][0]}
    calls = llm._engine.calls["decode_n"]
    llm.create_completion([9, 10, 11], max_tokens=4, temperature=0.0)           # (and off again: single sequences run ahead)
    assert llm._engine.n_top is None and llm._engine.calls["decode_n"] > calls
    chat = llm.create_chat_completion([{"role": "user", "content": "hello"}], max_tokens=5, temperature=0.0, logprobs=True, top_logprobs=2)
    assert len(chat["choices"][0]["logprobs"]["tokens"]) == 5
    assert llm.create_chat_completion([{"role": "user", "content": "hello"}], max_tokens=5, temperature=0.0)["choices"][0]["logprobs"] is None
    assert PagedFake.wrong is None
    llm.close()


def test_logprobs_with_echo_stop_and_end_of_text(tiny_path, monkeypatch):
    llm = make(tiny_path, monkeypatch)
    full = llm.create_completion("hello", max_tokens=20, temperature=0.0, echo=True, logprobs=1)["choices"][0]
    assert full["text"] == "hello" + "".join(full["logprobs"]["tokens"]) and full["logprobs"]["text_offset"][0] == 5
    text = full["text"][5:]
    cut = llm.create_completion("hello", max_tokens=20, temperature=0.0, stop=[text[6:9]], logprobs=1)["choices"][0]
    n = len(cut["logprobs"]["tokens"])
    assert cut["text"] == text[:text.index(text[6:9])] and len("".join(cut["logprobs"]["tokens"][:-1])) < max(1, len(cut["text"])) <= len("".join(cut["logprobs"]["tokens"]))
    assert all(len(v) == n for v in cut["logprobs"].values())
    none = llm.create_completion("hello", max_tokens=20, temperature=0.0, stop=[text[:2]], logprobs=1)["choices"][0]
    assert none["text"] == "" and none["logprobs"]["tokens"] == []
    PagedFake.eos_token, PagedFake.eos_after = llm._vocab.eot_id, 3
    ended = llm.create_completion("hello", max_tokens=20, temperature=0.0, logprobs=1)["choices"][0]
    assert ended["finish_reason"] == "stop" and len(ended["logprobs"]["tokens"]) == 3
    PagedFake.eos_after = None
    llm.close()


def test_logprobs_refusals(tiny_path, monkeypatch):
    llm = make(tiny_path, monkeypatch)
    for n in (-1, 65):
        with pytest.raises(ValueError):
            llm.create_completion([1, 2], max_tokens=2, logprobs=n)
    with pytest.raises(NotImplementedError):
        llm.create_completion([1, 2], max_tokens=2, logprobs=1, stream=True)
    llm.close()


def test_chats_that_ask_for_what_is_not_given(tiny_path, monkeypatch):
    """A chat's stream has no log probabilities and says so; numbers of alternatives outside 0..64 are the nearest one inside. Both ran before there were any."""
    llm = make(tiny_path, monkeypatch)
    ask = lambda **kw: llm.create_chat_completion([{"role": "user", "content": "hello"}], max_tokens=5, temperature=0.0, **kw)
    plain = list(ask(stream=True))
    with pytest.warns(UserWarning, match="log probabilities"):
        chunks = ask(stream=True, logprobs=True, top_logprobs=2)
    strip = lambda cs: [c["choices"][0] for c in cs]
    assert strip(chunks) == strip(plain) and llm._engine.n_top is None
    for asked, kept in ((65, 64), (10 ** 6, 64), (-1, 0)):
        lp = ask(logprobs=True, top_logprobs=asked)["choices"][0]["logprobs"]
        assert len(lp["tokens"]) == 5 and llm._engine.n_top == kept
    assert ask(logprobs=False, top_logprobs=65)["choices"][0]["logprobs"] is None
    monkeypatch.setattr(PagedFake, "set_logprobs", property(lambda self: (_ for _ in ()).throw(AttributeError())))      # an engine that has none
    with pytest.warns(UserWarning, match="log probabilities"):
        assert ask(logprobs=True)["choices"][0]["logprobs"] is None
    llm.close()


@pytest.mark.parametrize("share", [False, True])
def test_many_callers_with_one_prompt_in_front(tiny_path, monkeypatch, share):
    """Texts are the ones of single calls, whoever shares pages with whom; the shared prompt is evaluated once per run of callers that overlap."""
    llm = make(tiny_path, monkeypatch, n_seq_max=4, share_prefix=share)
    rng = np.random.default_rng(3)
    system = [int(t) for t in rng.integers(300, 500, size=150)]
    prompts = [(system[:n] + [int(t) for t in rng.integers(300, 500, size=m)]) for n, m in
               [(150, 5), (150, 9), (150, 1), (140, 30), (64, 60), (63, 60), (128, 3), (150, 5), (129, 1), (0, 20), (150, 70), (128, 1)]]
    want = []
    for p in prompts:
        llm.reset()
        want.append(llm.create_completion(p, max_tokens=16, temperature=0.0)["choices"][0]["text"])
    llm.reset()
    llm._engine.shared = 0
    PagedFake.delay = 0.002
    for _ in range(3):
        got, lps = [None] * len(prompts), [None] * len(prompts)

        def work(i):
            c = llm.create_completion(prompts[i], max_tokens=16, temperature=0.0, logprobs=i % 3 if i % 2 else None)["choices"][0]
            got[i], lps[i] = c["text"], c["logprobs"]
        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(prompts))]
        for t in threads:
            t.start()
        for t in threads:
            t.join(60)
        assert PagedFake.wrong is None and got == want
        for i, lp in enumerate(lps):
            assert (lp is None) if i % 2 == 0 else ("".join(lp["tokens"]) == want[i] and len(lp["token_logprobs"]) == 16)
    assert (llm._engine.shared > 0) == share
    assert len({p for s in range(4) for p in llm._engine.pages.table(s)}) + llm._engine.pages.free_pages == llm._engine.pages.num_blocks
    PagedFake.delay = 0.0
    # direct evaluation takes slot 0 over, whatever it shares
    llm.eval(system[:100])
    assert PagedFake.wrong is None
    llm.close()


def test_a_request_that_fails_gives_shared_pages_back(tiny_path, monkeypatch):
    llm = make(tiny_path, monkeypatch, n_seq_max=2, share_prefix=True)
    PagedFake.delay = 0.005
    prompt = list(range(300, 450))
    results = []
    t = threading.Thread(target=lambda: results.append(llm.create_completion(prompt, max_tokens=60, temperature=0.0)))
    t.start()
    while not llm._engine.calls["decode"]:
        pass
    PagedFake.fail_with = RuntimeError("no")
    with pytest.raises(RuntimeError, match="no"):
        llm.create_completion(prompt + [7], max_tokens=3)
    PagedFake.fail_with = None
    out = llm.create_completion(prompt + [8], max_tokens=3, temperature=0.0)
    t.join(60)
    PagedFake.delay = 0.0
    assert results and out["usage"]["completion_tokens"] == 3 and PagedFake.wrong is None
    llm.close()


def test_common_prefix():
    from llama_cpp.scheduler import common_prefix
    rng = np.random.default_rng(0)
    for n in (0, 1, 63, 64, 65, 128, 200):
        a = [int(t) for t in rng.integers(0, 9, size=n)]
        assert common_prefix(a, list(a)) == common_prefix(a, a + [1]) == common_prefix(a + [2], a) == n
        for i in range(0, n, 7):
            b = list(a)
            b[i] += 10
            assert common_prefix(a, b) == common_prefix(b, a) == i


def test_score_refuses_lists_that_do_not_go_together():
    """one list of wanted rows and one of tokens an entry: the native step reads a length for every entry"""
    from llama_cpp.engine import LayeredEngine
    eng, calls = LayeredEngine.__new__(LayeredEngine), []

    class Lib:
        @staticmethod
        def b2_step_scores(handle, n_entries, slots, lens, *rest):
            calls.append((n_entries, len(slots), len(lens)))
            return 0
    eng.lib, eng._h = Lib, None
    entries = [(0, [1, 2, 3]), (1, [4, 5])]
    for want, tokens in (([[0]], [[7]]), ([[0], [1]], [[7]]), ([[0]], [[7], [8]]), ([[0], [1], []], [[7], [8], []]), ([], []), ([[0], [2]], [[7], [8]]), ([[0], [1]], [[7], [8, 9]])):
        with pytest.raises(ValueError):
            eng.score(entries, want, tokens)
    assert not calls
    eng.score(entries, [[0], []], [[7], []])
    assert calls == [(2, 2, 2)]
