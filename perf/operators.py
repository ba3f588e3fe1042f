"""Operators over device memory, as cases that can be timed and checked: keys and values appended to a paged cache with their rotation, attention of a
batch over a prefix that all its sequences share, log probabilities of given tokens with entropy and alternatives. Together they score or continue
several answers to one prompt.

Every case is one call. `own` false: the operators in elementary torch operations, in 32 bits (angles in 64); true: the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

F32, F64 = torch.float32, torch.float64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    llama8b = dict(heads=32, kv_heads=8, dim=128, page=64)       # 8B shapes of the framework's benchmark
    tiny = dict(heads=32, kv_heads=4, dim=64, page=16)           # 1.1B shapes, small pages
    return [
        # a batched step of 32 chats: one new token each, behind a system prompt of 1000 tokens
        {"name": "append_step_32", "op": "append", **llama8b, "seqs": 32, "rows": 1, "rows_most": 1, "behind": 20, "behind_most": 500, "first": 1000, "input": "f32",
         "cache": "f16", "layout": "pairs", "fused": False},
        # prompts of several callers in one ragged call, rows cut from a joint projection, half-split rotation, odd lengths
        {"name": "append_ragged", "op": "append", **tiny, "seqs": 13, "rows": 3, "rows_most": 131, "behind": 0, "behind_most": 300, "first": 0, "input": "bf16",
         "cache": "bf16", "layout": "halves", "fused": True},
        # a long document, 16384 tokens in 8 parts
        {"name": "append_document", "op": "append", **llama8b, "seqs": 8, "rows": 2048, "rows_most": 2048, "behind": 0, "behind_most": 2048, "first": 0, "input": "f16",
         "cache": "f16", "layout": "pairs", "fused": True},
        # four callers of an app behind its 512-token system prompt, just started: the smallest call
        {"name": "shared_chat_4", "op": "shared", **llama8b, "seqs": 4, "rows": 1, "rows_most": 1, "prefix": 512, "own": 1, "own_most": 48, "cache": "f16"},
        # a serving replica: 32 chats behind one system prompt that ends inside a page
        {"name": "shared_batch_32", "op": "shared", **llama8b, "seqs": 32, "rows": 1, "rows_most": 1, "prefix": 1000, "own": 20, "own_most": 500, "cache": "f16"},
        # 64 questions to one document of an 8k window
        {"name": "shared_document_64", "op": "shared", **llama8b, "seqs": 64, "rows": 1, "rows_most": 1, "prefix": 8000, "own": 16, "own_most": 300, "cache": "bf16"},
        # 256 samples of one 8k prompt: the largest call
        {"name": "shared_samples_256", "op": "shared", **llama8b, "seqs": 256, "rows": 1, "rows_most": 1, "prefix": 8192, "own": 1, "own_most": 512, "cache": "f16"},
        # ranking: 40 candidate answers of 3 to 33 tokens, all their tokens at once
        {"name": "shared_rank_40", "op": "shared", **tiny, "seqs": 40, "rows": 3, "rows_most": 33, "prefix": 2048, "own": 3, "own_most": 33, "cache": "bf16"},
        # one token of one chat, five alternatives
        {"name": "logprobs_token", "op": "logprobs", "rows": 1, "vocab": 32000, "logits": "f32", "top": 5, "masked": False, "gap": 0},
        # a batched step with the vocabulary of the 8B model, 20 alternatives
        {"name": "logprobs_batch_32", "op": "logprobs", "rows": 32, "vocab": 128256, "logits": "f32", "top": 20, "masked": False, "gap": 0},
        # scoring a prompt: 16-bit logits of an odd vocabulary, rows with a gap between them, part of the entries masked out
        {"name": "logprobs_prompt_500", "op": "logprobs", "rows": 500, "vocab": 32003, "logits": "bf16", "top": 8, "masked": True, "gap": 5},
        # scoring a document: 1024 rows of the large vocabulary
        {"name": "logprobs_prompt_1024", "op": "logprobs", "rows": 1024, "vocab": 128256, "logits": "f32", "top": 5, "masked": False, "gap": 0},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    heads, kv_heads = rng.choice([(32, 8), (32, 4), (64, 8), (20, 5), (8, 8), (12, 2)])
    shape = dict(heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128]), page=rng.choice([16, 32, 48, 64, 128]))
    op = rng.choice(["append", "shared", "shared", "logprobs"])
    if op == "append":
        seqs = log_int(1, 64)
        most = log_int(1, max(1, 8192 // seqs))
        return {"op": op, **shape, "seqs": seqs, "rows": rng.randint(1 if seqs < 4 else 0, most), "rows_most": most, "behind": 0, "behind_most": log_int(1, 2000), "first": rng.choice([0, log_int(1, 100000)]),
                "input": rng.choice(["f32", "f16", "bf16"]), "cache": rng.choice(["f16", "bf16"]), "layout": rng.choice(["pairs", "halves"]), "fused": rng.random() < 0.5}
    if op == "shared":
        seqs = log_int(1, 200)
        rows, rows_most = (1, 1) if rng.random() < 0.6 else (rng.randint(1 if seqs < 4 else 0, 2), log_int(3, max(3, min(40, 1500 // seqs))))
        most = log_int(1, 500)
        return {"op": op, **shape, "heads": min(heads, 32), "seqs": seqs, "rows": rows, "rows_most": rows_most, "prefix": rng.choice([0, log_int(1, 300), log_int(64, 8000), log_int(64, 8000)]),
                "own": rng.randint(1, most), "own_most": most, "cache": rng.choice(["f16", "bf16"])}
    vocab = rng.choice([log_int(200, 3000), 32000, 50001, 128256])
    return {"op": op, "rows": log_int(1, max(1, min(2000, 100000000 // vocab))), "vocab": vocab, "logits": rng.choice(["f32", "f16", "bf16"]), "top": rng.choice([1, 5, 20, 64]),
            "masked": rng.random() < 0.3, "gap": rng.choice([0, 0, 1, 24])}


def spread(lo, hi, n):
    """n lengths over [lo, hi], the same for every seed: a case's work is known from the case."""
    return [lo + (i * 7919 + 13) % (hi - lo + 1) for i in range(n)]


def lengths(case):
    """new rows and own cached tokens (the new ones among them) of every sequence"""
    rows = spread(case["rows"], case["rows_most"], case["seqs"])
    if case["op"] == "append":
        return rows, [r + b for r, b in zip(rows, spread(case["behind"], case["behind_most"], case["seqs"]))]
    return rows, [max(r, o) for r, o in zip(rows, spread(case["own"], case["own_most"], case["seqs"]))]


def work(case):
    if case["op"] == "logprobs":
        size = TYPES[case["logits"]].itemsize
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * n}
    rows, held = lengths(case)
    R, H, G, D = sum(rows), case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        read, write = TYPES[case["input"]].itemsize, 2
        return {"bytes": R * (H + 2 * G) * D * (read + write), "flops": 3 * R * (H + G) * D}
    keys = sum(r * o - r * (r - 1) // 2 for r, o in zip(rows, held)) + R * case["prefix"]
    cached = case["prefix"] + sum(o for r, o in zip(rows, held) if r)
    return {"bytes": 2 * cached * G * D * 2 + 2 * R * H * D * 2, "flops": 4 * keys * H * D}


# ------------------------------------------------------------------------------------------------------------------ inputs
def inputs(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + 17)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    if case["op"] == "logprobs":
        R, V, k = case["rows"], case["vocab"], case["top"]
        x = 2.0 * normal(R, V)
        # a few likely tokens in every row, as a model's logits have them
        x.scatter_add_(1, torch.randint(0, V, (R, 6), device=dev, generator=g), 10.0 * torch.rand(R, 6, device=dev, generator=g))
        tokens = torch.randint(0, V, (R,), device=dev, generator=g, dtype=torch.int32)
        tokens[::2] = x[::2].argmax(1).to(torch.int32)
        if case["masked"]:       # entries a grammar or a padded vocabulary rules out; the asked token stays
            out = torch.rand(R, V, device=dev, generator=g) < 0.3
            out.scatter_(1, tokens[:, None].long(), False)
            x[out] = -math.inf
        logits = torch.zeros(R, V + case["gap"], device=dev, dtype=TYPES[case["logits"]])[:, :V]
        logits.copy_(x)
        return {"case": case, "logits": logits, "tokens": tokens, "logprob": torch.zeros(R, device=dev), "entropy": torch.zeros(R, device=dev),
                "top_logprob": torch.zeros(R, k, device=dev), "top_id": torch.zeros(R, k, device=dev, dtype=torch.int32)}

    rows, held = lengths(case)
    R, S, H, G, D, page = sum(rows), case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    cache = TYPES[case["cache"]]

    def ints(values):
        return torch.tensor(values, device=dev, dtype=torch.int32)

    # pages in random order: first the prefix's, then every sequence's own, and a few that nobody owns
    prefix = case.get("prefix", 0)
    n_prefix, n_own = -(-prefix // page), [-(-o // page) for o in held]
    n_pages = n_prefix + sum(n_own) + 2
    order = torch.randperm(n_pages, device=dev, generator=g).to(torch.int32)
    tables = torch.full((S, max(1, max(n_own))), -1, device=dev, dtype=torch.int32)
    at = n_prefix
    for s, n in enumerate(n_own):
        tables[s, :n] = order[at:at + n]
        at += n
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    state = {"case": case, "row_start": ints(starts), "held": ints(held), "pages": tables, "prefix_pages": order[:max(1, n_prefix)].contiguous(),
             "k_pool": normal(n_pages, G, page, D).to(cache), "v_pool": normal(n_pages, G, page, D).to(cache)}
    if case["op"] == "append":
        typ = TYPES[case["input"]]
        if case["fused"]:        # one projection's output, q | k | v
            joint = normal(R, (H + 2 * G) * D).to(typ)
            state.update(q=joint[:, :H * D].view(R, H, D), k=joint[:, H * D:(H + G) * D].view(R, G, D), v=joint[:, (H + G) * D:].view(R, G, D))
        else:
            state.update(q=normal(R, H, D).to(typ), k=normal(R, G, D).to(typ), v=normal(R, G, D).to(typ))
        base = 500000.0 if case["layout"] == "pairs" else 10000.0
        state["freqs"] = (base ** (-torch.arange(0, D, 2, device=dev, dtype=F64) / D)).to(F32)
        state["q_out"] = torch.zeros(R, H, D, device=dev, dtype=cache)
        return state
    # queries that look at some keys much more than at others: every head has a direction that a few tokens share
    lean = normal(G, 1, D)
    state["k_pool"] += (2.0 * lean * (torch.rand(n_pages, G, page, 1, device=dev, generator=g) < 0.02)).to(cache)
    state["q"] = (normal(R, G, H // G, D) + 0.7 * lean).to(cache).view(R, H, D)
    state["out"] = torch.zeros(R, H, D, device=dev, dtype=cache)
    return state


def prepare(case, seed):
    state = inputs(case, seed)
    if own:
        path = os.path.join(os.getcwd(), "llama-fastapi-k8s-gpu_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        from llama_cpp import device_ops
        state["ops"] = device_ops
        if case["op"] == "shared":
            n = device_ops.attention_shared_prefix_workspace(rows=sum(lengths(case)[0]), n_head=case["heads"], n_kv=case["kv_heads"], head_dim=case["dim"])
            state["workspace"] = torch.empty(n, device=state["q"].device, dtype=torch.uint8)
    return state


# -------------------------------------------------------------------------------------------------------------- plain forms
def places(state):
    """page and offset of every new row, and its position in its sequence"""
    rows, held = lengths(state["case"])
    start, dev, page = state["row_start"].long(), state["k_pool"].device, state["case"]["page"]
    row = torch.arange(sum(rows), device=dev)
    seq = (row[:, None] >= start[None, 1:]).sum(1)
    at = state["held"].long()[seq] - start[seq + 1] + row
    return state["pages"][seq, at // page].long(), at % page, at


def rotate(x, cos, sin, layout):
    if layout == "pairs":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def plain_append(state):
    case = state["case"]
    page, off, at = places(state)
    angle = (case["first"] + at).to(F64)[:, None] * state["freqs"].to(F64)
    cos, sin = angle.cos().to(F32)[:, None], angle.sin().to(F32)[:, None]
    cache = state["k_pool"].dtype
    state["k_pool"][page, :, off] = rotate(state["k"].to(F32), cos, sin, case["layout"]).to(cache)
    state["v_pool"][page, :, off] = state["v"].to(F32).to(cache)
    state["q_out"].copy_(rotate(state["q"].to(F32), cos, sin, case["layout"]))
    return state["k_pool"], state["v_pool"], state["q_out"]


def plain_shared(state):
    case = state["case"]
    rows, held = lengths(case)
    H, G, D, page, P = case["heads"], case["kv_heads"], case["dim"], case["page"], case["prefix"]

    def cached(pool, pages, n):          # [kv heads, tokens, dim]
        return pool[pages.long()].to(F32).transpose(0, 1).reshape(G, -1, D)[:, :n]

    q = state["q"].to(F32).view(-1, G, H // G, D).permute(1, 0, 2, 3)          # [kv heads, rows, heads of the group, dim]
    kp, vp = (cached(state[p], state["prefix_pages"], P) for p in ("k_pool", "v_pool"))
    shared = torch.einsum("grhd,gjd->grhj", q, kp) / math.sqrt(D)
    r0 = 0
    for s, (r, o) in enumerate(zip(rows, held)):
        if r == 0:
            continue
        pages = state["pages"][s, :-(-o // page)]
        k, v = cached(state["k_pool"], pages, o), cached(state["v_pool"], pages, o)
        score = torch.einsum("grhd,gjd->grhj", q[:, r0:r0 + r], k) / math.sqrt(D)
        ahead = torch.arange(o, device=k.device)[None, :] > torch.arange(o - r, o, device=k.device)[:, None]
        score = torch.cat([shared[:, r0:r0 + r], score.masked_fill(ahead[None, :, None], -math.inf)], -1)
        weight = torch.exp(score - score.amax(-1, keepdim=True))
        weight = weight / weight.sum(-1, keepdim=True)
        out = torch.einsum("grhj,gjd->grhd", weight[..., :P], vp) + torch.einsum("grhj,gjd->grhd", weight[..., P:], v)
        state["out"][r0:r0 + r] = out.permute(1, 0, 2, 3).reshape(r, H, D)
        r0 += r
    return state["out"]


def best(x, k):
    """[rows, k]: the k largest entries' ids, largest first, of equal ones the lowest id first; -1 past the end"""
    V = x.shape[1]
    left, ids = torch.ones_like(x, dtype=torch.bool), []
    number = torch.arange(V, device=x.device, dtype=torch.int32)
    for _ in range(min(k, V)):
        top = torch.where(left, x, -math.inf).amax(1, keepdim=True)
        ids.append(torch.where(left & (x == top), number, V).amin(1, keepdim=True))
        left.scatter_(1, ids[-1].long(), False)
    ids += [torch.full((x.shape[0], 1), -1, device=x.device, dtype=torch.int32)] * (k - len(ids))
    return torch.cat(ids, 1) if ids else torch.zeros(x.shape[0], 0, device=x.device, dtype=torch.int32)


def plain_logprobs(state):
    x = state["logits"].to(F32)
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    state["logprob"].copy_(((x.gather(1, state["tokens"][:, None].long()) - top) - log_total)[:, 0])
    spent = torch.where(e > 0, e * (x - top), 0.0).sum(1, keepdim=True)
    state["entropy"].copy_((log_total - spent / total)[:, 0])
    k = state["case"]["top"]
    ids = best(x, k)
    state["top_id"].copy_(ids)
    state["top_logprob"].copy_(torch.where(ids >= 0, (x.gather(1, ids.clamp(min=0).long()) - top) - log_total, -math.inf))
    return state["logprob"], state["entropy"], state["top_logprob"], state["top_id"]


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": plain_append, "shared": plain_shared, "logprobs": plain_logprobs}[op](state)
    ops, stream = state["ops"], torch.cuda.current_stream()
    if op == "append":
        ops.kv_append(state["k"], state["v"], state["k_pool"], state["v_pool"], state["pages"], state["row_start"], state["held"], q=state["q"],
                      q_out=state["q_out"], freqs=state["freqs"], layout=state["case"]["layout"], first_pos=state["case"]["first"], stream=stream)
        return state["k_pool"], state["v_pool"], state["q_out"]
    if op == "shared":
        ops.attention_shared_prefix(state["q"], state["k_pool"], state["v_pool"], state["prefix_pages"], state["case"]["prefix"], state["pages"],
                                    state["row_start"], state["held"], state["out"], state["workspace"], max_rows=state["case"]["rows_most"], stream=stream)
        return state["out"]
    ops.token_logprobs(state["logits"], state["tokens"], state["logprob"], state["entropy"], state["top_logprob"], state["top_id"], stream=stream)
    return state["logprob"], state["entropy"], state["top_logprob"], state["top_id"]


# -------------------------------------------------------------------------------------------------------- 64-bit definitions
def exact(case, seed):
    s = inputs(case, seed)
    if case["op"] == "logprobs":
        x = s["logits"].to(F64)
        R, V = x.shape
        lse = torch.logsumexp(x, 1)
        logp = x - lse[:, None]
        entropy = -torch.where(logp > -math.inf, logp.exp() * logp, 0.0).sum(1)
        k = min(case["top"], V)
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        top = torch.full((R, case["top"]), -math.inf, device=x.device, dtype=F64)
        top[:, :k] = logp.gather(1, ids)
        top_id = torch.full((R, case["top"]), -1, device=x.device, dtype=torch.int32)
        top_id[:, :k] = ids.to(torch.int32)
        return logp[torch.arange(R, device=x.device), s["tokens"].long()], entropy, top, top_id

    rows, held = lengths(case)
    G, D, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // G
    start = [sum(rows[:i]) for i in range(len(rows))]
    if case["op"] == "append":
        k_pool, v_pool, q_out = s["k_pool"].to(F64), s["v_pool"].to(F64), s["q"].to(F64).clone()
        for i, (r, o) in enumerate(zip(rows, held)):
            if r == 0:
                continue
            at = torch.arange(o - r, o, device=q_out.device)
            turn = torch.polar(torch.ones(1, 1, device=q_out.device, dtype=F64), (at + case["first"]).to(F64)[:, None] * s["freqs"].to(F64)[None])
            there = (s["pages"][i].long()[at // page], at % page)
            for what in ("k", "q"):
                x = s[what][start[i]:start[i] + r].to(F64)
                if case["layout"] == "pairs":
                    z = torch.view_as_complex(x.reshape(*x.shape[:-1], D // 2, 2).contiguous()) * turn[:, None]
                    y = torch.view_as_real(z).reshape(x.shape)
                else:
                    z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn[:, None]
                    y = torch.cat([z.real, z.imag], -1)
                if what == "k":
                    k_pool[there[0], :, there[1]] = y
                else:
                    q_out[start[i]:start[i] + r] = y
            v_pool[there[0], :, there[1]] = s["v"][start[i]:start[i] + r].to(F64)
        return k_pool, v_pool, q_out

    out = torch.zeros(sum(rows), case["heads"], D, device=s["q"].device, dtype=F64)
    P = case["prefix"]
    for g in range(G):
        flat = [s[p][:, g].to(F64) for p in ("k_pool", "v_pool")]          # [pages, page, dim]
        kp, vp = (f[s["prefix_pages"].long()].reshape(-1, D)[:P] for f in flat)
        q = s["q"][:, g * group:(g + 1) * group].to(F64)
        with_prefix = q @ kp.T
        for i, (r, o) in enumerate(zip(rows, held)):
            if r == 0:
                continue
            k, v = (f[s["pages"][i, :-(-o // page)].long()].reshape(-1, D)[:o] for f in flat)
            now = slice(start[i], start[i] + r)
            scores = torch.cat([with_prefix[now], q[now] @ k.T], -1) * D ** -0.5       # [r, group, P + o]
            seen = torch.arange(P + o, device=q.device)[None] <= (P + o - r + torch.arange(r, device=q.device))[:, None]
            weights = torch.softmax(scores.masked_fill(~seen[:, None], -math.inf), -1)
            out[now, g * group:(g + 1) * group] = weights[..., :P] @ vp + weights[..., P:] @ v
    return out
