"""Operators over a paged cache that is held in 4 bits, as cases that can be timed and checked: keys and values quantised as they are appended (and the new
rows read back), ranges of the cache read back, attention over it. Together they serve chats and prompts from a cache of a quarter of the size.

Every entry of a head is a 4-bit code of its group of 32 neighbours: scale = m / -8 in f16, m the group's entry of greatest magnitude (of m and -m the negative one);
code = round(entry / scale) + 8, held to 0 .. 15; the value that it stands for is scale * (code - 8).

Every case is one pass. `own` false: the operators in elementary torch operations, in 32 bits (angles in 64); true: the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

F32, F64 = torch.float32, torch.float64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 32


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    llama8b = dict(heads=32, kv_heads=8, dim=128, page=64)       # 8B shapes of the framework's benchmark
    tiny = dict(heads=32, kv_heads=4, dim=64, page=16)           # 1.1B shapes, small pages
    return [
        # a batched step of 32 chats: one new token each
        {"name": "append_step_32", "op": "append", **llama8b, "seqs": 32, "rows": 1, "rows_most": 1, "behind": 20, "behind_most": 1500, "first": 0, "input": "f32", "output": "f16",
         "layout": "pairs", "fused": False},
        # prompts of several callers in one ragged call, rows cut from a joint projection, half-split rotation, odd lengths
        {"name": "append_ragged", "op": "append", **tiny, "seqs": 13, "rows": 3, "rows_most": 131, "behind": 0, "behind_most": 300, "first": 1000, "input": "bf16", "output": "bf16",
         "layout": "halves", "fused": True},
        # a long document, 16384 tokens in 8 parts
        {"name": "append_document", "op": "append", **llama8b, "seqs": 8, "rows": 2048, "rows_most": 2048, "behind": 0, "behind_most": 2048, "first": 0, "input": "f16", "output": "f16",
         "layout": "pairs", "fused": True},
        # one chat's last 100 tokens, as a host that goes on with them in 16 bits takes them out: the smallest read
        {"name": "read_chat", "op": "read", **llama8b, "seqs": 1, "rows": 100, "rows_most": 100, "behind": 600, "behind_most": 600, "output": "f16"},
        # whole chats of odd lengths moved to another replica, pages of 48
        {"name": "read_ragged", "op": "read", "heads": 20, "kv_heads": 5, "dim": 128, "page": 48, "seqs": 24, "rows": 101, "rows_most": 2999, "behind": 0, "behind_most": 0,
         "output": "bf16"},
        # documents that are taken out whole, 65536 tokens
        {"name": "read_document", "op": "read", **llama8b, "seqs": 8, "rows": 8192, "rows_most": 8192, "behind": 0, "behind_most": 0, "output": "f16"},
        # the next token of one chat: the smallest call
        {"name": "attend_chat", "op": "attend", **llama8b, "seqs": 1, "rows": 1, "rows_most": 1, "behind": 699, "behind_most": 699, "output": "f16"},
        # the next token behind one long document, a 32k window
        {"name": "attend_long", "op": "attend", **llama8b, "seqs": 1, "rows": 1, "rows_most": 1, "behind": 32000, "behind_most": 32000, "output": "bf16"},
        # a batched step of 32 chats
        {"name": "attend_batch_32", "op": "attend", **llama8b, "seqs": 32, "rows": 1, "rows_most": 1, "behind": 20, "behind_most": 1500, "output": "f16"},
        # a full replica: 256 chats of up to 4096 tokens
        {"name": "attend_batch_256", "op": "attend", **llama8b, "seqs": 256, "rows": 1, "rows_most": 1, "behind": 16, "behind_most": 4095, "output": "f16"},
        # a few drafted tokens of 20 chats checked at once, small pages
        {"name": "attend_drafts_20", "op": "attend", **tiny, "seqs": 20, "rows": 2, "rows_most": 7, "behind": 100, "behind_most": 2000, "output": "bf16"},
        # a part of a prompt: 2048 new tokens behind 6000
        {"name": "attend_prompt", "op": "attend", **llama8b, "seqs": 1, "rows": 2048, "rows_most": 2048, "behind": 6000, "behind_most": 6000, "output": "f16"},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    heads, kv_heads = rng.choice([(32, 8), (32, 4), (64, 8), (20, 5), (8, 8), (12, 2)])
    shape = dict(heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128]), page=rng.choice([16, 32, 48, 64, 128]))
    op = rng.choice(["append", "read", "attend", "attend", "attend"])
    output = rng.choice(["f16", "bf16"])
    if op == "append":
        seqs = log_int(1, 64)
        most = log_int(1, max(1, 8192 // seqs))
        return {"op": op, **shape, "seqs": seqs, "rows": rng.randint(1 if seqs < 4 else 0, most), "rows_most": most, "behind": 0, "behind_most": log_int(1, 2000),
                "first": rng.choice([0, log_int(1, 100000)]), "input": rng.choice(["f32", "f16", "bf16"]), "output": output, "layout": rng.choice(["pairs", "halves"]),
                "fused": rng.random() < 0.5}
    if op == "read":
        seqs = log_int(1, 64)
        most = log_int(1, 30000 // seqs)
        return {"op": op, **shape, "seqs": seqs, "rows": rng.randint(1 if seqs < 4 else 0, most), "rows_most": most, "behind": 0, "behind_most": rng.choice([0, log_int(1, 1000)]),
                "output": rng.choice(["f32", "f16", "bf16"])}
    kind = rng.choice(["step", "step", "long", "drafts", "prompt"])
    if kind == "step":
        seqs = log_int(1, 256)
        return {"op": op, **shape, "seqs": seqs, "rows": 1, "rows_most": 1, "behind": 0, "behind_most": log_int(1, 4095 if seqs < 100 else 2000), "output": output}
    if kind == "long":
        most = log_int(4000, 32000)
        return {"op": op, **shape, "seqs": rng.randint(1, 4), "rows": 1, "rows_most": 1, "behind": rng.randint(0, most), "behind_most": most, "output": output}
    if kind == "drafts":
        seqs = log_int(1, 64)
        return {"op": op, **shape, "seqs": seqs, "rows": rng.randint(0 if seqs > 3 else 1, 2), "rows_most": log_int(2, 16), "behind": 0, "behind_most": log_int(1, 2000), "output": output}
    seqs = log_int(1, 6)
    most = log_int(17, 1400 // seqs)
    return {"op": op, **shape, "heads": min(heads, 32), "seqs": seqs, "rows": rng.randint(1, most), "rows_most": most, "behind": 0, "behind_most": log_int(1, 5000), "output": output}


def spread(lo, hi, n):
    """n lengths over [lo, hi], the same for every seed: a case's work is known from the case."""
    return [lo + (i * 7919 + 13) % (hi - lo + 1) for i in range(n)]


def lengths(case):
    """rows of the call and cached tokens (the rows among them) of every sequence"""
    rows = spread(case["rows"], case["rows_most"], case["seqs"])
    return rows, [r + b for r, b in zip(rows, spread(case["behind"], case["behind_most"], case["seqs"]))]


def work(case):
    rows, held = lengths(case)
    R, H, G, D = sum(rows), case["heads"], case["kv_heads"], case["dim"]
    token = 2 * G * (D // 2 + D // GROUP * 2)                    # bytes of a cached token
    out = TYPES[case["output"]].itemsize
    if case["op"] == "append":       # rows and queries read, queries and the cache written, the new rows read back
        return {"bytes": R * ((H + 2 * G) * D * TYPES[case["input"]].itemsize + H * D * out + 2 * token + 2 * G * D * out), "flops": 3 * R * (H + G) * D + 8 * R * G * D}
    if case["op"] == "read":
        return {"bytes": R * (token + 2 * G * D * out), "flops": 4 * R * G * D}
    keys = sum(r * o - r * (r - 1) // 2 for r, o in zip(rows, held))
    return {"bytes": sum(o for r, o in zip(rows, held) if r) * token + 2 * R * H * D * out, "flops": 4 * keys * H * D}


# ------------------------------------------------------------------------------------------------------------------ inputs
def inputs(case, seed):
    """tables in random order, the tokens that the cache holds before the call (token by token of every sequence), the call's own rows"""
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + 29)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def ints(values):
        return torch.tensor(values, device=dev, dtype=torch.int32)

    def starts(counts):
        at = [0]
        for c in counts:
            at.append(at[-1] + c)
        return ints(at)

    rows, held = lengths(case)
    S, R, H, G, D, page = case["seqs"], sum(rows), case["heads"], case["kv_heads"], case["dim"], case["page"]
    n_own = [-(-o // page) for o in held]
    n_pages = sum(n_own) + 2                                     # two that nobody owns
    order = torch.randperm(n_pages, device=dev, generator=g).to(torch.int32)
    tables = torch.full((S, max(1, max(n_own))), -1, device=dev, dtype=torch.int32)
    at = 0
    for s, n in enumerate(n_own):
        tables[s, :n] = order[at:at + n]
        at += n
    before = [o - r for r, o in zip(rows, held)] if case["op"] == "append" else held      # tokens that the cache holds before the call
    T = sum(before)
    # keys have a few entries of a head that are far larger than the others, values have none
    large = 1.0 + 7.0 * (torch.rand(G, D, device=dev, generator=g) < 0.03)
    state = {"case": case, "row_start": starts(rows), "held": ints(held), "pages": tables, "n_pages": n_pages, "before_start": starts(before), "before": ints(before)}
    cached = TYPES[case["output"]] if case["output"] != "f32" else torch.float16
    state["k_before"], state["v_before"] = (normal(T, G, D) * large).to(cached), normal(T, G, D).to(cached)
    out = TYPES[case["output"]]
    if case["op"] == "append":
        typ = TYPES[case["input"]]
        joint = normal(R, (H + 2 * G) * D)
        joint[:, H * D:(H + G) * D] *= large.view(-1)
        joint = joint.to(typ)
        parts = joint[:, :H * D].view(R, H, D), joint[:, H * D:(H + G) * D].view(R, G, D), joint[:, (H + G) * D:].view(R, G, D)
        state["q"], state["k"], state["v"] = parts if case["fused"] else (p.contiguous() for p in parts)
        base = 500000.0 if case["layout"] == "pairs" else 10000.0
        state["freqs"] = (base ** (-torch.arange(0, D, 2, device=dev, dtype=F64) / D)).to(F32)
        state["q_out"] = torch.zeros(R, H, D, device=dev, dtype=out)
    if case["op"] == "attend":
        # queries that look at some keys much more than at others: a few tokens' keys are their direction
        lean = normal(G, 1, D)
        state["k_before"] += 1.5 * lean.view(1, G, D).to(cached) * (torch.rand(T, G, 1, device=dev, generator=g) < 0.02)
        state["q"] = (0.6 * normal(R, G, H // G, D) + 0.6 * lean).to(out).view(R, H, D)
        state["out"] = torch.zeros(R, H, D, device=dev, dtype=out)
    else:
        state["k_back"], state["v_back"] = (torch.zeros(R, G, D, device=dev, dtype=out) for _ in range(2))
    return state


def prepare(case, seed):
    """The cache is what a program has filled by appending, in the form of the side that is asked."""
    state = inputs(case, seed)
    k, v = state.pop("k_before"), state.pop("v_before")
    G, D, page = case["kv_heads"], case["dim"], case["page"]
    dev = k.device
    if own:
        path = os.path.join(os.getcwd(), "llama-fastapi-k8s-gpu_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        from llama_cpp import device_ops
        state["ops"] = device_ops
        state["k_pool"], state["v_pool"] = (torch.zeros(state["n_pages"], G, page // 16, 9 * D, device=dev, dtype=torch.uint8) for _ in range(2))
        device_ops.kv_append_4bit(k, v, state["k_pool"], state["v_pool"], state["pages"], state["before_start"], state["before"], stream=torch.cuda.current_stream())
        if case["op"] == "attend":
            n = device_ops.attention_4bit_workspace(rows=sum(lengths(case)[0]), n_head=case["heads"], n_kv=G, head_dim=D)
            state["workspace"] = torch.empty(n, device=dev, dtype=torch.uint8)
    else:
        state["k_pool"], state["v_pool"] = ({"codes": torch.zeros(state["n_pages"], G, page, D, device=dev, dtype=torch.uint8),
                                             "scales": torch.zeros(state["n_pages"], G, page, D // GROUP, device=dev, dtype=torch.float16)} for _ in range(2))
        at = places(state["before_start"], state["before"], state["pages"], page, len(k))
        store(state["k_pool"], at, k.to(F32))
        store(state["v_pool"], at, v.to(F32))
    return state


# -------------------------------------------------------------------------------------------------------------- plain forms
def places(start, held, pages, page, n):
    """page, offset and position of rows 0 .. n - 1: each sequence's are the newest of its tokens"""
    start, row = start.long(), torch.arange(n, device=start.device)
    seq = torch.searchsorted(start[1:].contiguous(), row, right=True)
    at = held.long()[seq] - start[seq + 1] + row
    return pages[seq, at // page].long(), at % page, at


def quantise(x):
    """codes and scales of [..., dim] in 32 bits"""
    group = x.unflatten(-1, (-1, GROUP))
    high, low = group.amax(-1), group.amin(-1)
    scale = (torch.where(high > -low, high, low) / -8.0).clamp(-65504.0, 65504.0).to(torch.float16)
    codes = (torch.round(group / scale.to(F32)[..., None]) + 8.0).clamp(0.0, 15.0)
    return torch.where(scale[..., None] == 0, 8.0, codes).to(torch.uint8).flatten(-2), scale


def values(codes, scale):
    return ((codes.to(F32) - 8.0).unflatten(-1, (-1, GROUP)) * scale.to(F32)[..., None]).flatten(-2)


def store(pool, at, x):
    codes, scale = quantise(x)
    pool["codes"][at[0], :, at[1]] = codes
    pool["scales"][at[0], :, at[1]] = scale


def read(pool, at):
    return values(pool["codes"][at[0], :, at[1]], pool["scales"][at[0], :, at[1]])


def rotate(x, cos, sin, layout):
    if layout == "pairs":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def plain_append(state):
    case = state["case"]
    at = places(state["row_start"], state["held"], state["pages"], case["page"], len(state["k"]))
    angle = (case["first"] + at[2]).to(F64)[:, None] * state["freqs"].to(F64)
    cos, sin = angle.cos().to(F32)[:, None], angle.sin().to(F32)[:, None]
    store(state["k_pool"], at, rotate(state["k"].to(F32), cos, sin, case["layout"]))
    store(state["v_pool"], at, state["v"].to(F32))
    state["q_out"].copy_(rotate(state["q"].to(F32), cos, sin, case["layout"]))
    return plain_read(state) + (state["q_out"],)


def plain_read(state):
    at = places(state["row_start"], state["held"], state["pages"], state["case"]["page"], len(state["k_back"]))
    state["k_back"].copy_(read(state["k_pool"], at))
    state["v_back"].copy_(read(state["v_pool"], at))
    return state["k_back"], state["v_back"]


def plain_attend(state):
    """all sequences at once, padded to the longest"""
    case = state["case"]
    S, H, G, D, most = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["rows_most"]
    start, held, R = state["row_start"].long(), state["held"].long(), len(state["q"])
    rows = start[1:] - start[:-1]
    table = state["pages"].clamp(min=0).long()

    def cached(pool):                # [sequences, kv heads, tokens, dim]
        return values(pool["codes"][table].transpose(1, 2).flatten(2, 3), pool["scales"][table].transpose(1, 2).flatten(2, 3))

    i = torch.arange(most, device=start.device)
    row = torch.where(i < rows[:, None], start[:-1, None] + i, R)                              # [sequences, rows], R: none
    q = torch.cat([state["q"].to(F32), torch.zeros(1, H, D, device=start.device)])[row].view(S, most, G, H // G, D).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k = cached(state["k_pool"])
    score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(D)                                  # [sequences, kv heads, heads of the group * rows, tokens]
    seen = torch.arange(k.shape[2], device=start.device) < (held - rows)[:, None, None] + i[:, None] + 1
    score = score.unflatten(2, (-1, most)).masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    weight = (weight / torch.where(total == 0, 1.0, total)).flatten(2, 3)
    out = torch.matmul(weight, cached(state["v_pool"])).unflatten(2, (-1, most)).permute(0, 3, 1, 2, 4).reshape(S * most, H, D)
    state["out"].copy_(out[(row < R).view(-1)])
    return state["out"]


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": plain_append, "read": plain_read, "attend": plain_attend}[op](state)
    ops, stream = state["ops"], torch.cuda.current_stream()
    cache = state["k_pool"], state["v_pool"], state["pages"], state["row_start"], state["held"]
    if op == "append":
        ops.kv_append_4bit(state["k"], state["v"], *cache, freqs=state["freqs"], layout=state["case"]["layout"], first_pos=state["case"]["first"], q=state["q"], q_out=state["q_out"],
                           stream=stream)
        ops.kv_read_4bit(*cache, state["k_back"], state["v_back"], stream=stream)
        return state["k_back"], state["v_back"], state["q_out"]
    if op == "read":
        ops.kv_read_4bit(*cache, state["k_back"], state["v_back"], stream=stream)
        return state["k_back"], state["v_back"]
    ops.attention_4bit(state["q"], *cache, state["out"], state["workspace"], max_rows=state["case"]["rows_most"], stream=stream)
    return state["out"]


# -------------------------------------------------------------------------------------------------------- 64-bit definitions
def coded(x):
    """what the cache gives back for these rows, in 64 bits"""
    y = x.to(F64).reshape(*x.shape[:-1], -1, GROUP)
    m = torch.gather(y, -1, y.abs().argmax(-1, keepdim=True))
    m = torch.where((y == -m.abs()).any(-1, keepdim=True), -m.abs(), m)        # of m and -m the negative one
    s = (-m / 8).clamp(-65504.0, 65504.0).to(torch.float16).to(F64)
    c = torch.where(s == 0, 0.0, torch.round(y / torch.where(s == 0, 1.0, s))).clamp(-8, 7)
    return (c * s).reshape(x.shape)


def exact(case, seed):
    s = inputs(case, seed)
    rows, held = lengths(case)
    G, D = case["kv_heads"], case["dim"]
    if case["op"] == "append":
        k, q = s["k"].to(F64), s["q"].to(F64)
        pos = torch.cat([torch.arange(o - r, o) for r, o in zip(rows, held)]).to(k.device) + case["first"]
        turn = torch.polar(torch.ones(1, 1, 1, device=k.device, dtype=F64), (pos.to(F64)[:, None] * s["freqs"].to(F64))[:, None])

        def turned(x):
            if case["layout"] == "pairs":
                return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], D // 2, 2).contiguous()) * turn).reshape(x.shape)
            z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        return coded(turned(k)), coded(s["v"]), turned(q)

    ends = [0]
    for o in held:
        ends.append(ends[-1] + o)
    if case["op"] == "read":
        pick = torch.cat([torch.arange(e - r, e) for r, e in zip(rows, ends[1:])]).to(s["k_before"].device)
        return coded(s["k_before"][pick]), coded(s["v_before"][pick])

    out = torch.zeros(sum(rows), case["heads"], D, device=s["q"].device, dtype=F64)
    r0 = 0
    for i, (r, o) in enumerate(zip(rows, held)):
        if r == 0:
            continue
        k, v = (coded(s[n][ends[i]:ends[i + 1]]).transpose(0, 1) for n in ("k_before", "v_before"))       # [kv heads, tokens, dim]
        seen = torch.arange(o, device=k.device)[None] <= torch.arange(o - r, o, device=k.device)[:, None]
        q = s["q"][r0:r0 + r].to(F64).view(r, G, -1, D)
        for j in range(q.shape[2]):
            weights = torch.softmax((q[:, :, j].transpose(0, 1) @ k.transpose(1, 2) * D ** -0.5).masked_fill(~seen, -math.inf), -1)
            out[r0:r0 + r].view(r, G, -1, D)[:, :, j] = (weights @ v).transpose(0, 1)
        r0 += r
    return out
