"""Performance cases of the serving operators: many requests over one paged KV cache.

Kinds (key "kind" of a case):
  plan    the bookkeeping of a step: pages for the tokens that the requests bring, their block tables,
          positions and cache slots, from the requests' lengths
  paged   causal attention of each request's new tokens (one, or a chunk) over its pages
  prompt  causal attention of whole prompts of different lengths, packed one behind the other

Lengths: a plan's come from the seed; of the others the case fixes them, as they decide how much work a pass is.
"""
import math
import random

import torch

own = False

# query heads, kv heads, head size, attention scale (layer.GEMMA_4B, layer.GEMMA_27B, synth_gguf.E2B's local and global layers)
SHAPES = {"4b": (8, 4, 256, 256 ** -0.5), "27b": (32, 16, 128, 128 ** -0.5), "e2b": (8, 1, 256, 1.0), "e2b_global": (8, 1, 512, 1.0)}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step of a busy server: one token each, the smallest call
        {"name": "plan_decode", "kind": "plan", "seqs": 64, "tokens": 64, "one": True, "ctx": 4096, "page": 16, "pad": 0, "free": 1.2},
        # a step that takes in a burst of prompts, in a buffer with room to spare
        {"name": "plan_prompts", "kind": "plan", "seqs": 250, "tokens": 65000, "one": False, "ctx": 3000, "page": 16, "pad": 536, "free": 1.1},
        # the next token of one chat: latency
        {"name": "token_4b", "kind": "paged", "shape": "4b", "seqs": 1, "chunks": 0, "new": 1, "ctx": 1250, "page": 16, "act": "f32",
         "window": 0, "softcap": 0.0, "mix": 1},
        # decode of several chats with f32 caches
        {"name": "decode_4b_f32", "kind": "paged", "shape": "4b", "seqs": 16, "chunks": 0, "new": 1, "ctx": 8192, "page": 16, "act": "f32",
         "window": 0, "softcap": 0.0, "mix": 2},
        # decode of a full batch of the larger model with bf16 caches
        {"name": "decode_27b_bf16", "kind": "paged", "shape": "27b", "seqs": 64, "chunks": 0, "new": 1, "ctx": 8000, "page": 64, "act": "bf16",
         "window": 0, "softcap": 0.0, "mix": 3},
        # a local layer of the small model, eight query heads on one kv head, odd batch
        {"name": "decode_e2b_local", "kind": "paged", "shape": "e2b", "seqs": 33, "chunks": 0, "new": 1, "ctx": 4096, "page": 16, "act": "bf16",
         "window": 512, "softcap": 0.0, "mix": 4},
        # one chunk of a long prompt behind what is cached already, f32
        {"name": "chunk_4b_f32", "kind": "paged", "shape": "4b", "seqs": 1, "chunks": 1, "new": 512, "ctx": 1501, "page": 16, "act": "f32",
         "window": 0, "softcap": 0.0, "mix": 5},
        # chunks of three prompts next to the decode of 21 requests, soft-capped scores
        {"name": "mixed_27b_bf16", "kind": "paged", "shape": "27b", "seqs": 24, "chunks": 3, "new": 500, "ctx": 4000, "page": 32, "act": "bf16",
         "window": 0, "softcap": 50.0, "mix": 6},
        # a short question to the small model
        {"name": "prompt_short", "kind": "prompt", "shape": "e2b", "seqs": 1, "tokens": 37, "act": "f32", "window": 0, "softcap": 0.0, "mix": 7},
        # three prompts with the reference's f32 activations
        {"name": "prompt_4b_f32", "kind": "prompt", "shape": "4b", "seqs": 3, "tokens": 2048, "act": "f32", "window": 0, "softcap": 0.0, "mix": 8},
        # five prompts through a sliding-window layer
        {"name": "prompt_4b_local", "kind": "prompt", "shape": "4b", "seqs": 5, "tokens": 4099, "act": "bf16", "window": 512, "softcap": 0.0, "mix": 9},
        # two long documents through the larger model: the largest case
        {"name": "prompt_27b_bf16", "kind": "prompt", "shape": "27b", "seqs": 2, "tokens": 8192, "act": "bf16", "window": 0, "softcap": 0.0, "mix": 10},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "paged", "paged", "prompt"])
    if kind == "plan":
        seqs, one = _log_int(rng, 1, 600), rng.random() < 0.5
        return {"kind": kind, "seqs": seqs, "tokens": seqs if one else seqs + _log_int(rng, 1, 60000), "one": one, "ctx": _log_int(rng, 16, 8192),
                "page": rng.choice([8, 16, 32, 64, 100, 256]), "pad": rng.choice([0, rng.randint(1, 500)]), "free": rng.choice([1.0, 1.3, 0.8])}
    shape, act = rng.choice(sorted(SHAPES)), rng.choice(sorted(DTYPES))
    nh, nkv, D, _ = SHAPES[shape]
    case = {"kind": kind, "shape": shape, "act": act, "window": rng.choice([0, 0, 512, rng.randint(1, 1500)]),
            "softcap": rng.choice([0.0, 0.0, 50.0]), "mix": rng.randint(1, 10 ** 6)}
    if kind == "paged":
        case["page"] = rng.choice([8, 16, 16, 32, 64, 100, 256])
        case["new"], case["ctx"] = (1 if rng.random() < 0.5 else _log_int(rng, 2, 600)), _log_int(rng, 16, 12000)
        # caches of at most 2 GiB in all, no more products than the largest listed case
        length = case["ctx"] + case["new"]
        most = min(64, 2 ** 31 // (8 * nkv * D * length), 2 ** 36 // (nh * D * case["new"] * length))
        case["seqs"] = _log_int(rng, 1, max(1, most))
        case["chunks"] = 0 if case["new"] == 1 else rng.choice([case["seqs"], rng.randint(1, case["seqs"])])
        return case
    case["tokens"] = _log_int(rng, 1, {"4b": 4096, "27b": 4096, "e2b": 4096, "e2b_global": 2048}[shape])
    case["seqs"] = _log_int(rng, 1, min(16, case["tokens"]))
    return case


# ---- lengths and seeded data ---------------------------------------------------------------

def _cut(rng, total, parts):
    """`total` in `parts` ragged lengths of at least 1."""
    at = sorted(rng.randint(0, total - parts) for _ in range(parts - 1))
    return [b - a + 1 for a, b in zip([0] + at, at + [total - parts])]


def _lengths(case):
    """(tokens in the cache before, new tokens) of each request."""
    rng = random.Random(case["mix"])
    n = case["seqs"]
    if case["kind"] == "prompt":
        return [0] * n, _cut(rng, case["tokens"], n)
    new = [(rng.randint((case["new"] + 1) // 2, case["new"]) if n > 1 else case["new"]) if i < case["chunks"] else 1 for i in range(n)]
    ctx = [rng.randint(case["ctx"] // 8, case["ctx"]) if n > 1 else case["ctx"] for _ in range(n)]
    at = list(range(n))
    rng.shuffle(at)
    return ctx, [new[i] for i in at]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def _cumulated(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _pages(n, page):
    return -(-n // page)


def _plan_inputs(case, seed):
    rng = random.Random(int(seed) * 7919 + 13)
    n, page = case["seqs"], case["page"]
    longest = 1 if case["one"] else 2 * case["tokens"] // n
    new, left = [], case["tokens"]
    for _ in range(n):
        new.append(min(left, 1 if case["one"] else rng.randint(0, longest)))
        left -= new[-1]
    ctx = [rng.randint(0, case["ctx"]) for _ in range(n)]
    have = [_pages(c, page) for c in ctx]
    need = sum(_pages(c + m, page) - h for c, m, h in zip(ctx, new, have))
    free = max(1, int(need * case["free"]))
    most = _pages(case["ctx"] + longest, page) + 1
    g = _gen(seed)
    pool = torch.randperm(sum(have) + free, generator=g, device="cuda", dtype=torch.int32)
    at = _ints(_cumulated(have)[:-1]).long()[:, None] + torch.arange(most, device="cuda")
    held = torch.arange(most, device="cuda") < _ints(have)[:, None]
    table = torch.where(held, pool[at.clamp(max=pool.numel() - 1)], -1)
    return {"ctx": _ints(ctx), "new": _ints(new), "free": pool[sum(have):].contiguous(), "table": table, "most": most}


def _inputs(case, seed):
    """The tensors an attention pass reads."""
    g = _gen(seed)
    nh, nkv, D, _ = SHAPES[case["shape"]]
    dt = DTYPES[case["act"]]
    ctx, new = _lengths(case)
    total = [c + m for c, m in zip(ctx, new)]
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda", dtype=dt)  # noqa: E731
    t = {"q": randn(sum(new), nh * D), "cu": _ints(_cumulated(new)), "len": _ints(total)}
    if case["shape"].startswith("e2b"):
        # this model scales its scores by its query norm's weights, not by the head size: scores of a deviation of four
        t["q"] = (t["q"].float() * (4 * D ** -0.5)).to(dt)
    if case["kind"] == "prompt":
        t["k"], t["v"] = randn(sum(new), nkv * D), randn(sum(new), nkv * D)
        return t
    page = case["page"]
    held = [_pages(x, page) for x in total]
    most, pool = max(held), sum(held) + 3
    ids = torch.randperm(pool, generator=g, device="cuda", dtype=torch.int32)
    at = _ints(_cumulated(held)[:-1]).long()[:, None] + torch.arange(most, device="cuda")
    t["table"] = torch.where(torch.arange(most, device="cuda") < _ints(held)[:, None], ids[at.clamp(max=pool - 1)], -1)
    t["pages"] = pool
    t["k"], t["v"] = randn(pool * page, nkv * D), randn(pool * page, nkv * D)
    return t


_device = None


def _dev():
    """The program's device and its one stream."""
    global _device
    if _device is None:
        from ziglm_amd.device import HipDevice
        _device = HipDevice()
    return _device


def _act(case):
    from ziglm_amd import bridge
    return bridge.F32 if case["act"] == "f32" else bridge.BF16


def prepare(case, seed):
    if case["kind"] == "plan":
        t = _plan_inputs(case, seed)
        n, cap = case["seqs"], case["tokens"] + case["pad"]
        like = lambda m, dt=torch.int32: torch.empty(m, device="cuda", dtype=dt)  # noqa: E731
        s = {"case": case, "t": t, "cap": cap}
        if own:
            s["out"] = {"cu": like(n + 1), "len": like(n), "pos": like(cap), "slot": like(cap, torch.int64), "table": t["table"], "state": like(2)}
        return s
    t = _inputs(case, seed)
    nh, nkv, D, _ = SHAPES[case["shape"]]
    ctx, new = _lengths(case)
    s = {"case": case, "t": t, "most_new": max(new), "most": max(c + m for c, m in zip(ctx, new))}
    if own:
        # what a serving program keeps: the output buffer and the workspace
        s["out"] = torch.empty_like(t["q"])
        n, T = case["seqs"], t["q"].shape[0]
        if case["kind"] == "paged":
            need = _dev().attentionPagedWorkspaceBytes(_act(case), n, T, s["most"], nh, nkv, D, case["window"])
        else:
            need = _dev().attentionPromptWorkspaceBytes(_act(case), n, T, nh, nkv, D, case["window"])
        s["ws"] = torch.empty(max(16, need), device="cuda", dtype=torch.uint8)
    return s


# ---- the passes ----------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return _plain_plan(state) if state["case"]["kind"] == "plan" else _plain_attention(state)


def _run_own(s):
    case, t, dev = s["case"], s["t"], _dev()
    n = case["seqs"]
    p = lambda x: x.data_ptr()  # noqa: E731
    if case["kind"] == "plan":
        o = s["out"]
        dev.pagedPlan(p(t["ctx"]), p(t["new"]), n, case["page"], t["most"], p(t["free"]), t["free"].numel(), None, p(o["table"]), s["cap"],
                      p(o["cu"]), p(o["len"]), p(o["pos"]), p(o["slot"]), p(o["state"]))
        return o
    nh, nkv, D, scale = SHAPES[case["shape"]]
    T = t["q"].shape[0]
    if case["kind"] == "paged":
        dev.attentionPaged(_act(case), p(t["q"]), p(t["k"]), p(t["v"]), p(s["out"]), t["pages"], case["page"], nkv * D, p(t["table"]),
                           t["table"].shape[1], p(t["cu"]) if case["chunks"] else None, p(t["len"]), n, T, s["most"], nh, nkv, D, scale,
                           case["softcap"], case["window"], p(s["ws"]), s["ws"].numel())
    else:
        dev.attentionPrompt(_act(case), p(t["q"]), p(t["k"]), p(t["v"]), p(s["out"]), nh * D, nkv * D, p(t["cu"]), n, T, nh, nkv, D, scale,
                            case["softcap"], case["window"], p(s["ws"]), s["ws"].numel())
    return s["out"]


def _plain_plan(s):
    case, t, cap = s["case"], s["t"], s["cap"]
    page, most = case["page"], t["most"]
    ctx, free, table = t["ctx"].long(), t["free"], t["table"]
    # the tokens that fit the table and the token buffer
    new = torch.minimum(t["new"].long().clamp(min=0), (most * page - ctx).clamp(min=0))
    new = torch.minimum(new, (cap - (new.cumsum(0) - new)).clamp(min=0))
    # their pages, in the order of the requests; where the free list ends, the tokens that have a page
    have = (ctx + page - 1) // page
    need = (ctx + new + page - 1) // page - have
    first = need.cumsum(0) - need
    got = torch.minimum((free.numel() - first).clamp(min=0), need)
    new = torch.minimum(new, (have + got) * page - ctx)
    cu = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    j = torch.arange(most, device="cuda") - have[:, None]
    fresh = (j >= 0) & (j < got[:, None])
    table = torch.where(fresh, free[(first[:, None] + j).clamp(0, free.numel() - 1)], table)
    at = torch.arange(cap, device="cuda")
    of = torch.searchsorted(cu[1:], at, right=True).clamp(max=case["seqs"] - 1)
    pos = ctx[of] + at - cu[of]
    slot = table[of, (pos // page).clamp(max=most - 1)].long() * page + pos % page
    real = at < cu[-1]
    dropped = t["new"].long().clamp(min=0).sum() - cu[-1]
    return {"cu": cu.int(), "len": (ctx + new).int(), "pos": torch.where(real, pos, -1).int(), "slot": torch.where(real, slot, -1),
            "table": table, "state": torch.stack([got.sum(), dropped]).int()}


def _plain_attention(s):
    case, t = s["case"], s["t"]
    nh, nkv, D, scale = SHAPES[case["shape"]]
    n, Q, L = case["seqs"], s["most_new"], s["most"]
    T = t["q"].shape[0]
    cu = t["cu"].long()
    key = torch.arange(L, device="cuda")
    if case["kind"] == "paged":
        rows = t["table"].long().clamp(min=0)[:, key // case["page"]] * case["page"] + key % case["page"]
    else:
        rows = (cu[:-1, None] + key).clamp(max=T - 1)
    # [n][kv heads][...], requests padded to the longest
    k = t["k"][rows].view(n, L, nkv, D).float().permute(0, 2, 3, 1).contiguous()
    v = t["v"][rows].view(n, L, nkv, D).float().permute(0, 2, 1, 3).contiguous()
    at = (cu[:-1, None] + torch.arange(Q, device="cuda")).clamp(max=T - 1)
    q = t["q"][at].view(n, Q, nkv, nh // nkv, D).float().permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, D)
    x = (q @ k) * scale
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    x = x.view(n, nkv, nh // nkv, Q, L)
    pos = (t["len"].long() - (cu[1:] - cu[:-1]))[:, None] + torch.arange(Q, device="cuda")
    hide = key > pos[..., None]
    if case["window"]:
        hide = hide | (key <= pos[..., None] - case["window"])
    x = x.masked_fill_(hide[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    total = x.sum(-1, keepdim=True)
    o = (x.view(n, nkv, -1, L) @ v).view(n, nkv, nh // nkv, Q, D) / total
    tok = torch.arange(T, device="cuda")
    of = torch.searchsorted(cu[1:], tok, right=True)
    return o.permute(0, 3, 1, 2, 4)[of, tok - cu[of]].reshape(T, nh * D).to(t["q"].dtype)


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    if case["kind"] == "plan":
        n, cap = case["seqs"], case["tokens"] + case["pad"]
        fresh = case["tokens"] // case["page"] + n // 2
        return {"bytes": 4 * (2 * n) + 8 * fresh + 4 * (2 * n + 3) + 12 * cap, "flops": 4 * case["tokens"]}
    nh, nkv, D, _ = SHAPES[case["shape"]]
    es = 4 if case["act"] == "f32" else 2
    ctx, new = _lengths(case)
    seen, pairs = 0, 0
    for c, m in zip(ctx, new):
        win = case["window"] or c + m
        seen += min(c, win - 1) + m
        # sum over i < m of min(c + i + 1, win)
        rise = max(0, min(m, win - c))
        pairs += rise * c + rise * (rise + 1) // 2 + (m - rise) * win
    return {"bytes": es * (2 * nh * D * sum(new) + 2 * nkv * D * seen), "flops": 4 * pairs * nh * D}


# ---- the same in 64 bits, without the framework -----------------------------------------------

def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    t = _inputs(case, seed)
    nh, nkv, D, scale = SHAPES[case["shape"]]
    g = nh // nkv
    ctx, new = _lengths(case)
    q = t["q"].view(-1, nh, D)
    out = torch.empty((q.shape[0], nh, D), device="cuda", dtype=torch.float64)
    a = 0
    for i, (c, m) in enumerate(zip(ctx, new)):
        if case["kind"] == "paged":
            ids = t["table"][i, :_pages(c + m, case["page"])].long()
            rows = (ids[:, None] * case["page"] + torch.arange(case["page"], device="cuda")).reshape(-1)[:c + m]
        else:
            rows = torch.arange(a, a + m, device="cuda")
        far = torch.arange(c, c + m, device="cuda")[:, None] - torch.arange(c + m, device="cuda")[None]
        hide = far < 0
        if case["window"]:
            hide |= far >= case["window"]
        for h in range(nh):
            k, v = (t[x][rows].view(-1, nkv, D)[:, h // g].double() for x in ("k", "v"))
            s = (q[a:a + m, h].double() @ k.T) * scale
            if case["softcap"]:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            out[a:a + m, h] = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ v
        a += m
    return out.view(-1, nh * D)
