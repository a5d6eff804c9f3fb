"""The operators of a serving step over a paged key-value cache, as measured cases.

A program that serves many requests at once runs, a step:

  plan       one call: from the requests' lengths the pages they take or give
             back, each new token's slot and position, the ragged offsets
  store      a layer: the step's k and v rows into their slots of the cache
  attention  a layer: each request's new queries over its pages
  logprobs   one call: log probabilities of the chosen tokens, the entropy
             and the most likely alternatives

`run` computes a case with elementary torch operations in 32 bits, or (`own`)
with the library's calls.  Sizes: the model's 24 query and 4 key/value heads of
256 and its vocabulary of 248320, and generic ones beside them; 1 to 509
requests, caches of 1 to 32768 positions, drafts being verified and chunks of
prompts among the decoded tokens.
"""
import importlib
import math

import torch

own = False


def _bh():
    return importlib.import_module("ternary-bonsai-inference_amd")


def listed():
    return [
        # a step of a few decoders: one new token each
        {"name": "plan_decode", "kind": "plan", "reqs": 16, "tokens": 16, "page": 16,
         "ctx": 4096, "chunk": 1},
        # a busy server's step: decoders, finished requests, prompts arriving
        {"name": "plan_prompts", "kind": "plan", "reqs": 509, "tokens": 8192, "page": 32,
         "ctx": 8192, "chunk": 2048},
        # one layer's append for a batch of decoders
        {"name": "store_decode", "kind": "store", "tokens": 32, "heads": 4, "hd": 256,
         "page": 16, "f16": True, "by_head": False},
        # one layer's append for a chunk of a prompt, pages laid out head by head
        {"name": "store_prompt", "kind": "store", "tokens": 4001, "heads": 4, "hd": 256,
         "page": 64, "f16": False, "by_head": True},
        # one conversation, one new token
        {"name": "attn_one", "kind": "attn", "reqs": 1, "ctx": 5000, "new": 1, "chunk": 0,
         "page": 16, "f16": True, "q_heads": 24, "heads": 4, "hd": 256, "by_head": False},
        # a batch of decoders whose caches run from short to long
        {"name": "attn_batch", "kind": "attn", "reqs": 64, "ctx": 16384, "new": 1, "chunk": 0,
         "page": 16, "f16": True, "q_heads": 24, "heads": 4, "hd": 256, "by_head": False},
        # the same over the f32 cache, which is the framework's default
        {"name": "attn_batch_f32", "kind": "attn", "reqs": 13, "ctx": 8192, "new": 1, "chunk": 0,
         "page": 48, "f16": False, "q_heads": 24, "heads": 4, "hd": 256, "by_head": False},
        # drafts of up to 8 tokens being verified, other heads
        {"name": "attn_draft", "kind": "attn", "reqs": 24, "ctx": 8192, "new": 8, "chunk": 0,
         "page": 32, "f16": True, "q_heads": 32, "heads": 8, "hd": 128, "by_head": True},
        # a chunk of a prompt in the same step as decoders
        {"name": "attn_chunk", "kind": "attn", "reqs": 8, "ctx": 8192, "new": 1, "chunk": 512,
         "page": 64, "f16": True, "q_heads": 24, "heads": 4, "hd": 256, "by_head": False},
        # the sampled tokens of a few decoders, as a client asks for them
        {"name": "logprobs_decode", "kind": "logprobs", "rows": 8, "vocab": 248320, "top": 20,
         "temp": 1.0, "pad": 0, "banned": False},
        # a prompt scored token by token
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 512, "vocab": 248320, "top": 5,
         "temp": 1.0, "pad": 0, "banned": False},
        # a small odd vocabulary, some tokens banned, no alternatives wanted
        {"name": "logprobs_plain", "kind": "logprobs", "rows": 61, "vocab": 32003, "top": 0,
         "temp": 0.7, "pad": 29, "banned": True},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["plan", "store", "attn", "attn", "logprobs"])
    if kind == "plan":
        chunk = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 17, 2048)])
        reqs = _log_int(rng, 1, 509)
        return {"kind": kind, "reqs": reqs, "tokens": max(reqs, _log_int(rng, 8, 8192)),
                "page": rng.choice([16, 32, 64, 128, 24, 100]), "ctx": _log_int(rng, 64, 8192),
                "chunk": chunk}
    if kind == "store":
        heads, hd = rng.choice([(4, 256), (8, 128), (2, 64), (3, 80)])
        return {"kind": kind, "tokens": _log_int(rng, 1, 4001), "heads": heads, "hd": hd,
                "page": rng.choice([16, 32, 64, 128, 24]), "f16": rng.random() < 0.5,
                "by_head": rng.random() < 0.3}
    if kind == "logprobs":
        rows = _log_int(rng, 1, 512)
        vocab = rng.choice([248320, _log_int(rng, 1000, 248320)])
        return {"kind": kind, "rows": rows, "vocab": vocab,
                "top": rng.choice([0, 1, 5, 20, rng.randint(2, 32)]),
                "temp": rng.choice([1.0, 0.7, round(rng.uniform(0.3, 1.5), 3)]),
                "pad": rng.choice([0, 0, rng.randint(1, 200)]), "banned": rng.random() < 0.4}
    q_heads, heads, hd = rng.choice([(24, 4, 256), (24, 4, 256), (32, 8, 128), (16, 2, 64),
                                     (9, 3, 128), (8, 8, 64)])
    form = rng.choice(["decode", "decode", "draft", "chunk"])
    page = rng.choice([16, 16, 32, 64, 128, 48])
    case = {"kind": kind, "page": page, "f16": rng.random() < 0.65, "q_heads": q_heads,
            "heads": heads, "hd": hd, "by_head": rng.random() < 0.3, "chunk": 0, "new": 1}
    if form == "decode":
        case["reqs"] = _log_int(rng, 1, 96)
        case["ctx"] = min(_log_int(rng, 32, 32768), 480000 // case["reqs"])
    elif form == "draft":
        case["reqs"], case["new"] = _log_int(rng, 1, 32), rng.randint(2, 10)
        case["ctx"] = min(_log_int(rng, 32, 16384), 160000 // case["reqs"])
    else:
        case["reqs"], case["chunk"] = rng.randint(1, 8), _log_int(rng, 17, 512)
        case["ctx"] = _log_int(rng, 600, 8192)
    if not case["f16"]:
        case["ctx"] = max(16, case["ctx"] // 2)
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _host(seed):
    return torch.Generator().manual_seed(seed)


def _lengths(case, seed):
    """Host lists: positions in each request's cache after the step, and new tokens."""
    g = _host(seed)
    reqs, ctx = case["reqs"], case["ctx"]
    # long tails, as conversations have them: most caches well under the longest
    u = torch.rand(reqs, generator=g, dtype=torch.float64)
    total = (ctx * torch.exp(-2.0 * u)).long().clamp(min=1)
    if reqs == 1:
        total[0] = ctx - int(u[0] * ctx / 50)
    new = torch.randint(1, case["new"] + 1, (reqs,), generator=g)
    if case["chunk"]:
        new[reqs // 2] = case["chunk"]
        total[reqs // 2] = max(int(total[reqs // 2]), case["chunk"])
    return torch.maximum(total, new).tolist(), new.tolist()


def _cache(case, n_pages, seed):
    """K and V [page][position][head][dim] in the case's layout and type."""
    dt = torch.float16 if case["f16"] else torch.float32
    page, heads, hd = case["page"], case["heads"], case["hd"]
    shape = (n_pages, heads, page, hd) if case["by_head"] else (n_pages, page, heads, hd)
    g = _gen(seed)
    k, v = (torch.randn(shape, generator=g, device="cuda", dtype=dt) for _ in range(2))
    if case["by_head"]:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return k, v


def prepare(case, seed):
    s = {"case": case}
    {"plan": _prepare_plan, "store": _prepare_store, "attn": _prepare_attn,
     "logprobs": _prepare_logprobs}[case["kind"]](s, case, seed)
    if own:  # the argument blocks that a program with fixed buffers keeps
        s["args"] = _arguments(s, case)
    return s


def _prepare_plan(s, case, seed):
    g = _host(seed)
    reqs, page, ctx = case["reqs"], case["page"], case["ctx"]
    width = -(-(ctx + case["chunk"]) // page) + 1
    cached = (ctx * torch.rand(reqs, generator=g, dtype=torch.float64) ** 2).long()
    new = torch.ones(reqs, dtype=torch.long)
    u = torch.rand(reqs, generator=g)
    if case["chunk"] > 1:
        long = u < 0.05
        new[long] = torch.randint(1, case["chunk"] + 1, (int(long.sum()),), generator=g)
        cached[u < 0.02] = 0
    new[(u > 0.95) & (cached > 0)] = -1  # finished: its pages go back
    have = -(-cached // page)
    n_pages = reqs * width + 8
    order = torch.randperm(n_pages, generator=g).int()
    table = torch.full((reqs, width), -1, dtype=torch.int32)
    used = torch.arange(width)[None, :] < have[:, None]
    taken = int(have.sum())
    table[used] = order[:taken]
    # the rest of the pool is held elsewhere, but for about what a step takes
    n_free = min(n_pages - taken, case["tokens"] // page + reqs // 2 + 4)
    free = torch.full((n_pages,), -1, dtype=torch.int32)
    free[:n_free] = order[taken:taken + n_free]
    dev = dict(device="cuda")
    s.update(cached=cached.int().to(**dev), new=new.int().to(**dev), table=table.to(**dev),
             free=free.to(**dev), n_free=torch.tensor([n_free], dtype=torch.int32, **dev))
    i32 = dict(dtype=torch.int32, **dev)
    s.update(kv_len=torch.zeros(reqs, **i32), q_start=torch.zeros(reqs + 1, **i32),
             slots=torch.zeros(case["tokens"], **i32), pos=torch.zeros(case["tokens"], 4, **i32),
             n_free_out=torch.zeros(1, **i32), refused=torch.zeros(1, **i32))


def _prepare_store(s, case, seed):
    n, page = case["tokens"], case["page"]
    n_pages = 2 * n // page + 9
    k_cache, v_cache = _cache(case, n_pages, seed)
    g = _gen(seed + 1)
    elems = case["heads"] * case["hd"]
    rows = [torch.randn((n, elems), generator=g, device="cuda") for _ in range(2)]
    # chunks of consecutive positions in shuffled pages, a few padding tokens
    blocks = torch.randperm(n_pages, generator=g, device="cuda")
    t = torch.arange(n, device="cuda") + seed % page
    slots = blocks[t // page] * page + t % page
    slots[torch.rand(n, generator=g, device="cuda") < 0.02] = -1
    s.update(k=rows[0], v=rows[1], slots=slots.int(), k_cache=k_cache, v_cache=v_cache)


def _prepare_attn(s, case, seed):
    total, new = _lengths(case, seed)
    page, reqs = case["page"], case["reqs"]
    have = [-(-t // page) for t in total]
    width, n_pages = max(have) + 1, sum(have) + 3
    order = torch.randperm(n_pages, generator=_host(seed + 2)).int()
    table = torch.full((reqs, width), -1, dtype=torch.int32)
    used = torch.arange(width)[None, :] < torch.tensor(have)[:, None]
    table[used] = order[:sum(have)]
    k_cache, v_cache = _cache(case, n_pages, seed)
    n_tok = reqs * case["new"] + case["chunk"]  # the step's buffers: the last rows may be padding
    start = torch.zeros(reqs + 1, dtype=torch.int32)
    start[1:] = torch.tensor(new).cumsum(0)
    q = torch.randn((n_tok, case["q_heads"], case["hd"]), generator=_gen(seed + 1), device="cuda")
    s.update(q=q, out=torch.zeros_like(q), k_cache=k_cache, v_cache=v_cache,
             table=table.cuda(), q_start=start.cuda(),
             kv_len=torch.tensor(total, dtype=torch.int32, device="cuda"),
             max_new=max(new), longest=max(total))


def _prepare_logprobs(s, case, seed):
    rows, vocab = case["rows"], case["vocab"]
    g = _gen(seed)
    wide = torch.randn((rows, vocab + case["pad"]), generator=g, device="cuda")
    # logits of a language model: a wide bulk, a few tokens far above it; coarse
    # values, so that some are equal
    wide.mul_(2.5).mul_(64.0).round_().div_(64.0)
    at = torch.randint(0, vocab, (rows, 6), generator=g, device="cuda")
    lift = 8.0 + 6.0 * torch.rand((rows, 6), generator=g, device="cuda")
    wide.scatter_(1, at, lift)
    x = wide[:, :vocab]
    tokens = at[:, 0].clone()
    far = torch.rand(rows, generator=g, device="cuda") < 0.3
    tokens[far] = torch.randint(0, vocab, (rows,), generator=g, device="cuda")[far]
    if case["banned"]:
        x[:, torch.randint(0, vocab, (vocab // 10,), generator=g, device="cuda")] = -math.inf
    f32 = dict(dtype=torch.float32, device="cuda")
    s.update(x=x, tokens=tokens.int(), logprob=torch.zeros(rows, **f32),
             entropy=torch.zeros(rows, **f32),
             top_ids=torch.zeros((rows, case["top"]), dtype=torch.int32, device="cuda"),
             top_logprobs=torch.zeros((rows, case["top"]), **f32))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _arguments(s, case):
    bh = _bh()
    if case["kind"] == "plan":
        return bh.make_paged_plan_args(
            s["cached"], s["new"], s["table"], s["free"], s["n_free"], case["page"],
            kv_len=s["kv_len"], q_start=s["q_start"], slots=s["slots"], pos=s["pos"],
            n_free_out=s["n_free_out"], n_refused=s["refused"])
    if case["kind"] == "store":
        return bh.make_paged_cache(s["k_cache"], s["v_cache"])
    if case["kind"] == "attn":
        cache = bh.make_paged_cache(s["k_cache"], s["v_cache"])
        return bh.make_attention_paged_args(cache, s["q"], s["q_start"], s["kv_len"], s["table"],
                                            out=s["out"], max_new=s["max_new"])
    return bh.make_token_logprobs_args(
        s["x"], s["tokens"], n_top=case["top"], inv_temp=1.0 / case["temp"],
        logprob=s["logprob"], entropy=s["entropy"], top_ids=s["top_ids"],
        top_logprobs=s["top_logprobs"])


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        bh = _bh()
        if kind == "plan":
            bh.paged_plan(s["args"])
        elif kind == "store":
            bh.kv_store_paged(s["args"], s["k"], s["v"], s["slots"])
        elif kind == "attn":
            bh.attention_paged(s["args"])
        else:
            bh.token_logprobs(s["args"])
    else:
        {"plan": _plain_plan, "store": _plain_store, "attn": _plain_attn,
         "logprobs": _plain_logprobs}[kind](s, case)
    return _outputs(s, kind)


def _outputs(s, kind):
    if kind == "plan":
        names = ("kv_len", "q_start", "slots", "pos", "table", "free", "n_free_out", "refused")
    elif kind == "store":
        names = ("k_cache", "v_cache")
    elif kind == "attn":
        names = ("out",)
    else:
        names = ("logprob", "entropy") + (("top_ids", "top_logprobs") if s["case"]["top"] else ())
    return {n: s[n] for n in names}


def _plain_plan(s, case):
    page, n_tok = case["page"], case["tokens"]
    cached, new = s["cached"].long(), s["new"].long()
    table, free = s["table"], s["free"]
    reqs, width = table.shape
    dev = table.device
    out_of_use = new < 0
    grow = new.clamp(min=0)
    have = torch.where(cached > 0, (cached + page - 1) // page, 0)
    too_long = ~out_of_use & (cached + grow > width * page)
    grow = torch.where(too_long, 0, grow)
    need = torch.where(out_of_use | too_long, 0, (cached + grow + page - 1) // page - have)
    # pages given back, request by request and block by block, onto the stack
    block = torch.arange(width, device=dev)[None, :]
    back = out_of_use[:, None] & (block < have[:, None])
    at = back.reshape(-1).long().cumsum(0) - 1 + s["n_free"]
    padded = torch.cat([free, free.new_zeros(1)])
    padded[torch.where(back.reshape(-1), at, free.numel())] = table.reshape(-1)
    free.copy_(padded[:-1])
    avail = s["n_free"].long() + back.sum()
    # who fits: running totals over the requests, in order
    ok = ~out_of_use & ~too_long
    refused = too_long | (ok & (need > 0) & (need.cumsum(0) > avail))
    refused |= ok & (grow > 0) & (grow.cumsum(0) > n_tok)
    need = torch.where(refused, 0, need)
    grow = torch.where(refused, 0, grow)
    first = need.cumsum(0) - need
    j = block - have[:, None]
    fresh = (j >= 0) & (j < need[:, None])
    pick = (avail - 1 - first[:, None] - j).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[pick], table))
    s["n_free_out"].copy_(avail - need.sum())
    s["refused"].copy_(refused.sum())
    kv_len = torch.where(out_of_use | refused, 0, cached + grow)
    s["kv_len"].copy_(kv_len)
    ends = grow.cumsum(0)
    s["q_start"][0] = 0
    s["q_start"][1:] = ends
    t = torch.arange(n_tok, device=dev)
    r = torch.searchsorted(ends, t, right=True).clamp(max=reqs - 1)
    live = t < ends[-1]
    p = torch.where(live, kv_len[r] - ends[r] + t, 0)
    slot = table[r, (p // page).clamp(max=width - 1)].long() * page + p % page
    s["slots"].copy_(torch.where(live, slot, -1))
    s["pos"].copy_(p[:, None].expand(-1, 4))


def _plain_store(s, case):
    page, heads, hd = case["page"], case["heads"], case["hd"]
    slots = s["slots"].long()
    keep = slots >= 0
    # a padding token stores what is there already
    at = torch.where(keep, slots, 0)
    for rows, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        new = rows.view(-1, heads, hd).to(cache.dtype)[keep]
        cache[at[keep] // page, at[keep] % page] = new


def _plain_attn(s, case):
    page, q_heads, heads, hd = case["page"], case["q_heads"], case["heads"], case["hd"]
    q, kv_len, start, longest = s["q"], s["kv_len"].long(), s["q_start"].long(), s["longest"]
    reqs, dev = kv_len.numel(), q.device
    n_new = start[1:] - start[:-1]
    j = torch.arange(longest, device=dev)
    pages = s["table"].long()[:, j // page].clamp(min=0)
    k = s["k_cache"][pages, j % page].float()  # [request][position][head][dim]
    v = s["v_cache"][pages, j % page].float()
    t = torch.arange(s["max_new"], device=dev)
    row = (start[:-1, None] + t).clamp(max=q.shape[0] - 1)
    group = q_heads // heads
    qs = q[row].view(reqs, -1, heads, group, hd).permute(0, 2, 1, 3, 4).reshape(
        reqs, heads, -1, hd)
    score = torch.matmul(qs, k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(hd)
    seen = j <= (kv_len - n_new)[:, None, None] + t[None, :, None]
    seen = seen & (t[None, :] < n_new[:, None])[:, :, None]
    seen = seen[:, None, :, None, :].expand(-1, -1, -1, group, -1).reshape(
        reqs, 1, -1, longest)
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top.isinf(), 0.0, top))
    e = e / e.sum(-1, keepdim=True).clamp(min=1e-38)
    o = torch.matmul(e, v.permute(0, 2, 1, 3).contiguous())
    o = o.view(reqs, heads, -1, group, hd).permute(0, 2, 1, 3, 4).reshape(reqs, -1, q_heads, hd)
    live = t[None, :] < n_new[:, None]
    s["out"][row[live]] = o[live]


def _plain_logprobs(s, case):
    x = s["x"]
    top = x.amax(-1, keepdim=True)
    z = (x - top) * (1.0 / case["temp"])
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    s["logprob"].copy_((z.gather(1, s["tokens"].long()[:, None]) - log_total)[:, 0])
    mean = torch.where(e > 0, e * z, 0.0).sum(-1, keepdim=True) / total
    s["entropy"].copy_((log_total - mean)[:, 0])
    if case["top"]:
        ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :case["top"]]
        s["top_ids"].copy_(ids)
        s["top_logprobs"].copy_(z.gather(1, ids) - log_total)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "plan":
        # lengths in and out; per token its slot and four positions
        return {"bytes": 16 * case["reqs"] + 20 * case["tokens"], "flops": 0}
    if kind == "store":
        e = 2 if case["f16"] else 4
        return {"bytes": case["tokens"] * (case["heads"] * case["hd"] * 2 * (4 + e) + 4),
                "flops": 0}
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}
    total, new = _lengths(case, 0)  # other seeds: lengths of the same distribution
    e = 2 if case["f16"] else 4
    seen = sum(sum(range(t - n + 1, t + 1)) for t, n in zip(total, new))
    return {"bytes": 2 * e * case["heads"] * case["hd"] * sum(total)
            + 8 * sum(new) * case["q_heads"] * case["hd"],
            "flops": 4 * case["hd"] * case["q_heads"] * seen}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "plan":
        return None  # whole numbers only
    if kind == "store":
        page = case["page"]
        got = {}
        for name, rows in (("k_cache", s["k"]), ("v_cache", s["v"])):
            cache = s[name].double()
            flat = rows.double().view(-1, case["heads"], case["hd"])
            slots = s["slots"].long()
            i = torch.nonzero(slots >= 0)[:, 0]
            cache.index_put_((slots[i].div(page, rounding_mode="floor"), slots[i] % page), flat[i])
            got[name] = cache
        return got
    if kind == "attn":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        start, total = s["q_start"].tolist(), s["kv_len"].tolist()
        group = case["q_heads"] // case["heads"]
        for r, n in enumerate(total):
            pages = s["table"][r, :-(-n // case["page"])].long()
            k, v = (c[pages].flatten(0, 1)[:n].double() for c in (s["k_cache"], s["v_cache"]))
            a, b = start[r], start[r + 1]
            mask = torch.ones((b - a, n), dtype=torch.bool, device="cuda").tril(n - (b - a))
            for h in range(case["q_heads"]):
                w = s["q"][a:b, h].double() @ k[:, h // group].t().contiguous()
                w = (w / case["hd"] ** 0.5).masked_fill(~mask, -math.inf).softmax(-1)
                out[a:b, h] = w @ v[:, h // group].contiguous()
        return {"out": out}
    got = {"logprob": [], "entropy": [], "top_logprobs": []}
    for r in range(case["rows"]):
        p = torch.log_softmax(s["x"][r].double() / case["temp"], -1)
        got["logprob"].append(p[s["tokens"][r].long()])
        got["entropy"].append(-torch.special.xlogy(p.exp(), p.exp()).sum())
        if case["top"]:
            got["top_logprobs"].append(torch.sort(p, descending=True)[0][:case["top"]])
    if not case["top"]:
        del got["top_logprobs"]
    got = {n: torch.stack(v) for n, v in got.items()}
    return {**got, "top_ids": None} if case["top"] else got
