"""More operators of a serving step, as measured cases: the model's recurrent layers
for many requests at once, and beam search.

A program that serves many requests of a hybrid model (gated-delta-net layers and
attention layers) runs, beside the plan, the append and the log probabilities:

  conv    a recurrent layer: causal conv + SiLU + L2 norms of the ragged
          requests' tokens, each with its cache in a slot of a pool
  gdn     the same layer: the gated delta rule, each request's state in a slot;
          a step may read one slot and write another
  attn    an attention layer of requests that share a long prefix (the beams of
          one prompt, the users of one system prompt)
  select  a step of beam search: the best continuations of each group's beams
  reorder the beams' page tables put in order and, a layer, the pages of beams
          that went on twice copied

`run` computes a case with elementary torch operations in 32 bits (64 where sums
decide an order), or (`own`) with the library's calls.  Sizes: the model's 16 / 48
recurrent heads of 128 (10240 conv channels), 24 / 4 attention heads of 256, its
vocabulary of 248320, and generic ones beside them.
"""
import importlib
import math

import torch

own = False


def _bh():
    return importlib.import_module("ternary-bonsai-inference_amd")


def listed():
    return [
        # one conversation, one new token: a recurrent layer's state read and written
        {"name": "gdn_one", "kind": "gdn", "reqs": 1, "new": 1, "prompts": 0, "chunk": 0,
         "h_k": 16, "h_v": 48, "s": 128, "inplace": False},
        # a batch of decoders, states advanced in place
        {"name": "gdn_decode", "kind": "gdn", "reqs": 64, "new": 1, "prompts": 0, "chunk": 0,
         "h_k": 16, "h_v": 48, "s": 128, "inplace": True},
        # prompts arriving beside decoders
        {"name": "gdn_prompts", "kind": "gdn", "reqs": 24, "new": 1, "prompts": 3, "chunk": 1500,
         "h_k": 16, "h_v": 48, "s": 128, "inplace": False},
        # the conv of the batch of decoders
        {"name": "conv_decode", "kind": "conv", "reqs": 64, "new": 1, "prompts": 0, "chunk": 0,
         "ch": 10240, "l2": 4096, "head": 128, "taps": 4, "pad": 0, "inplace": False},
        # and of the prompts
        {"name": "conv_prompts", "kind": "conv", "reqs": 24, "new": 1, "prompts": 3, "chunk": 1500,
         "ch": 10240, "l2": 4096, "head": 128, "taps": 4, "pad": 0, "inplace": False},
        # eight beams of one prompt, a few words in
        {"name": "attn_beams", "kind": "attn", "groups": 1, "per": 8, "prefix": 4096, "tail": 100,
         "new": 1, "page": 16, "f16": True, "q_heads": 24, "heads": 4, "hd": 256,
         "by_head": False},
        # many users of one system prompt
        {"name": "attn_system", "kind": "attn", "groups": 1, "per": 64, "prefix": 8192,
         "tail": 2000, "new": 1, "page": 16, "f16": True, "q_heads": 24, "heads": 4, "hd": 256,
         "by_head": False},
        # beams of several prompts over the f32 cache, other heads
        {"name": "attn_groups_f32", "kind": "attn", "groups": 5, "per": 6, "prefix": 3000,
         "tail": 150, "new": 1, "page": 48, "f16": False, "q_heads": 32, "heads": 8, "hd": 128,
         "by_head": True},
        # the beams of one prompt, their ends of text apart from their continuations
        {"name": "select_one", "kind": "select", "groups": 1, "width": 4, "vocab": 248320,
         "best": 8, "temp": 1.0, "pad": 0, "fresh": False},
        # beams of many prompts
        {"name": "select_many", "kind": "select", "groups": 32, "width": 8, "vocab": 248320,
         "best": 16, "temp": 1.0, "pad": 0, "fresh": False},
        # one prompt's beams, a few words in
        {"name": "reorder_one", "kind": "reorder", "groups": 1, "width": 4, "prefix": 4096,
         "tail": 60, "page": 16, "f16": True, "heads": 4, "hd": 256, "by_head": False},
        # many prompts' beams
        {"name": "reorder_many", "kind": "reorder", "groups": 16, "width": 8, "prefix": 2000,
         "tail": 300, "page": 16, "f16": True, "heads": 4, "hd": 256, "by_head": False},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_step(rng, most_reqs):
    """Requests of a step of a recurrent layer: decoders, drafts or prompts among them."""
    form = rng.choice(["decode", "decode", "draft", "prompts"])
    case = {"reqs": _log_int(rng, 1, most_reqs), "new": 1, "prompts": 0, "chunk": 0,
            "inplace": rng.random() < 0.5}
    if form == "draft":
        case["reqs"], case["new"] = _log_int(rng, 1, most_reqs // 2), rng.randint(2, 9)
    elif form == "prompts":
        case["reqs"], case["prompts"] = rng.randint(1, 24), rng.randint(1, 3)
        case["reqs"] = max(case["reqs"], case["prompts"])
        case["chunk"] = _log_int(rng, 17, 1500)
    return case


def draw(rng):
    kind = rng.choice(["gdn", "gdn", "conv", "attn", "attn", "select", "reorder"])
    if kind == "gdn":
        h_k, h_v, s = rng.choice([(16, 48, 128), (16, 48, 128), (4, 12, 128), (8, 16, 64)])
        return {"kind": kind, **_draw_step(rng, 64), "h_k": h_k, "h_v": h_v, "s": s}
    if kind == "conv":
        ch, l2, head, taps = rng.choice([(10240, 4096, 128, 4), (10240, 4096, 128, 4),
                                         (1280, 512, 64, 4), (2050, 0, 0, 3)])
        return {"kind": kind, **_draw_step(rng, 64), "ch": ch, "l2": l2, "head": head,
                "taps": taps, "pad": rng.choice([0, 0, rng.randint(1, 99)])}
    if kind == "select":
        width = rng.randint(1, 16)
        return {"kind": kind, "width": width,
                "groups": _log_int(rng, 1, max(1, 256 // width)),
                "vocab": rng.choice([248320, _log_int(rng, 1000, 248320)]),
                "best": rng.choice([width, min(32, 2 * width), rng.randint(1, 32)]),
                "temp": rng.choice([1.0, 0.7, round(rng.uniform(0.3, 1.5), 3)]),
                "pad": rng.choice([0, 0, rng.randint(1, 99)]), "fresh": rng.random() < 0.25}
    if kind == "reorder":
        heads, hd = rng.choice([(4, 256), (8, 128), (2, 64), (3, 80)])
        width = rng.randint(1, 16)
        return {"kind": kind, "width": width, "groups": _log_int(rng, 1, max(1, 128 // width)),
                "prefix": _log_int(rng, 1, 4096), "tail": _log_int(rng, 1, 300),
                "page": rng.choice([16, 16, 32, 64, 24]), "f16": rng.random() < 0.65,
                "heads": heads, "hd": hd, "by_head": rng.random() < 0.3}
    q_heads, heads, hd = rng.choice([(24, 4, 256), (24, 4, 256), (32, 8, 128), (16, 2, 64),
                                     (9, 3, 128), (8, 8, 64)])
    form = rng.choice(["beams", "beams", "system", "draft"])
    case = {"kind": kind, "page": rng.choice([16, 16, 32, 64, 48]), "f16": rng.random() < 0.65,
            "q_heads": q_heads, "heads": heads, "hd": hd, "by_head": rng.random() < 0.3, "new": 1}
    if form == "beams":
        case["per"] = rng.randint(2, 16)
        case["groups"] = _log_int(rng, 1, max(1, 64 // case["per"]))
        case["prefix"], case["tail"] = _log_int(rng, 64, 8192), _log_int(rng, 1, 500)
    else:
        case["groups"], case["per"] = 1, _log_int(rng, 4, 64)
        case["prefix"], case["tail"] = _log_int(rng, 64, 8192), _log_int(rng, 16, 2000)
        if form == "draft":
            case["per"], case["new"] = _log_int(rng, 2, 16), rng.randint(2, 8)
    if not case["f16"]:
        case["prefix"] = max(32, case["prefix"] // 2)
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _host(seed):
    return torch.Generator().manual_seed(seed)


def _new_tokens(case, seed):
    """New tokens of each request of a recurrent layer's step."""
    g = _host(seed)
    new = torch.randint(1, case["new"] + 1, (case["reqs"],), generator=g)
    if case["prompts"]:
        at = torch.randperm(case["reqs"], generator=g)[:case["prompts"]]
        new[at] = torch.randint(case["chunk"] // 2 + 1, case["chunk"] + 1, (case["prompts"],),
                                generator=g)
    return new.tolist()


def _slots(case, seed):
    """(slots in the pool, slot read, slot written): a quarter of the prompts are new."""
    g = _host(seed + 3)
    reqs = case["reqs"]
    order = torch.randperm(2 * reqs + 1, generator=g)
    src, dst = order[:reqs].clone(), order[reqs:2 * reqs].clone()
    if case["inplace"]:
        dst = src.clone()
    if case["prompts"]:
        src[torch.rand(reqs, generator=g) < 0.25] = -1
    return 2 * reqs + 1, src.int(), dst.int()


def prepare(case, seed):
    s = {"case": case}
    {"gdn": _prepare_gdn, "conv": _prepare_conv, "attn": _prepare_attn,
     "select": _prepare_select, "reorder": _prepare_reorder}[case["kind"]](s, case, seed)
    if own:  # the argument blocks that a program with fixed buffers keeps
        s["args"] = _arguments(s, case)
    return s


def _prepare_step(s, case, seed):
    new = _new_tokens(case, seed)
    n_tok = case["reqs"] * case["new"] + case["prompts"] * case["chunk"]  # the last: padding
    start = torch.zeros(case["reqs"] + 1, dtype=torch.int32)
    start[1:] = torch.tensor(new).cumsum(0)
    n_slots, src, dst = _slots(case, seed)
    s.update(new=new, q_start=start.cuda(), src=src.cuda(), dst=dst.cuda())
    return n_tok, n_slots


def _prepare_gdn(s, case, seed):
    n_tok, n_slots = _prepare_step(s, case, seed)
    h_k, h_v, n = case["h_k"], case["h_v"], case["s"]
    g = _gen(seed)
    # q, k and v lie side by side in a token's row, as the conv leaves them
    rows = torch.randn((n_tok, (2 * h_k + h_v) * n), generator=g, device="cuda")
    q = rows[:, :h_k * n].view(n_tok, h_k, n)
    k = rows[:, h_k * n:2 * h_k * n].view(n_tok, h_k, n)
    v = rows[:, 2 * h_k * n:].view(n_tok, h_v, n)
    for x in (q, k):
        x.div_(x.square().sum(-1, keepdim=True).sqrt())
    u = torch.rand((n_tok, h_v), generator=g, device="cuda")
    gate = -torch.exp(u * 7.0 - 6.5)  # decays from 0.998 to 0.2 a token
    beta = torch.sigmoid(torch.randn((n_tok, h_v), generator=g, device="cuda"))
    state = torch.randn((n_slots, h_v, n, n), generator=g, device="cuda").mul_(0.2)
    s.update(q=q, k=k, v=v, gate=gate, beta=beta, state=state,
             attn=torch.zeros((n_tok, h_v, n), device="cuda"))


def _prepare_conv(s, case, seed):
    n_tok, n_slots = _prepare_step(s, case, seed)
    ch, taps = case["ch"], case["taps"]
    g = _gen(seed)
    x = torch.randn((n_tok, ch + case["pad"]), generator=g, device="cuda")[:, :ch]
    w = torch.randn((ch, taps), generator=g, device="cuda").mul_(0.5)
    state = torch.randn((n_slots, ch, taps - 1), generator=g, device="cuda")
    s.update(x=x, w=w, state=state, out=torch.zeros((n_tok, ch), device="cuda"))


def _pool(case, n_pages, seed):
    """K and V [page][position][head][dim] in the case's layout and type."""
    dt = torch.float16 if case["f16"] else torch.float32
    page, heads, hd = case["page"], case["heads"], case["hd"]
    shape = (n_pages, heads, page, hd) if case["by_head"] else (n_pages, page, heads, hd)
    g = _gen(seed)
    k, v = (torch.randn(shape, generator=g, device="cuda", dtype=dt) for _ in range(2))
    if case["by_head"]:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return k, v


def _attn_lengths(case, seed):
    """Shared positions of each group, own positions and new tokens of each request."""
    g = _host(seed)
    reqs = case["groups"] * case["per"]
    u = torch.rand(case["groups"], generator=g, dtype=torch.float64)
    shared = (case["prefix"] * (1.0 - 0.25 * u)).long().clamp(min=1)
    if case["groups"] == 1:
        shared[0] = case["prefix"] - int(u[0] * case["prefix"] / 50)
    shared -= shared % case["page"]  # whole pages are shared
    new = torch.randint(1, case["new"] + 1, (reqs,), generator=g)
    tail = 1 + (case["tail"] * torch.rand(reqs, generator=g, dtype=torch.float64) ** 2).long()
    return shared.tolist(), torch.maximum(tail, new).tolist(), new.tolist()


def _tables(case, shared, tail, seed):
    """(table, pages in the pool): a group's rows begin with the same pages."""
    page, per = case["page"], len(tail) // len(shared)
    first = [n // page for n in shared]
    rest = [-(-n // page) for n in tail]
    most = case["prefix"] // page, (case["tail"] + 8) // page + 1  # whatever the lengths
    width = sum(most)
    n_pages = len(shared) * most[0] + len(tail) * most[1] + 3
    order = torch.randperm(n_pages, generator=_host(seed + 2)).int()
    table = torch.full((len(tail), width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(first):
        table[i * per:(i + 1) * per, :n] = order[at:at + n]
        at += n
    for r, n in enumerate(rest):
        table[r, first[r // per]:first[r // per] + n] = order[at:at + n]
        at += n
    return table, n_pages


def _prepare_attn(s, case, seed):
    shared, tail, new = _attn_lengths(case, seed)
    per, reqs = case["per"], len(tail)
    table, n_pages = _tables(case, shared, tail, seed)
    k_cache, v_cache = _pool(case, n_pages, seed)
    total = [shared[r // per] + n for r, n in enumerate(tail)]
    n_tok = reqs * case["new"]
    start = torch.zeros(reqs + 1, dtype=torch.int32)
    start[1:] = torch.tensor(new).cumsum(0)
    q = torch.randn((n_tok, case["q_heads"], case["hd"]), generator=_gen(seed + 1), device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    s.update(q=q, out=torch.zeros_like(q), k_cache=k_cache, v_cache=v_cache, table=table.cuda(),
             q_start=start.cuda(), kv_len=torch.tensor(total, **i32),
             group=torch.tensor([r // per for r in range(reqs)], **i32),
             group_start=torch.arange(0, reqs + 1, per, **i32),
             shared=torch.tensor(shared, **i32), max_new=max(new), longest=max(total),
             max_group=max(sum(new[i:i + per]) for i in range(0, reqs, per)))


def _prepare_select(s, case, seed):
    rows, vocab, width = case["groups"] * case["width"], case["vocab"], case["width"]
    g = _gen(seed)
    wide = torch.randn((rows, vocab + case["pad"]), generator=g, device="cuda")
    # logits of a language model: a wide bulk of coarse values, a few tokens far above it
    wide.mul_(2.5).mul_(64.0).round_().div_(64.0)
    at = torch.randint(0, vocab, (rows, 12), generator=g, device="cuda")
    wide.scatter_(1, at, 8.0 + 6.0 * torch.rand((rows, 12), generator=g, device="cuda"))
    # some tokens banned
    wide[:, torch.randint(0, vocab, (vocab // 50,), generator=g, device="cuda")] = -math.inf
    score = -20.0 * torch.rand((rows,), generator=g, device="cuda") - 5.0
    if case["fresh"]:  # the first step: one beam a group
        score.view(-1, width)[:, 1:] = -math.inf
    shape = (case["groups"], case["best"])
    s.update(x=wide[:, :vocab], score=score,
             inv_temp=float(torch.tensor(1.0 / case["temp"], dtype=torch.float32)),
             parent=torch.zeros(shape, dtype=torch.int32, device="cuda"),
             token=torch.zeros(shape, dtype=torch.int32, device="cuda"),
             score_out=torch.zeros(shape, device="cuda"))


def _reorder_lengths(case, seed):
    g = _host(seed)
    groups, width, page = case["groups"], case["width"], case["page"]
    u = torch.rand(groups, generator=g, dtype=torch.float64)
    shared = (case["prefix"] * (1.0 - 0.5 * u)).long()
    shared -= shared % page
    tail = 1 + (case["tail"] * (1.0 - 0.3 * torch.rand(groups, generator=g))).long()
    # the better beams have more children
    parent = (width * torch.rand((groups, width), generator=g) ** 1.7).int()
    return shared.tolist(), tail.tolist(), parent


def _prepare_reorder(s, case, seed):
    shared, tail, parent = _reorder_lengths(case, seed)
    groups, width = case["groups"], case["width"]
    rows = groups * width
    table, n_pages = _tables(case, shared, [tail[r // width] for r in range(rows)], seed)
    k_cache, v_cache = _pool(case, n_pages, seed)
    i32 = dict(dtype=torch.int32, device="cuda")
    parent = parent + (torch.arange(groups, dtype=torch.int32) * width)[:, None]
    order = torch.randperm(2 * rows, generator=_host(seed + 4)).int().cuda()
    begin = torch.tensor(shared, **i32).repeat_interleave(width)
    s.update(k_cache=k_cache, v_cache=v_cache, table=table.cuda(), parent=parent.cuda(),
             copy_from=torch.zeros(rows, **i32), src=torch.zeros(rows, **i32),
             dst=order[:rows].clone(), spare=order[rows:].clone(), begin=begin,
             end=begin + torch.tensor(tail, **i32).repeat_interleave(width), longest=max(tail))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _arguments(s, case):
    bh = _bh()
    kind = case["kind"]
    if kind == "gdn":
        return bh.make_gdn_ragged_args(
            s["q"], s["k"], s["v"], s["gate"], s["beta"], s["state"], s["q_start"], s["src"],
            s["dst"], attn=s["attn"], max_new=max(s["new"]))
    if kind == "conv":
        return bh.make_conv_ragged_args(
            s["x"], s["w"], s["state"], s["q_start"], s["src"], s["dst"], out=s["out"],
            l2_dim=case["l2"], head_dim=case["head"], max_new=max(s["new"]))
    if kind == "attn":
        cache = bh.make_paged_cache(s["k_cache"], s["v_cache"])
        return bh.make_attention_shared_args(
            cache, s["q"], s["q_start"], s["kv_len"], s["table"], s["group"], s["group_start"],
            s["shared"], out=s["out"], max_new=s["max_new"], max_group_new=s["max_group"])
    if kind == "select":
        return bh.make_beam_select_args(
            s["x"], s["score"], case["width"], case["best"], inv_temp=s["inv_temp"],
            parent=s["parent"], token=s["token"], score_out=s["score_out"])
    cache = bh.make_paged_cache(s["k_cache"], s["v_cache"])
    order = bh.make_beam_reorder_args(s["parent"], s["table"], copy_from=s["copy_from"],
                                      src_slot=s["src"], dst_slot=s["dst"],
                                      spare_slot=s["spare"])
    return order, bh.make_kv_copy_args(cache, s["table"], s["copy_from"], s["begin"], s["end"])


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        bh = _bh()
        if kind == "gdn":
            bh.gdn_ragged(s["args"])
        elif kind == "conv":
            bh.conv1d_silu_ragged(s["args"])
        elif kind == "attn":
            bh.attention_shared(s["args"])
        elif kind == "select":
            bh.beam_select(s["args"])
        else:
            bh.beam_reorder(s["args"][0])
            bh.kv_copy_paged(s["args"][1])
    else:
        {"gdn": _plain_gdn, "conv": _plain_conv, "attn": _plain_attn, "select": _plain_select,
         "reorder": _plain_reorder}[kind](s, case)
    names = {"gdn": ("attn", "state"), "conv": ("out", "state"), "attn": ("out",),
             "select": ("parent", "token", "score_out"),
             "reorder": ("table", "copy_from", "src", "dst", "spare", "k_cache", "v_cache")}[kind]
    return {n: s[n] for n in names}


def _read_slots(s):
    """The requests' states from their slots; zeros where they begin."""
    src = s["src"].long()
    state = s["state"][src.clamp(min=0)]
    return state.masked_fill_((src < 0).view(-1, *[1] * (state.dim() - 1)), 0.0)


def _plain_gdn(s, case):
    new, n = s["new"], case["s"]
    # the longest first: the requests with a t-th token are the first ones
    order = sorted(range(len(new)), key=lambda r: -new[r])
    at = torch.tensor(order, device="cuda")
    m = _read_slots(s)[at]
    start = s["q_start"].long()[:-1][at]
    head = torch.arange(case["h_v"], device="cuda") % case["h_k"]
    scale = 1.0 / math.sqrt(n)
    active = len(new)
    for t in range(max(new)):  # one token of each request at a time: the recurrence
        while new[order[active - 1]] <= t:
            active -= 1
        rows, mt = start[:active] + t, m[:active]
        q = s["q"][rows][:, head][:, :, None, :]
        k = s["k"][rows][:, head][:, :, None, :]
        mt.mul_(torch.exp(s["gate"][rows])[:, :, None, None])
        delta = (s["v"][rows] - (mt * k).sum(-1)) * s["beta"][rows][:, :, None]
        mt.add_(delta[..., None] * k)
        s["attn"][rows] = (mt * q).sum(-1) * scale
    s["state"][s["dst"].long()[at]] = m


def _plain_conv(s, case):
    x, taps, ch = s["x"], case["taps"], case["ch"]
    start, old = s["q_start"].long(), _read_slots(s)  # [request][channel][taps - 1]
    live = int(sum(s["new"]))
    t = torch.arange(live, device="cuda")
    r = torch.searchsorted(start[1:], t, right=True)
    acc = torch.zeros((live, ch), device="cuda")
    for j in range(taps):
        p = t - start[r] - (taps - 1) + j  # position in the request
        cached = old[r, :, (p + taps - 1).clamp(max=taps - 2)]
        acc += s["w"][:, j] * torch.where((p >= 0)[:, None], x[(start[r] + p).clamp(min=0)], cached)
    y = acc / (1.0 + torch.exp(-acc))
    if case["l2"]:
        z = y[:, :case["l2"]].reshape(live, -1, case["head"])
        z = z / z.square().sum(-1, keepdim=True).sqrt().clamp(min=1e-6)
        y = torch.cat([z.reshape(live, -1), y[:, case["l2"]:]], 1)
    s["out"][:live] = y
    # the last inputs of each request, cached ones among them where it had few
    p = (start[1:] - start[:-1])[:, None] - (taps - 1) + torch.arange(taps - 1, device="cuda")
    rows = x[(start[:-1, None] + p).clamp(min=0)].transpose(1, 2)
    at = (p + taps - 1).clamp(max=taps - 2)[:, None, :].expand(-1, ch, -1)
    s["state"][s["dst"].long()] = torch.where((p >= 0)[:, None, :], rows, old.gather(2, at))


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
    seen = seen[:, None, :, None, :].expand(-1, -1, -1, group, -1).reshape(reqs, 1, -1, longest)
    score = score.masked_fill(~seen, -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    e = e / e.sum(-1, keepdim=True)
    o = torch.matmul(e, v.permute(0, 2, 1, 3).contiguous())
    o = o.view(reqs, heads, -1, group, hd).permute(0, 2, 1, 3, 4).reshape(reqs, -1, q_heads, hd)
    live = t[None, :] < n_new[:, None]
    s["out"][row[live]] = o[live]


def _plain_select(s, case):
    # in 64 bits: rounding must not put two beams' continuations out of order
    x = s["x"].double()
    z = (x - x.amax(-1, keepdim=True)) * s["inv_temp"]
    score = s["score"].double()[:, None] + (z - torch.log(torch.exp(z).sum(-1, keepdim=True)))
    score = score.view(case["groups"], -1)
    best, at = torch.sort(score, dim=-1, descending=True, stable=True)
    best, at = best[:, :case["best"]], at[:, :case["best"]]
    base = torch.arange(case["groups"], device="cuda")[:, None] * case["width"]
    s["parent"].copy_(torch.where(best.isinf(), -1, base + at // case["vocab"]))
    s["token"].copy_(torch.where(best.isinf(), -1, at % case["vocab"]))
    s["score_out"].copy_(best)


def _plain_reorder(s, case):
    width, page = case["width"], case["page"]
    i = torch.arange(width, device="cuda")
    base = torch.arange(case["groups"], device="cuda")[:, None] * width
    p = s["parent"].long() - base
    same = p[:, :, None] == p[:, None, :]
    first = same.int().argmax(-1)  # of the parent's children
    heir = first == i
    childless = ~(p[:, :, None] == i).any(1)
    free = torch.sort(childless.int(), dim=-1, descending=True, stable=True)[1]
    nth = (~heir).long().cumsum(-1) - 1
    row = base + torch.where(heir, p, free.gather(1, nth.clamp(min=0)))
    s["table"].copy_(s["table"][row.reshape(-1)])
    copy = torch.where(heir, -1, base + first).reshape(-1)
    s["copy_from"].copy_(copy)
    written = s["dst"].clone()
    s["src"].copy_(written[s["parent"].long().reshape(-1)])
    s["dst"].copy_(s["spare"])
    s["spare"].copy_(written)
    # the pages' positions of the beams that are copied
    at = s["begin"].long()[:, None] + torch.arange(s["longest"], device="cuda")
    r, j = torch.nonzero((at < s["end"][:, None]) & (copy >= 0)[:, None], as_tuple=True)
    at = at[r, j]
    to = s["table"][r, at // page].long()
    of = s["table"][copy[r], at // page].long()
    for cache in (s["k_cache"], s["v_cache"]):
        cache[to, at % page] = cache[of, at % page]


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    # other seeds: lengths of the same distribution
    if kind == "gdn":
        h_k, h_v, n = case["h_k"], case["h_v"], case["s"]
        tokens = sum(_new_tokens(case, 0))
        fresh = sum(1 for x in _slots(case, 0)[1].tolist() if x < 0)
        return {"bytes": 4 * h_v * n * n * (2 * case["reqs"] - fresh)
                + tokens * 4 * (2 * h_k * n + 2 * h_v * n + 2 * h_v),
                "flops": 7 * tokens * h_v * n * n}
    if kind == "conv":
        ch, taps = case["ch"], case["taps"]
        tokens = sum(_new_tokens(case, 0))
        return {"bytes": 8 * tokens * ch + 8 * case["reqs"] * ch * (taps - 1) + 4 * ch * taps,
                "flops": tokens * (ch * (2 * taps + 4) + 3 * case["l2"])}
    if kind == "attn":
        shared, tail, new = _attn_lengths(case, 0)
        e, hd = (2 if case["f16"] else 4), case["hd"]
        seen = sum(sum(range(shared[r // case["per"]] + t - n + 1,
                             shared[r // case["per"]] + t + 1))
                   for r, (t, n) in enumerate(zip(tail, new)))
        return {"bytes": 2 * e * case["heads"] * hd * (sum(shared) + sum(tail))
                + 8 * sum(new) * case["q_heads"] * hd,
                "flops": 4 * hd * case["q_heads"] * seen}
    if kind == "select":
        n = case["groups"] * case["width"] * case["vocab"]
        return {"bytes": 4 * n + 4 * case["groups"] * (case["width"] + 3 * case["best"]),
                "flops": 4 * n}
    shared, tail, parent = _reorder_lengths(case, 0)
    e, rows = (2 if case["f16"] else 4), case["groups"] * case["width"]
    copies = sum(tail[i] * (case["width"] - len(set(p))) for i, p in enumerate(parent.tolist()))
    blocks = sum(-(-(a + b) // case["page"]) for a, b in zip(shared, tail)) * case["width"]
    return {"bytes": 2 * 2 * e * case["heads"] * case["hd"] * copies + 8 * blocks + 32 * rows,
            "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    return {"gdn": _exact_gdn, "conv": _exact_conv, "attn": _exact_attn,
            "select": _exact_select, "reorder": _exact_reorder}[case["kind"]](s, case)


def _exact_gdn(s, case):
    attn, state = s["attn"].double(), s["state"].double()
    old, rep = state.clone(), -(-case["h_v"] // case["h_k"])
    start = s["q_start"].tolist()
    for r, (src, dst) in enumerate(zip(s["src"].tolist(), s["dst"].tolist())):
        m = old[src].clone() if src >= 0 else torch.zeros_like(old[0])
        for t in range(start[r], start[r + 1]):
            q = s["q"][t].double().repeat(rep, 1)[:case["h_v"], :, None]
            k = s["k"][t].double().repeat(rep, 1)[:case["h_v"], :, None]
            m = m * s["gate"][t].double().exp()[:, None, None]
            wrong = s["v"][t].double() - torch.bmm(m, k)[..., 0]
            m = m + torch.bmm((wrong * s["beta"][t].double()[:, None])[..., None],
                              k.transpose(1, 2).contiguous())
            attn[t] = torch.bmm(m, q)[..., 0] / case["s"] ** 0.5
        state[dst] = m
    return {"attn": attn, "state": state}


def _exact_conv(s, case):
    out, state = s["out"].double(), s["state"].double()
    old, taps = state.clone(), case["taps"]
    start = s["q_start"].tolist()
    for r, (src, dst) in enumerate(zip(s["src"].tolist(), s["dst"].tolist())):
        a, b = start[r], start[r + 1]
        past = old[src].t() if src >= 0 else torch.zeros_like(old[0]).t()
        line = torch.cat([past, s["x"][a:b].double()])  # oldest first
        y = (line.unfold(0, taps, 1) * s["w"].double()).sum(-1)
        y = y * torch.special.expit(y)
        if case["l2"]:
            z = y[:, :case["l2"]].unflatten(1, (-1, case["head"]))
            y[:, :case["l2"]] = (z / z.norm(dim=-1, keepdim=True).clamp(min=1e-6)).flatten(1)
        out[a:b] = y
        state[dst] = line[line.shape[0] - taps + 1:].t()
    return {"out": out, "state": state}


def _exact_attn(s, case):
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


def _exact_select(s, case):
    got = []
    for g in range(case["groups"]):
        rows = slice(g * case["width"], (g + 1) * case["width"])
        p = torch.log_softmax(s["x"][rows].double() * s["inv_temp"], -1)
        all_of = (p + s["score"][rows].double()[:, None]).flatten()
        got.append(torch.topk(all_of, case["best"])[0])
    return {"parent": None, "token": None, "score_out": torch.stack(got)}


def _exact_reorder(s, case):
    """The caches after the copies, beam by beam (the rest is whole numbers)."""
    width, page = case["width"], case["page"]
    table, parent = s["table"].tolist(), s["parent"].tolist()
    got = {n: None for n in ("table", "copy_from", "src", "dst", "spare")}
    for name in ("k_cache", "v_cache"):
        cache = s[name].double()
        for g, children in enumerate(parent):
            first = {}
            for i, p in enumerate(children):
                first.setdefault(p, i)
            left = iter([g * width + r for r in range(width) if g * width + r not in first])
            for i, p in enumerate(children):
                if first[p] == i:
                    continue
                to, of = table[next(left)], table[p]
                for b in range(s["begin"][p] // page, -(-int(s["end"][p]) // page)):
                    low = max(int(s["begin"][p]) - b * page, 0)
                    high = min(int(s["end"][p]) - b * page, page)
                    cache[to[b], low:high] = s[name][of[b], low:high].double()
        got[name] = cache
    return got
