"""The paged KV cache and what works on it, as cases that can be timed and compared: a server that decodes many requests
of unlike length out of one pool of pages calls these once per step (plan) and once per layer (append, attn).

Families ("kind"):

  plan    block tables, slot maps and positions from the requests' lengths; pages taken from and given back to a free list
  append  RoPE on q and k of a ragged batch of tokens, k and v rounded to f16 into the pages their slots name
  attn    causal grouped-query attention of every request's new tokens over its pages: single tokens, drafts, prompt chunks

With ``own`` false ``run`` computes them in elementary torch operations; with ``own`` true through
``fast_llm_b200.paged``. Lengths follow from the case alone, tables and values from the seed.
"""
import math

import torch

own = False

FREQ_BASE = 500000.0


def listed():
    return [
        # One decode step of a small server: every request gets one token. Latency.
        dict(name="plan_decode_16", kind="plan", n_seq=16, past=4096, new=1, page=16, mix="decode"),
        # A busy server's step: decodes, prompts of up to 500 tokens, rewound drafts, requests that end.
        dict(name="plan_mixed_500", kind="plan", n_seq=500, past=3000, new=500, page=16, mix="mixed"),
        # The 8B shape, one token for each of 16 requests. Latency.
        dict(name="append_decode_16", kind="append", n_tok=16, n_q=32, n_kv=8, dim=128, page=16, act="f32"),
        # A large prompt chunk at the 8B shape.
        dict(name="append_chunk_8k", kind="append", n_tok=8192, n_q=32, n_kv=8, dim=128, page=64, act="f32"),
        # An odd number of tokens, small heads, f16 activations.
        dict(name="append_1001_f16", kind="append", n_tok=1001, n_q=28, n_kv=4, dim=64, page=32, act="f16"),
        # One request, one token, a short context. Latency.
        dict(name="attn_decode_1", kind="attn", n_seq=1, past=1023, new=1, n_q=32, n_kv=8, dim=128, page=16, act="f32", mix="decode"),
        # 16 requests of 5500 to 8192 keys, one token each (the 8B shape).
        dict(name="attn_decode_16", kind="attn", n_seq=16, past=8191, new=1, n_q=32, n_kv=8, dim=128, page=16, act="f32", mix="decode"),
        # Long contexts, one token each.
        dict(name="attn_decode_64k", kind="attn", n_seq=4, past=65000, new=1, n_q=32, n_kv=8, dim=128, page=64, act="f32", mix="decode"),
        # Draft verification: 8 positions for each of 4 requests.
        dict(name="attn_verify_8", kind="attn", n_seq=4, past=4096, new=8, n_q=32, n_kv=8, dim=128, page=16, act="f32", mix="chunk"),
        # A prompt of 4096 tokens from its start, f32 activations as the decoder has them.
        dict(name="attn_prompt_4k", kind="attn", n_seq=1, past=0, new=4096, n_q=32, n_kv=8, dim=128, page=64, act="f32", mix="chunk"),
        # Two prompts' chunks beside six decodes, f16 activations, small heads, groups of 7.
        dict(name="attn_mixed_f16", kind="attn", n_seq=8, past=6001, new=777, n_q=28, n_kv=4, dim=64, page=32, act="f16", mix="mixed"),
        # A chunk of 2048 tokens late in a long prompt, f16 activations.
        dict(name="attn_chunk_32k_f16", kind="attn", n_seq=1, past=30000, new=2048, n_q=32, n_kv=8, dim=128, page=128, act="f16", mix="chunk"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attn", "attn", "attn"])
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "plan":
        mix = rng.choice(["decode", "mixed"])
        return dict(kind=kind, n_seq=_log(rng, 1, 1000), past=_log(rng, 16, 20000), new=1 if mix == "decode" else _log(rng, 2, 500), page=page, mix=mix)
    n_kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 4, 5, 7, 8])
    heads = dict(n_q=n_kv * group, n_kv=n_kv, dim=rng.choice([64, 128, 128]), page=page, act=rng.choice(["f32", "f32", "f16"]))
    if kind == "append":
        return dict(kind=kind, n_tok=_log(rng, 1, 4096), **heads)
    mix = rng.choice(["decode", "decode", "chunk", "mixed"])
    if mix == "decode":
        n_seq = _log(rng, 1, 64)
        return dict(kind=kind, n_seq=n_seq, past=_log(rng, 1, min(65000, 260000 // n_seq)), new=1, mix=mix, **heads)
    n_seq, new = rng.randint(1, 6), _log(rng, 2, 1500)
    return dict(kind=kind, n_seq=n_seq, past=_log(rng, 1, min(20000, 12000000 // (n_seq * new))), new=new, mix=mix, **heads)


# ---- lengths, from the case alone ------------------------------------------------------------------------------

def _lengths(case):
    """(past, new) of every request: past within a third of the largest, new within a quarter; "mixed": three of four
    requests decode one token."""
    past, new = [], []
    for s in range(case["n_seq"]):
        past.append(case["past"] - s * 37 * max(1, case["past"] // 501) % (case["past"] // 3 + 1))
        one = case["mix"] == "decode" or (case["mix"] == "mixed" and s % 4 != 1)
        new.append(1 if one else case["new"] - s * 13 % (case["new"] // 4 + 1))
    return past, new


def _plan_lengths(case):
    """(held, past, new) of every request of a step: "mixed" has new prompts, rewound drafts, ended and idle requests."""
    past, new = _lengths(case)
    held = list(past)
    if case["mix"] == "mixed":
        for s in range(case["n_seq"]):
            if s % 16 == 1:      # a prompt that begins
                held[s] = past[s] = 0
            elif s % 16 == 3:    # some of the last draft was not taken
                past[s] = max(0, held[s] - 1 - s % 40)
            elif s % 16 == 6:    # the request has ended
                past[s] = new[s] = 0
            elif s % 16 == 10:   # idle in this step
                new[s] = 0
    return held, past, new


def _pages(n, page):
    return -(-n // page)


# ---- inputs ----------------------------------------------------------------------------------------------------

_CTX = []


def _context():
    """One library context per process, as in a program that uses the library."""
    if not _CTX:
        from fast_llm_b200 import capi
        _CTX.append(capi.Context(0))
    return _CTX[0]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _act(case):
    return torch.float16 if case["act"] == "f16" else torch.float32


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(rows, n_pages, gen):
    """Block table whose row s names rows[s] pages of a shuffled pool, and the pages that are left."""
    perm = torch.randperm(n_pages, device="cuda", generator=gen).int()
    width, count = max(rows), _ints(rows).long()
    j = torch.arange(width, device="cuda")
    at = (count.cumsum(0) - count)[:, None] + j[None, :]
    table = torch.where(j[None, :] < count[:, None], perm[at.clamp(max=n_pages - 1)], -1).int().contiguous()
    return table, perm[sum(rows):]


def prepare(case, seed):
    gen, page = _gen(seed), case["page"]
    st = {"case": case}
    if case["kind"] == "plan":
        held, past, new = _plan_lengths(case)
        rows = [_pages(h, page) for h in held]
        width = max(_pages(max(h, p + n), page) for h, p, n in zip(held, past, new)) + 1
        n_pages = sum(_pages(max(h, p + n), page) for h, p, n in zip(held, past, new)) + 7
        table, left = _table(rows, n_pages, gen)
        wide = torch.full((len(rows), width), -1, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table[:, :width]
        free = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
        free[:left.numel()] = left
        st.update(held=_ints(held), past=_ints(past), new=_ints(new), table=wide, free=free, free_count=_ints([left.numel()]),
                  n_pages=n_pages, max_tokens=sum(new) + 5)
        if own:
            st.update(ctx=_context(), q_start=_ints([0] * (len(rows) + 1)), kv_len=_ints([0] * len(rows)), free_count_out=_ints([0]),
                      pos=_ints([0] * st["max_tokens"]), slot=_ints([0] * st["max_tokens"]))
        return st
    n_q, n_kv, dim, act = case["n_q"], case["n_kv"], case["dim"], _act(case)
    if case["kind"] == "append":
        n = case["n_tok"]
        n_pages = _pages(n, page) * 2 + 3
        # q, k and v are parts of the rows that one projection wrote
        qkv = torch.randn((n, (n_q + 2 * n_kv) * dim), device="cuda", generator=gen).to(act)
        slot = torch.randperm(n_pages * page, device="cuda", generator=gen)[:n].int()
        pos = torch.randint(0, 120000, (n,), device="cuda", generator=gen, dtype=torch.int32)
        k = torch.zeros((n_pages, n_kv, page, dim), dtype=torch.float16, device="cuda")
        st.update(qkv=qkv, slot=slot, pos=pos, k=k, v=torch.zeros_like(k))
        if own:
            from fast_llm_b200 import paged
            st.update(cache=paged.PagedCache(_context(), k, st["v"], n_pages, page, n_kv, dim), q_out=torch.empty((n, n_q * dim), dtype=act, device="cuda"))
        return st
    past, new = _lengths(case)
    rows = [_pages(p + n, page) for p, n in zip(past, new)]
    n_pages = sum(rows) + 5
    table, _ = _table(rows, n_pages, gen)
    k = torch.randn((n_pages, n_kv, page, dim), device="cuda", generator=gen, dtype=torch.float16)
    v = torch.randn((n_pages, n_kv, page, dim), device="cuda", generator=gen, dtype=torch.float16)
    n = sum(new)
    st.update(q=torch.randn((n, n_q * dim), device="cuda", generator=gen).to(act), k=k, v=v, table=table, n=n, max_new=max(new),
              kv_len=_ints([p + m for p, m in zip(past, new)]), q_start=_ints([sum(new[:s]) for s in range(len(new) + 1)]))
    if own:
        from fast_llm_b200 import paged
        st.update(cache=paged.PagedCache(_context(), k, v, n_pages, page, n_kv, dim), out=torch.empty((n, n_q * dim), dtype=act, device="cuda"))
    return st


# ---- one pass --------------------------------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attn": _own_attn}[case["kind"]](case, st)
    return {"plan": _plain_plan, "append": _plain_append, "attn": _plain_attn}[case["kind"]](case, st)


def _own_plan(case, st):
    from fast_llm_b200 import paged
    paged.plan(st["ctx"], st["held"], st["past"], st["new"], st["table"], st["free"], st["free_count"], st["free_count_out"],
               st["q_start"], st["kv_len"], st["pos"], st["slot"], page_size=case["page"])
    return {"table": st["table"], "free_count": st["free_count_out"], "free": st["free"], "q_start": st["q_start"],
            "kv_len": st["kv_len"], "pos": st["pos"], "slot": st["slot"]}


def _own_append(case, st):
    nq, nk = case["n_q"] * case["dim"], case["n_kv"] * case["dim"]
    qkv = st["qkv"]
    st["cache"].append(qkv[:, :nq], qkv[:, nq:nq + nk], qkv[:, nq + nk:], st["pos"], st["slot"], st["q_out"], freq_base=FREQ_BASE)
    return {"q": st["q_out"], "k": st["k"], "v": st["v"]}


def _own_attn(case, st):
    st["cache"].attn(st["q"], st["table"], st["q_start"], st["kv_len"], st["max_new"], 1.0 / math.sqrt(case["dim"]), st["out"])
    return st["out"]


def _plain_plan(case, st):
    page, held, past, new = case["page"], st["held"].long(), st["past"].long(), st["new"].long()
    n_tok, dev = st["max_tokens"], held.device
    have, need = (held + page - 1) // page, (past + new + page - 1) // page
    give, take = (have - need).clamp(min=0), (need - have).clamp(min=0)
    # the stack after the surplus pages went on it, in order of (request, block)
    j = torch.arange(st["table"].shape[1], device=dev)[None, :]
    given = (j >= need[:, None]) & (j < have[:, None])
    count = st["free_count"].long()
    at = torch.arange(st["n_pages"], device=dev)
    order = torch.where(given, (given.reshape(-1).cumsum(0) - 1 + count).view(given.shape), st["n_pages"])   # the cell behind the stack: not given
    stack = torch.cat([st["free"], st["free"].new_zeros(1)])
    stack[order.reshape(-1)] = st["table"].reshape(-1)
    stack = stack[:-1]
    top = count + give.sum()
    # demands from its top, in the same order
    taken = (j >= have[:, None]) & (j < need[:, None])
    source = (top - 1 - ((take.cumsum(0) - take)[:, None] + j - have[:, None])).clamp(0, st["n_pages"] - 1)
    table = torch.where(taken, stack[source], st["table"])
    left = top - take.sum()
    free = torch.where((at >= count) & (at < left), stack, st["free"])
    q_end = new.cumsum(0)
    q_start = torch.cat([q_end.new_zeros(1), q_end])
    i = torch.arange(n_tok, device=dev)
    s = torch.searchsorted(q_end, i, right=True).clamp(max=held.numel() - 1)
    live = i < q_end[-1]
    pos = torch.where(live, past[s] + i - q_start[s], -1)
    slot = torch.where(live, table[s, pos.clamp(min=0) // page] * page + pos % page, -1)
    return {"table": table.int(), "free_count": left.int(), "free": free.int(), "q_start": q_start.int(), "kv_len": (past + new).int(),
            "pos": pos.int(), "slot": slot.int()}


def _plain_append(case, st):
    n_q, n_kv, dim, act, page = case["n_q"], case["n_kv"], case["dim"], _act(case), case["page"]
    x = st["qkv"].float().view(-1, n_q + 2 * n_kv, dim)
    freq = FREQ_BASE ** (-2.0 * torch.arange(dim // 2, device=x.device, dtype=torch.float64) / dim)
    angle = st["pos"].double()[:, None] * freq[None, :]
    c, s = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    a, b = x[:, :n_q + n_kv, 0::2], x[:, :n_q + n_kv, 1::2]
    turned = torch.stack([a * c - b * s, a * s + b * c], dim=-1).reshape(x.shape[0], n_q + n_kv, dim)
    at, row = (st["slot"] // page).long(), (st["slot"] % page).long()
    st["k"][at, :, row] = turned[:, n_q:].half()
    st["v"][at, :, row] = x[:, n_q + n_kv:].half()
    return {"q": turned[:, :n_q].reshape(-1, n_q * dim).to(act), "k": st["k"], "v": st["v"]}


def _plain_attn(case, st):
    n_q, n_kv, dim, page = case["n_q"], case["n_kv"], case["dim"], case["page"]
    group, n_seq, n, max_new = n_q // n_kv, case["n_seq"], st["n"], st["max_new"]
    start, length = st["q_start"][:-1].long(), st["kv_len"].long()
    new = st["q_start"][1:].long() - start
    i = torch.arange(max_new, device=start.device)
    at = (start[:, None] + i[None, :]).clamp(max=n - 1)
    # requests padded to the longest: q [request][KV head][token, head of its group][dim], K and V [request][KV head][key][dim]
    q = st["q"].float().view(n, n_kv, group, dim)[at].permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, max_new * group, dim)
    pages = st["table"].clamp(min=0).long()
    keys = torch.arange(pages.shape[1] * page, device=start.device)
    there = (keys[None, :] < length[:, None])[:, None, :, None]
    k = st["k"][pages].permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, -1, dim).float()
    v = torch.where(there, st["v"][pages].permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, -1, dim).float(), 0.0)
    score = (q @ k.transpose(2, 3)).view(n_seq, n_kv, max_new, group, -1).mul_(1.0 / math.sqrt(dim))
    seen = keys[None, None, :] <= (length - new)[:, None, None] + i[None, :, None]
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1).reshape(n_seq, n_kv, max_new * group, 1)
    o = p.view(n_seq, n_kv, max_new * group, -1) @ v
    o = torch.where(total == 0, 0.0, o / total).view(n_seq, n_kv, max_new, group, dim).permute(0, 2, 1, 3, 4).reshape(n_seq, max_new, n_q * dim)
    return o[i[None, :] < new[:, None]].to(_act(case))


# ---- the definition, in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "plan":
        return None   # whole numbers
    st = prepare(case, seed)
    n_q, n_kv, dim, page = case["n_q"], case["n_kv"], case["dim"], case["page"]
    if case["kind"] == "append":
        x = st["qkv"].double().view(-1, n_q + 2 * n_kv, dim)
        pairs = torch.view_as_complex(x.view(*x.shape[:2], dim // 2, 2).contiguous())
        theta = torch.pow(torch.full((dim // 2,), FREQ_BASE, dtype=torch.float64, device=x.device), -torch.arange(0, dim, 2, device=x.device).double() / dim)
        pairs = torch.view_as_real(pairs * torch.polar(torch.ones_like(theta), st["pos"].double()[:, None] * theta)[:, None, :]).flatten(2)
        k, v = (torch.zeros((st["k"].shape[0] * page, n_kv, dim), dtype=torch.float64, device=x.device) for _ in range(2))
        k[st["slot"].long()], v[st["slot"].long()] = pairs[:, n_q:n_q + n_kv], x[:, n_q + n_kv:]
        k, v = (t.view(-1, page, n_kv, dim).transpose(1, 2) for t in (k, v))
        return {"q": pairs[:, :n_q].reshape(-1, n_q * dim), "k": k, "v": v}
    out = torch.zeros((st["n"], n_q, dim), dtype=torch.float64, device="cuda")
    past, new = _lengths(case)
    first = 0
    for s, (p, m) in enumerate(zip(past, new)):
        rows = st["table"][s, :_pages(p + m, page)].long()
        for h in range(n_q):
            k = st["k"][rows, h * n_kv // n_q].reshape(-1, dim)[:p + m].double()
            v = st["v"][rows, h * n_kv // n_q].reshape(-1, dim)[:p + m].double()
            a = st["q"][first:first + m].view(m, n_q, dim)[:, h].double() @ k.t() / math.sqrt(dim)
            a += torch.full((m, p + m), -math.inf, dtype=torch.float64, device="cuda").triu(p + 1)
            out[first:first + m, h] = a.softmax(-1) @ v
        first += m
    return out.view(st["n"], n_q * dim)


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    page = case["page"]
    if case["kind"] == "plan":
        held, past, new = _plan_lengths(case)
        moved = sum(abs(_pages(p + n, page) - _pages(h, page)) for h, p, n in zip(held, past, new))
        # lengths, first tokens, pages moved (read and written), the tail page of each request, positions and slots
        return {"bytes": 4.0 * (6 * len(held) + 2 * moved + 2 * (sum(new) + 5)), "flops": float(sum(new) + 8 * len(held))}
    n_q, n_kv, dim, size = case["n_q"], case["n_kv"], case["dim"], 2 if case["act"] == "f16" else 4
    if case["kind"] == "append":
        n = case["n_tok"]
        return {"bytes": float(n * ((2 * n_q + 2 * n_kv) * dim * size + 2 * n_kv * dim * 2 + 8)), "flops": 3.0 * n * (n_q + n_kv) * dim}
    past, new = _lengths(case)
    pairs = sum(m * p + m * (m + 1) // 2 for p, m in zip(past, new))
    kv = sum(p + m for p, m in zip(past, new)) * n_kv * dim * 2 * 2
    return {"bytes": float(kv + 2 * sum(new) * n_q * dim * size + 4 * sum(_pages(p + m, page) for p, m in zip(past, new))),
            "flops": 4.0 * dim * n_q * pairs}
