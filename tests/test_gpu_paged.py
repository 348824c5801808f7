"""GPU tests of the paged KV cache (fl_b200_paged_plan / _append / _attn) against plain implementations in 64 bits.

Tolerances. Attention: an output is sum_j p_j v_j / sum_j p_j. With A the largest scale * sum_d |q_d k_jd| of a row, a score is off by
at most 2^-22 A (q as two f16 parts: half a step of 2^-11 twice) + 8 * 2^-23 A (a chain of eight tensor instructions that
truncate) + 2^-23 A (parts added, exponent rounded), below 2^-19 A; numerator and denominator: twice that. The probabilities: 2^-22 (ex2), 2^-22
(two parts) and the sums' roundings, below 2^-18. So (A + 1) 2^-18 sum_j p_j |v_j| / sum_j p_j. f16 activations: one part of p, 2^-11 more of
that sum, and half a step of the result."""
import math

import numpy as np
import pytest

from fast_llm_b200 import capi

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16}
CANARY = 7.25


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make(seed, seqs, n_q, n_kv, dim, page, act, spare=3, kv_scale=1.0):
    """seqs: (kv_len, new) per sequence. Rows of the pools that hold no key are NaN, table entries behind the last page garbage."""
    from fast_llm_b200 import paged   # noqa: F401  (needs torch)
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-L // page) for L, _ in seqs]
    n_pages, width = sum(need) + spare, max(max(need), 1) + 2
    perm = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.full((len(seqs), width), 1 << 30, dtype=torch.int32, device="cuda")
    table[:, -1] = -5
    k = torch.full((n_pages, n_kv, page, dim), float("nan"), device="cuda", dtype=torch.float16)
    v = k.clone()
    at, ks, vs = 0, [], []
    for s, (L, _) in enumerate(seqs):
        pg = perm[at:at + need[s]]
        at += need[s]
        table[s, :need[s]] = pg
        kk = (kv_scale * torch.randn((n_kv, need[s] * page, dim), generator=g, device="cuda")).half()
        vv = torch.randn((n_kv, need[s] * page, dim), generator=g, device="cuda").half()
        kk[:, L:] = float("nan")
        vv[:, L:] = float("nan")
        if need[s]:
            k[pg.long()] = kk.view(n_kv, need[s], page, dim).transpose(0, 1)
            v[pg.long()] = vv.view(n_kv, need[s], page, dim).transpose(0, 1)
        ks.append(kk[:, :L])
        vs.append(vv[:, :L])
    n = sum(m for _, m in seqs)
    rows = n + 2   # two rows behind the last sequence
    wide = torch.randn((rows, n_q * dim + 16), generator=g, device="cuda").to(DT[act])
    out = torch.full((rows, n_q * dim + 8), CANARY, device="cuda", dtype=DT[act])
    lse = torch.full((rows, n_q, 2), CANARY, device="cuda")
    start = np.concatenate([[0], np.cumsum([m for _, m in seqs])]).tolist()
    return dict(k=k, v=v, table=table, q=wide[:, 8:8 + n_q * dim], out=out[:, :n_q * dim], out_all=out, lse=lse, q_start=ints(start),
                kv_len=ints([L for L, _ in seqs]), ks=ks, vs=vs, n=n, n_pages=n_pages, max_new=max(m for _, m in seqs), start=start)


def expect(c, seqs, n_q, n_kv, dim, scale, act):
    """(want, bound, lse) in 64 bits, for the rows of all sequences."""
    rows = c["q"].shape[0]
    want, tol = (torch.zeros((rows, n_q, dim), dtype=torch.float64, device="cuda") for _ in range(2))
    lse = torch.zeros((rows, n_q, 2), dtype=torch.float64, device="cuda")
    q = c["q"].double().view(rows, n_q, dim)
    for s, (L, m) in enumerate(seqs):
        for h in range(n_q):
            k, v = c["ks"][s][h * n_kv // n_q].double(), c["vs"][s][h * n_kv // n_q].double()
            for i0 in range(0, m, 512):
                i1 = min(m, i0 + 512)
                a = slice(c["start"][s] + i0, c["start"][s] + i1)
                x = q[a, h] @ k.t() * scale
                size = (q[a, h].abs() @ k.t().abs() * scale)
                lim = L - m + torch.arange(i0, i1, device="cuda")
                seen = torch.arange(L, device="cuda")[None, :] <= lim[:, None]
                x = torch.where(seen, x, -math.inf)
                A = torch.where(seen, size, 0.0).amax(-1, keepdim=True) if L else torch.zeros((i1 - i0, 1), device="cuda", dtype=torch.float64)
                top = x.amax(-1, keepdim=True) if L else torch.full((i1 - i0, 1), -math.inf, device="cuda", dtype=torch.float64)
                p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
                p = torch.where(seen, p, 0.0)
                den = p.sum(-1, keepdim=True)
                div = torch.where(den == 0, 1.0, den)
                want[a, h] = p @ v / div
                spread = p @ v.abs() / div
                tol[a, h] = (A + 1) * 2.0 ** -18 * spread
                if act == "f16":
                    tol[a, h] += 2.0 ** -11 * spread + 2.0 ** -11 * want[a, h].abs() + 2.0 ** -25
                lse[a, h, 0], lse[a, h, 1] = top[:, 0], den[:, 0]
    return want, tol, lse


def attn(ctx, c, n_q, n_kv, dim, page, scale, lse=True, max_new=None):
    from fast_llm_b200 import paged
    cache = paged.PagedCache(ctx, c["k"], c["v"], c["n_pages"], page, n_kv, dim)
    torch.cuda.synchronize()
    cache.attn(c["q"], c["table"], c["q_start"], c["kv_len"], max_new or c["max_new"], scale, c["out"], c["lse"] if lse else None)
    ctx.sync()


def check(ctx, c, seqs, n_q, n_kv, dim, scale, act, what=""):
    want, tol, lse = expect(c, seqs, n_q, n_kv, dim, scale, act)
    got, n = c["out"].double().view(-1, n_q, dim), c["n"]
    assert ctx.status() == 0
    off = (got[:n] - want[:n]).abs()
    assert torch.isfinite(got[:n]).all(), what
    worst = (off / (tol[:n] + 1e-300)).max().item() if n else 0.0
    assert (off <= tol[:n]).all(), (what, worst)
    assert (c["out"][n:] == CANARY).all() and (c["out_all"][:, n_q * dim:] == CANARY).all(), "wrote outside its rows"
    m, s = c["lse"][:n, :, 0].double(), c["lse"][:n, :, 1].double()
    none = lse[:n, :, 0] == -math.inf
    assert (m[none] == -math.inf).all() and (s[none] == 0).all()
    total = m + torch.log(s)
    ref = lse[:n, :, 0] + torch.log(lse[:n, :, 1])
    # log of the sum: off by the scores' 2^-19 A and the sum's 2^-18
    A = 2.0 ** 19 * 2.0 ** -18 * 40
    assert ((total - ref)[~none].abs() <= A * 2.0 ** -19 + 2.0 ** -20 * ref[~none].abs()).all()
    assert (c["lse"][n:] == CANARY).all()


SEQS = {
    "one": [(1, 1)],
    "edges": [(5, 1), (63, 1), (64, 1), (65, 1), (128, 1), (129, 1), (1, 1)],
    "idle": [(100, 0), (17, 1), (0, 0), (40, 2), (33, 0)],
    "no_key": [(0, 1), (2, 5), (70, 3)],
    "draft": [(300, 4), (77, 3), (4, 4)],
    "rows": [(37, 17), (200, 5), (1000, 40)],
    "chunk": [(130, 130), (257, 129), (64, 64)],
    "long": [(20011, 1), (3, 1)],
    "longer_chunk": [(5003, 300)],
    "mixed": [(900, 1), (515, 260), (4097, 1), (1, 1), (700, 64), (31, 31)],
}


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("n_q,n_kv,dim,page", [(32, 8, 128, 16), (4, 1, 64, 32), (10, 2, 128, 64), (7, 1, 128, 128), (14, 2, 64, 256), (16, 16, 64, 16), (34, 1, 64, 64)])
@pytest.mark.parametrize("name", list(SEQS))
def test_attention_against_64_bits(ctx, name, n_q, n_kv, dim, page, act):
    seqs = SEQS[name]
    c = make(len(name) + n_q + dim + page, seqs, n_q, n_kv, dim, page, act)
    attn(ctx, c, n_q, n_kv, dim, page, 1.0 / math.sqrt(dim))
    check(ctx, c, seqs, n_q, n_kv, dim, 1.0 / math.sqrt(dim), act, name)


def test_attention_of_many_sequences(ctx):
    rng = np.random.default_rng(3)
    seqs = [(int(L), int(min(L, m))) for L, m in zip(rng.integers(1, 400, 700), rng.choice([1, 1, 1, 2, 30], 700))]
    c = make(5, seqs, 8, 2, 128, 16, "f32")
    attn(ctx, c, 8, 2, 128, 16, 0.1)
    check(ctx, c, seqs, 8, 2, 128, 0.1, "f32")


@pytest.mark.parametrize("q_size,k_size", [(1e-6, 1.0), (3e4, 1e-3), (1e30, 1e-4), (8.0, 4.0)])
def test_attention_scales(ctx, q_size, k_size):
    """Rows of q far from 1: they are brought to the middle of the f16 range by a power of two."""
    seqs = [(200, 3), (130, 70)]
    c = make(9, seqs, 8, 2, 128, 16, "f32", kv_scale=k_size)
    c["q"].mul_(q_size)
    scale = 1.0 / math.sqrt(128) if q_size < 100 else 1.0 / (q_size * k_size * math.sqrt(128))
    attn(ctx, c, 8, 2, 128, 16, scale)
    check(ctx, c, seqs, 8, 2, 128, scale, "f32")


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("seqs", [[(70, 3)], [(90, 40)], [(300, 140), (66, 2)]])
def test_masked_keys_may_hold_anything(ctx, seqs, act):
    """NaN and infinities in keys that a row does not attend leave it alone; in values that it attends they arrive."""
    n_q, n_kv, dim, page = 8, 2, 64, 16
    c = make(21, seqs, n_q, n_kv, dim, page, act)
    clean = {n: t.clone() for n, t in c.items() if torch.is_tensor(t)}
    L, m = seqs[0]
    j = L - 2   # attended by the last two tokens only
    pg, r = int(c["table"][0, j // page]), j % page
    c["k"][pg, 0, r, 5] = float("nan")
    c["v"][pg, 0, r, 3] = float("inf")
    c["v"][pg, 1, r, 7] = -float("inf")
    c["v"][pg, 1, r, 9] = float("nan")
    attn(ctx, c, n_q, n_kv, dim, page, 0.125)
    got = c["out"].clone().view(-1, n_q, dim)
    attn(ctx, dict(clean, n_pages=c["n_pages"], max_new=c["max_new"]), n_q, n_kv, dim, page, 0.125)
    ref = clean["out"].view(-1, n_q, dim)
    assert torch.equal(got[:m - 2], ref[:m - 2])          # rows in front of the key
    assert torch.equal(got[m:], ref[m:])
    for i in (m - 2, m - 1):
        assert torch.isnan(got[i, :4]).all()               # a NaN score
        assert (got[i, 4:, 7] == -math.inf).all() and torch.isnan(got[i, 4:, 9]).all()
        keep = [d for d in range(dim) if d not in (7, 9)]
        assert torch.equal(got[i, 4:][:, keep], ref[i, 4:][:, keep])
    ctx.status()


def test_attention_lengths_that_break_the_bounds(ctx):
    """Sequences whose lengths do not fit the call are left out and reported; the others are computed."""
    seqs = [(100, 2), (50, 1), (80, 3)]
    c = make(4, seqs, 8, 2, 128, 16, "f32")
    c["kv_len"][1] = c["table"].shape[1] * 16 + 1
    attn(ctx, c, 8, 2, 128, 16, 0.1)
    assert ctx.status() == 4
    assert (c["out"][2] == CANARY).all()
    c["kv_len"][1] = 50
    keep = c["out"].clone()
    attn(ctx, c, 8, 2, 128, 16, 0.1)
    assert ctx.status() == 0
    assert torch.equal(keep[:2], c["out"][:2]) and torch.equal(keep[3:], c["out"][3:])
    c["out"].fill_(CANARY)
    attn(ctx, c, 8, 2, 128, 16, 0.1, max_new=2)   # the third has more
    assert ctx.status() == 4
    assert (c["out"][3:6] == CANARY).all() and torch.equal(keep[:2], c["out"][:2])
    for bad in ([0, 2, 1, 6], [0, 2, 3, 900], [-1, 2, 3, 6]):
        attn(ctx, dict(c, q_start=ints(bad)), 8, 2, 128, 16, 0.1)
        assert ctx.status() == 4


@pytest.mark.parametrize("seqs", [[(200, 1)], [(200, 90)]])
@pytest.mark.parametrize("page", [-1, 10 ** 9, None])
def test_attention_bad_pages(ctx, seqs, page):
    """Keys on a page outside the pool count as zero vectors: nothing is read out of bounds, and it is reported."""
    c = make(6, seqs, 8, 2, 128, 16, "f32")
    c["table"][0, 3] = c["n_pages"] if page is None else page
    attn(ctx, c, 8, 2, 128, 16, 0.1)
    assert ctx.status() == 3
    for x in c["ks"] + c["vs"]:
        x[:, 48:64] = 0
    check(ctx, c, seqs, 8, 2, 128, 0.1, "f32")


def test_results_repeat(ctx):
    """Several CTAs share a block of rows: their records are added in order, whichever arrives last."""
    for seqs in ([(9000, 1), (40, 1)], [(3000, 200), (700, 9)]):
        c = make(8, seqs, 32, 8, 128, 16, "f32")
        attn(ctx, c, 32, 8, 128, 16, 0.1)
        first = c["out"].clone()
        for _ in range(5):
            attn(ctx, c, 32, 8, 128, 16, 0.1)
            assert torch.equal(first, c["out"])


# ---- append ------------------------------------------------------------------------------------------------------------------


def append_expect(x, pos, n_rot, base):
    """RoPE in 64 bits on x [tokens][heads][dim]."""
    y = x.double().clone()
    ang = pos.double()[:, None] * torch.pow(torch.tensor(base, dtype=torch.float64, device="cuda"), -torch.arange(0, n_rot, 2, device="cuda").double() / max(n_rot, 1))
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = y[..., 0:n_rot:2].clone(), y[..., 1:n_rot:2].clone()
    y[..., 0:n_rot:2], y[..., 1:n_rot:2] = a * c - b * s, a * s + b * c
    return y


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("n_q,n_kv,dim,page,n_tok,n_rot,base", [
    (32, 8, 128, 16, 1, 128, 500000.0), (32, 8, 128, 16, 16, 128, 500000.0), (4, 4, 64, 64, 777, 64, 10000.0), (7, 1, 128, 32, 5000, 128, 1000000.0),
    (6, 2, 64, 256, 33, 20, 10000.0), (6, 2, 128, 128, 33, 0, 0.0), (0, 2, 64, 16, 9, 64, 10000.0)])
def test_append(ctx, n_q, n_kv, dim, page, n_tok, n_rot, base, act):
    from fast_llm_b200 import paged
    g = torch.Generator(device="cuda").manual_seed(n_tok + dim)
    n_pages = -(-n_tok // page) + 2
    k0 = torch.randn((n_pages, n_kv, page, dim), generator=g, device="cuda").half()
    v0 = torch.randn((n_pages, n_kv, page, dim), generator=g, device="cuda").half()
    k, v = k0.clone(), v0.clone()
    rows = torch.randn((n_tok, (n_q + 2 * n_kv) * dim + 8), generator=g, device="cuda").to(DT[act])
    qs, ks, vs = rows[:, :n_q * dim], rows[:, n_q * dim:(n_q + n_kv) * dim], rows[:, (n_q + n_kv) * dim:(n_q + 2 * n_kv) * dim]
    pos = torch.randint(0, 1 << 20, (n_tok,), generator=g, device="cuda", dtype=torch.int32)
    slot = torch.randperm(n_pages * page, generator=g, device="cuda")[:n_tok].int()
    pos[0] = 0
    if n_tok > 8:
        pos[3], slot[3] = -1, -1     # a row behind the last token
        slot[5] = -1                 # rotated, not appended
    q_out = torch.full((n_tok, n_q * dim + 16), CANARY, device="cuda", dtype=DT[act]) if n_q else None
    cache = paged.PagedCache(ctx, k, v, n_pages, page, n_kv, dim)
    torch.cuda.synchronize()
    cache.append(qs if n_q else None, ks, vs, pos, slot, q_out[:, :n_q * dim] if n_q else None, freq_base=base, n_rot=n_rot)
    ctx.sync()
    assert ctx.status() == 0
    live = pos >= 0
    put = live & (slot >= 0)
    # products and sums in f32: 3 roundings of |x| <= |a| + |b|, sine and cosine off by 2^-22; then the type's half step
    def close(got, want, size, eps):
        assert ((got.double() - want).abs() <= 2.0 ** -21 * size + eps * want.abs() + 2.0 ** -25).all()
    eps = 2.0 ** -11 if act == "f16" else 0.0
    if n_q:
        x = qs.reshape(n_tok, n_q, dim)
        size = x.double().abs().view(n_tok, n_q, dim // 2, 2).sum(-1, keepdim=True).expand(-1, -1, -1, 2).reshape(n_tok, n_q, dim)
        got = q_out[:, :n_q * dim].reshape(n_tok, n_q, dim)
        close(got[live], append_expect(x, pos, n_rot, base)[live], size[live], eps)
        assert (got[~live] == CANARY).all() and (q_out[:, n_q * dim:] == CANARY).all()
    x = ks.reshape(n_tok, n_kv, dim)
    size = x.double().abs().view(n_tok, n_kv, dim // 2, 2).sum(-1, keepdim=True).expand(-1, -1, -1, 2).reshape(n_tok, n_kv, dim)
    pg, r = (slot[put] // page).long(), (slot[put] % page).long()
    close(k[pg, :, r], append_expect(x, pos, n_rot, base)[put], size[put], 2.0 ** -11)
    assert torch.equal(v[pg, :, r], vs.reshape(n_tok, n_kv, dim)[put].half())
    k[pg, :, r], v[pg, :, r] = k0[pg, :, r], v0[pg, :, r]
    assert torch.equal(k, k0) and torch.equal(v, v0)        # nothing else was written


def test_append_in_place_and_bad_slots(ctx):
    from fast_llm_b200 import paged
    k, v = torch.zeros((4, 2, 16, 64), device="cuda", dtype=torch.float16), torch.zeros((4, 2, 16, 64), device="cuda", dtype=torch.float16)
    q = torch.randn((3, 4 * 64), device="cuda")
    kk = torch.randn((3, 2 * 64), device="cuda")
    cache = paged.PagedCache(ctx, k, v, 4, 16, 2, 64)
    pos, slot = ints([5, 6, 7]), ints([3, 64, 2 ** 31 - 1])
    want = append_expect(q.view(3, 4, 64), pos, 64, 10000.0)
    torch.cuda.synchronize()
    cache.append(q, kk, kk, pos, slot, q, freq_base=10000.0)
    ctx.sync()
    assert ctx.status() == 3
    assert ((q.double().view(3, 4, 64) - want).abs() < 1e-5).all()
    assert (v[0, :, 3] == kk[0].view(2, 64).half()).all()
    v[0, :, 3] = 0
    assert (v == 0).all()


# ---- plan --------------------------------------------------------------------------------------------------------------------


def plan_expect(held, past, new, table, free, count, page, max_tok):
    """One sequence and one page at a time."""
    up = lambda n: -(-n // page)   # noqa: E731
    table, free = [list(r) for r in table], list(free)
    stack, pos, slot = list(free[:count]), [], []
    for s in range(len(held)):
        stack += table[s][up(past[s] + new[s]):up(held[s])]
    before = len(stack)
    for s in range(len(held)):
        for j in range(up(held[s]), up(past[s] + new[s])):
            table[s][j] = stack.pop()
        for p in range(past[s], past[s] + new[s]):
            pos.append(p)
            slot.append(table[s][p // page] * page + p % page)
    if len(stack) > count:
        free[count:len(stack)] = stack[count:]
    assert before >= len(stack)
    fill = [-1] * (max_tok - len(pos))
    start = np.concatenate([[0], np.cumsum(new)]).tolist()
    return dict(table=table, free=free, count=len(stack), pos=pos + fill, slot=slot + fill, start=start, length=[p + n for p, n in zip(past, new)])


def plan_state(rng, n_seq, page, kinds, longest, most_new):
    held, past, new = [], [], []
    for _ in range(n_seq):
        kind, h = rng.choice(kinds), int(rng.integers(0, longest))
        p, n = h, 1
        if kind == "prompt":
            h = p = 0
            n = int(rng.integers(1, most_new + 1))
        elif kind == "chunk":
            n = int(rng.integers(0, most_new + 1))
        elif kind == "rewind":
            p = int(rng.integers(0, h + 1))
        elif kind == "end":
            p = n = 0
        held.append(h)
        past.append(p)
        new.append(n)
    return held, past, new


def run_plan(ctx, held, past, new, table, free, count, page, max_tok, in_place=False):
    from fast_llm_b200 import paged
    t, f, n = ints(table), ints(free), len(held)
    h, cin = ints(held), ints([count])
    cout, klen = (cin, h) if in_place else (ints([-9]), ints([-9] * n))
    start, pos, slot = ints([-9] * (n + 1)), ints([-9] * max_tok), ints([-9] * max_tok)
    torch.cuda.synchronize()
    paged.plan(ctx, h, ints(past), ints(new), t, f, cin, cout, start, klen, pos, slot, page_size=page)
    ctx.sync()
    return dict(table=t.tolist(), free=f.tolist(), count=cout.item(), pos=pos.tolist(), slot=slot.tolist(), start=start.tolist(), length=klen.tolist())


@pytest.mark.parametrize("n_seq,page,kinds,longest,most_new", [
    (1, 16, ["decode"], 40, 1), (3, 16, ["prompt"], 1, 20), (16, 16, ["decode"], 300, 1), (40, 32, ["decode", "rewind", "end", "prompt", "chunk"], 500, 90),
    (700, 16, ["decode", "rewind", "end", "prompt", "chunk"], 200, 60), (513, 64, ["end", "rewind"], 900, 1), (100, 256, ["chunk", "end"], 3000, 700), (4096, 16, ["decode", "end"], 60, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(ctx, n_seq, page, kinds, longest, most_new, in_place):
    rng = np.random.default_rng(n_seq + page)
    up = lambda n: -(-n // page)   # noqa: E731
    held, past, new = plan_state(rng, n_seq, page, kinds, longest, most_new)
    width = max(up(max(h, p + n)) for h, p, n in zip(held, past, new)) + 1
    n_pages = sum(up(max(h, p + n)) for h, p, n in zip(held, past, new)) + 3
    perm, at, table = rng.permutation(n_pages).tolist(), 0, []
    for h in held:
        table.append(perm[at:at + up(h)] + [-3] * (width - up(h)))
        at += up(h)
    free = perm[at:] + [-7] * at
    max_tok = sum(new) + 5
    got = run_plan(ctx, held, past, new, table, free, n_pages - at, page, max_tok, in_place)
    assert ctx.status() == 0
    assert got == plan_expect(held, past, new, table, free, n_pages - at, page, max_tok)


def test_plan_takes_the_last_page_and_no_more(ctx):
    table, free = [[0, -1, -1], [1, 2, -1]], [5, 4, 3]
    got = run_plan(ctx, [16, 32], [16, 20], [17, 20], table, free, 2, 16, 37)    # needs 2 + 1 pages, 2 there
    assert ctx.status() == 5
    assert got == dict(table=table, free=free, count=2, pos=[-1] * 37, slot=[-1] * 37, start=[0, 0, 0], length=[-9, -9])
    got = run_plan(ctx, [16, 32], [16, 20], [17, 12], table, free, 2, 16, 29)    # needs 2, 2 there, 29 tokens
    assert ctx.status() == 0 and got["table"] == [[0, 4, 5], [1, 2, -1]] and got["count"] == 0
    got = run_plan(ctx, [16, 32], [16, 20], [17, 12], table, free, 2, 16, 28)    # a token too many
    assert ctx.status() == 5 and got["pos"] == [-1] * 28 and got["count"] == 2
    # what one sequence gives back another takes in the same step
    got = run_plan(ctx, [16, 32], [16, 0], [17, 0], table, free, 0, 16, 20)
    assert ctx.status() == 0 and got["table"] == [[0, 2, 1], [1, 2, -1]] and got["count"] == 0


@pytest.mark.parametrize("held,past,new,count", [([-1], [0], [1], 2), ([4], [5], [1], 2), ([4], [4], [-1], 2), ([40], [40], [9], 2), ([49], [1], [1], 2), ([4], [4], [1], -1),
                                                 ([4], [4], [1], 4), ([4], [4], [2 ** 31 - 1], 2)])
def test_plan_refuses_impossible_lengths(ctx, held, past, new, count):
    table, free = [[0, 1, 2]], [5, 4, 3]
    got = run_plan(ctx, held, past, new, table, free, count, 16, 3)
    assert ctx.status() == 4
    assert got == dict(table=table, free=free, count=count, pos=[-1] * 3, slot=[-1] * 3, start=[0, 0], length=[-9])
