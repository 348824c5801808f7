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


@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("wrong", [-1, 1 << 28, (1 << 31) - 1, -(1 << 31)])
def test_plan_of_pages_that_no_pool_has(ctx, page, wrong):
    """Their slots are -1, not another page's whose number is the same in 31 bits."""
    n = page + 3
    got = run_plan(ctx, [n, n], [n, n], [1, 1], [[1, wrong], [2, 0]], [3, 4], 2, page, 3)          # a page held
    assert ctx.status() == 3
    assert got["slot"] == [-1, 3, -1] and got["pos"] == [n, n, -1] and got["length"] == [n + 1, n + 1]
    got = run_plan(ctx, [page, n], [page, n], [2, 1], [[1, -9], [2, 0]], [3, wrong], 2, page, 3)   # a page taken
    assert ctx.status() == 3
    assert got["slot"] == [-1, -1, 3] and got["table"] == [[1, wrong], [2, 0]] and got["count"] == 1


# ---- together ----------------------------------------------------------------------------------------------------------------


class Server:
    """Requests that come, grow, are rewound and go, over one layer: plan, append and attention as a server calls them, beside a
    plain copy of every request's rotated keys and values."""

    def __init__(self, ctx, n_seq, blocks, n_pages, page, n_q, n_kv, dim, act, max_tokens, base=10000.0):
        from fast_llm_b200 import paged
        self.paged, self.ctx, self.page, self.n_q, self.n_kv, self.dim, self.act, self.base = paged, ctx, page, n_q, n_kv, dim, act, base
        self.k = torch.full((n_pages, n_kv, page, dim), float("nan"), device="cuda", dtype=torch.float16)
        self.v = self.k.clone()
        self.cache = paged.PagedCache(ctx, self.k, self.v, n_pages, page, n_kv, dim)
        self.table = torch.full((n_seq, blocks), -1, dtype=torch.int32, device="cuda")
        self.free, self.count = torch.arange(n_pages, dtype=torch.int32, device="cuda"), ints([n_pages])
        self.held, self.past, self.new = ints([0] * n_seq), ints([0] * n_seq), ints([0] * n_seq)
        self.q_start = ints([0] * (n_seq + 1))
        self.pos, self.slot = ints([0] * max_tokens), ints([0] * max_tokens)
        self.rows = torch.zeros((max_tokens, (n_q + 2 * n_kv) * dim), device="cuda", dtype=DT[act])
        self.q = torch.zeros((max_tokens, n_q * dim), device="cuda", dtype=DT[act])
        self.out = torch.full((max_tokens, n_q * dim), CANARY, device="cuda", dtype=DT[act])
        self.keys = [torch.zeros((0, n_kv, dim), device="cuda", dtype=torch.float16) for _ in range(n_seq)]
        self.values = [torch.zeros((0, n_kv, dim), device="cuda", dtype=torch.float16) for _ in range(n_seq)]
        self.scale = 1.0 / math.sqrt(dim)

    def step(self, max_new):
        """What the device runs; held becomes the new lengths, the count of free pages is kept in place."""
        nq, nk, w = self.n_q * self.dim, self.n_kv * self.dim, self.rows
        self.paged.plan(self.ctx, self.held, self.past, self.new, self.table, self.free, self.count, self.count, self.q_start, self.held, self.pos, self.slot,
                        page_size=self.page)
        self.cache.append(w[:, :nq], w[:, nq:nq + nk], w[:, nq + nk:], self.pos, self.slot, self.q, freq_base=self.base)
        self.cache.attn(self.q, self.table, self.q_start, self.held, max_new, self.scale, self.out)

    def check(self, past, new):
        """The rows of the last step against 64 bits, from the plain copies."""
        first = 0
        for s, (p, m) in enumerate(zip(past, new)):
            pos = torch.arange(p, p + m, device="cuda")
            x = self.rows[first:first + m].view(m, self.n_q + 2 * self.n_kv, self.dim)
            turned = append_expect(x[:, :self.n_q + self.n_kv], pos, self.dim, self.base)
            # the stored keys may round the other way where the f32 rotation lies on the border: they are read back
            slot = self.slot[first:first + m].long()
            k = self.k[slot // self.page, :, slot % self.page]
            assert ((k.double() - turned[:, self.n_q:]).abs() <= 2.0 ** -10 * turned[:, self.n_q:].abs() + 2.0 ** -20).all()
            v = self.v[slot // self.page, :, slot % self.page]
            assert torch.equal(v, x[:, self.n_q + self.n_kv:].half())
            self.keys[s] = torch.cat([self.keys[s][:p], k])
            self.values[s] = torch.cat([self.values[s][:p], v])
            q = self.q[first:first + m].view(m, self.n_q, self.dim)
            size = x[:, :self.n_q].double().abs().amax().item() if m else 0
            assert ((q.double() - turned[:, :self.n_q]).abs() <= (2.0 ** -20 + (2.0 ** -11 if self.act == "f16" else 0)) * 2 * size).all()
            got = self.out[first:first + m].double().view(m, self.n_q, self.dim)
            for h in range(self.n_q):
                kk, vv = (t[s][:, h * self.n_kv // self.n_q].double() for t in (self.keys, self.values))
                a = q[:, h].double() @ kk.t() * self.scale
                A = (q[:, h].double().abs() @ kk.t().abs() * self.scale).amax(-1, keepdim=True) if m else 0
                a = a.masked_fill(torch.arange(p + m, device="cuda")[None, :] > pos[:, None], -math.inf)
                w = a.softmax(-1)
                tol = (A + 1) * 2.0 ** -18 * (w @ vv.abs())
                if self.act == "f16":
                    tol = tol + 2.0 ** -11 * (w @ vv.abs()) + 2.0 ** -11 * (w @ vv).abs() + 2.0 ** -25
                assert ((got[:, h] - w @ vv).abs() <= tol).all(), (s, h)
            first += m
        assert (self.out[first:] == CANARY).all()
        self.out.fill_(CANARY)


STEPS = [  # (kept, new) per request; kept below the length: rewound, (0, 0): ended
    [(0, 70), (0, 5), (0, 1), (0, 0)],
    [(70, 1), (5, 1), (1, 1), (0, 150)],
    [(71, 1), (6, 4), (2, 1), (150, 33)],
    [(72, 1), (7, 3), (0, 0), (183, 1)],      # a draft is rewound by three tokens, a request ends
    [(73, 90), (10, 1), (0, 40), (180, 2)],   # its row is used again
    [(0, 0), (0, 0), (0, 0), (182, 1)],
    [(0, 3), (0, 200), (0, 0), (0, 0)],
]


@pytest.mark.parametrize("n_q,n_kv,dim,page,act", [(8, 2, 128, 16, "f32"), (8, 2, 64, 32, "f16"), (5, 1, 128, 64, "f32")])
def test_a_server(ctx, n_q, n_kv, dim, page, act):
    g = torch.Generator(device="cuda").manual_seed(dim)
    srv = Server(ctx, 4, 20, 40, page, n_q, n_kv, dim, act, 300)
    pages = 40
    for step in STEPS:
        past, new = [p for p, _ in step], [m for _, m in step]
        srv.rows.copy_(torch.randn(srv.rows.shape, generator=g, device="cuda"))
        srv.past.copy_(ints(past))
        srv.new.copy_(ints(new))
        srv.step(max(new))
        ctx.sync()
        assert ctx.status() == 0
        srv.check(past, new)
        pages_used = sum(-(-(p + m) // page) for p, m in step)
        assert srv.count.item() == pages - pages_used
        # every page is in one place
        used = [x for s, (p, m) in enumerate(step) for x in srv.table[s, :-(-(p + m) // page)].tolist()]
        assert sorted(used + srv.free[:srv.count.item()].tolist()) == list(range(pages))


def test_a_captured_step(ctx):
    """A step recorded once into a graph and replayed for other lengths: everything comes from the device."""
    from fast_llm_b200 import capi as c_
    own = c_.Context(0)
    try:
        srv = Server(own, 4, 20, 40, 16, 8, 2, 128, "f32", 300)
        g = torch.Generator(device="cuda").manual_seed(1)
        stream = torch.cuda.ExternalStream(own.stream())
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with pytest.raises(capi.Fl200Error) as e:          # the first call of a context allocates
            with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
                srv.cache.attn(srv.q, srv.table, srv.q_start, srv.held, 200, srv.scale, srv.out)
        assert "capture" in str(e.value)
        torch.cuda.synchronize()
        srv.cache.attn(srv.q, srv.table, srv.q_start, srv.held, 200, srv.scale, srv.out)
        own.sync()
        assert own.status() == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            srv.step(200)
        for step in STEPS:
            past, new = [p for p, _ in step], [m for _, m in step]
            srv.rows.copy_(torch.randn(srv.rows.shape, generator=g, device="cuda"))
            srv.past.copy_(ints(past))
            srv.new.copy_(ints(new))
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            torch.cuda.synchronize()
            assert own.status() == 0
            srv.check(past, new)
        del graph
    finally:
        own.close()


def test_calls_in_a_row_and_two_contexts(ctx):
    """Calls of unlike shapes without a wait between them share the context's scratch; another context has its own."""
    from fast_llm_b200 import paged
    shapes = [([(900, 1), (300, 1)], 32, 8, 128, 16, "f32"), ([(700, 300)], 8, 2, 128, 64, "f32"), ([(50, 1), (400, 90)], 8, 8, 64, 32, "f16"), ([(5000, 4)], 4, 1, 128, 16, "f32"),
              ([(300, 20)] * 9, 16, 8, 64, 16, "f32")]
    cases = [make(30 + i, *s) for i, s in enumerate(shapes)]
    other = capi.Context(0)
    try:
        for c, s in zip(cases, shapes):
            c["caches"] = [paged.PagedCache(x, c["k"], c["v"], c["n_pages"], s[4], s[2], s[3]) for x in (ctx, other)]
            c["outs"] = [torch.full_like(c["out_all"], CANARY) for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(6):
            for i in (0, 1):
                for c, s in zip(cases, shapes):
                    c["caches"][i].attn(c["q"], c["table"], c["q_start"], c["kv_len"], c["max_new"], 0.1, c["outs"][i][:, :s[1] * s[3]])
        ctx.sync()
        other.sync()
        assert ctx.status() == 0 and other.status() == 0
        for c, (seqs, n_q, n_kv, dim, page, act) in zip(cases, shapes):
            assert torch.equal(c["outs"][0], c["outs"][1])
            c["out"], c["out_all"] = c["outs"][0][:, :n_q * dim], c["outs"][0]
            want, tol, _ = expect(c, seqs, n_q, n_kv, dim, 0.1, act)
            got = c["out"].double().view(-1, n_q, dim)
            assert ((got[:c["n"]] - want[:c["n"]]).abs() <= tol[:c["n"]]).all()
            assert (c["out"][c["n"]:] == CANARY).all()
    finally:
        other.close()


@pytest.mark.parametrize("new", [1, 40])
def test_pools_past_32_bit_offsets(ctx, new):
    """Pools of more than 2^32 bytes and 2^31 values: pages at their very end, read and written."""
    from fast_llm_b200 import paged
    n_kv, dim, page, n_q = 8, 128, 64, 32
    n_pages = (1 << 31) // (n_kv * dim * page) + 70
    k = torch.zeros((n_pages, n_kv, page, dim), device="cuda", dtype=torch.float16)
    v = torch.zeros_like(k)
    cache = paged.PagedCache(ctx, k, v, n_pages, page, n_kv, dim)
    L = 200
    table = ints([[n_pages - 1, n_pages - 3, 0, n_pages - 40]])
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((L, (n_q + 2 * n_kv) * dim), generator=g, device="cuda")
    slot = (table[0].long()[torch.arange(L, device="cuda") // page] * page + torch.arange(L, device="cuda") % page).int()
    nq, nk = n_q * dim, n_kv * dim
    q = torch.zeros((L, nq), device="cuda")
    torch.cuda.synchronize()
    cache.append(x[:, :nq], x[:, nq:nq + nk], x[:, nq + nk:], torch.arange(L, device="cuda", dtype=torch.int32), slot, q, freq_base=10000.0)
    out = torch.zeros((new, nq), device="cuda")
    cache.attn(q[L - new:], table, ints([0, new]), ints([L]), new, 0.088, out)
    ctx.sync()
    assert ctx.status() == 0
    at = slot.long()
    kk, vv = (t[at // page, :, at % page] for t in (k, v))
    assert torch.equal(vv, x[:, nq + nk:].view(L, n_kv, dim).half()) and (kk != 0).any(-1).all()
    c = dict(q=q[L - new:], ks=[kk.transpose(0, 1)], vs=[vv.transpose(0, 1)], start=[0, new])
    want, tol, _ = expect(c, [(L, new)], n_q, n_kv, dim, 0.088, "f32")
    assert ((out.double().view(new, n_q, dim) - want).abs() <= tol).all()


def test_a_prompt_of_131072_tokens(ctx):
    """One sequence of 2^26 tiles and more: shares and owners of tiles past 32-bit products."""
    from fast_llm_b200 import paged
    N, n_q, dim, page = 131072, 128, 64, 256
    g = torch.Generator(device="cuda").manual_seed(12)
    k, v = (torch.randn((N // page, 1, page, dim), generator=g, device="cuda").half() for _ in range(2))
    table = torch.randperm(N // page, generator=g, device="cuda").int().view(1, -1)
    q = torch.empty((N, n_q * dim), device="cuda", dtype=torch.float16).normal_(generator=g)
    out = torch.full_like(q, CANARY)
    cache = paged.PagedCache(ctx, k, v, N // page, page, 1, dim)
    torch.cuda.synchronize()
    cache.attn(q, table, ints([0, N]), ints([N]), N, 0.125, out)
    ctx.sync()
    assert ctx.status() == 0
    kk, vv = (t[table[0].long()].reshape(N, dim).double() for t in (k, v))
    for tok in (0, 1, 2, 127, 128, 4097, 65535, 65536, 100001, N - 2, N - 1):
        x = q[tok].double().view(n_q, dim) @ kk[:tok + 1].t() * 0.125
        A = (q[tok].double().abs().view(n_q, dim) @ kk[:tok + 1].abs().t() * 0.125).amax(-1, keepdim=True)
        p = torch.softmax(x, -1)
        want, spread = p @ vv[:tok + 1], p @ vv[:tok + 1].abs()
        tol = (A + 1) * 2.0 ** -18 * spread + 2.0 ** -11 * spread + 2.0 ** -11 * want.abs() + 2.0 ** -25
        assert ((out[tok].double().view(n_q, dim) - want).abs() <= tol).all(), tok


@pytest.mark.parametrize("n_q,n_kv,dim", [(4, 1, 128), (4, 1, 64), (10, 5, 128), (32, 8, 64)])
@pytest.mark.parametrize("new", [1, 2, 3, 4])
def test_few_rows_over_long_caches(ctx, n_q, n_kv, dim, new):
    """Up to 296 records of up to 16 rows: more than are added at once; a CTA may be the last of two blocks."""
    seqs = [(40001, new), (33, 1), (5000, new)]
    c = make(dim + new, seqs, n_q, n_kv, dim, 64, "f32")
    attn(ctx, c, n_q, n_kv, dim, 64, 1.0 / math.sqrt(dim))
    check(ctx, c, seqs, n_q, n_kv, dim, 1.0 / math.sqrt(dim), "f32")
    first = c["out"].clone()
    attn(ctx, c, n_q, n_kv, dim, 64, 1.0 / math.sqrt(dim))
    assert torch.equal(first, c["out"])


@pytest.mark.parametrize("seed", range(16))
def test_ragged_batches_of_few_rows(ctx, seed):
    """Lengths, heads and counts at random: ends of shares fall anywhere among the sequences' tiles."""
    rng = np.random.default_rng(seed)
    n_kv = int(rng.choice([1, 2, 5, 8]))
    group = int(rng.choice([1, 2, 4]))
    most = 16 // group if seed % 2 else 1
    longest = int(rng.choice([70, 700, 7000]))
    seqs = [(int(L), int(min(m, L))) for L, m in zip(rng.integers(0, longest, 1 + 2 * seed), rng.integers(0, most + 1, 1 + 2 * seed))] + [(longest, 1)]
    dim, act = (64, "f16") if seed % 3 == 0 else (128, "f32")
    c = make(100 + seed, seqs, n_kv * group, n_kv, dim, 16, act)
    attn(ctx, c, n_kv * group, n_kv, dim, 16, 0.1)
    check(ctx, c, seqs, n_kv * group, n_kv, dim, 0.1, act)


def test_long_chunk_over_many_tiles(ctx):
    """Many tiles per piece: contexts go out and come back a quarter at a time; one key outweighs all others late in the walk, so
    that every sum changes its reference."""
    n_q, n_kv, dim, page = 8, 1, 128, 64
    for act in ("f32", "f16"):
        seqs = [(9000, 70)]
        c = make(77, seqs, n_q, n_kv, dim, page, act)
        for j in (3000, 6500):       # keys along q's mean direction, far larger than the others
            pg, r = int(c["table"][0, j // page]), j % page
            big = (4 + j // 1000) * torch.sign(c["q"][0].view(n_q, dim)[0]).half()
            c["k"][pg, 0, r] = big
            c["ks"][0][0, j] = big
        attn(ctx, c, n_q, n_kv, dim, page, 0.088)
        check(ctx, c, seqs, n_q, n_kv, dim, 0.088, act)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("key", [0, 130])
def test_a_row_of_one_key_keeps_its_value(ctx, dim, key):
    """Prompts whose rows attend one key alone, or one that outweighs the others by 2^-100 over up to eight tiles: the result is that key's
    value. Off by: the probability's two parts 2^-21 (cut after 10 bits, then half a step of 2^-11), the two products' sum cut to 24 bits 2^-23, the row's
    sum, its inverse, the products with the inverse and with the change of reference 2^-24 each: below 2^-20."""
    n_q, n_kv, page = 32, 8, 64
    seqs = [(1000, 1000), (900, 900), (700, 700), (1000, 1000)]   # about 450 blocks of rows: most are one CTA's
    c = make(dim + key, seqs, n_q, n_kv, dim, page, "f32", kv_scale=0.1)
    c["q"].abs_().add_(1.0)
    for s in range(len(seqs)):
        c["k"][int(c["table"][s, key // page]), :, key % page] = 4.0
    attn(ctx, c, n_q, n_kv, dim, page, 0.6)    # 0.6 sum q k: above 150 for the key, below 25 for the others
    assert ctx.status() == 0
    for s, (L, m) in enumerate(seqs):
        want = c["vs"][s][:, key].double().repeat_interleave(n_q // n_kv, 0)
        got = c["out"].double().view(-1, n_q, dim)[c["start"][s] + key:c["start"][s] + m]
        assert ((got - want).abs() <= 2.0 ** -20 * want.abs()).all(), ((got - want).abs() / want.abs()).max().item()
        first = c["vs"][s][:, 0].double().repeat_interleave(n_q // n_kv, 0)
        assert ((c["out"].double().view(-1, n_q, dim)[c["start"][s]] - first).abs() <= 2.0 ** -20 * first.abs()).all()


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("below", [20.3, 30.6, 35.4])
def test_many_keys_far_below_the_largest(ctx, act, below):
    """One key, and 20000 at 2^-below of it with values of one sign. A probability is held in two parts to 2^-21 of itself or to 2^-36 of the
    row's largest (f16: one part, 2^-11 or 2^-37)."""
    n_q, dim, page, N, new = 128, 64, 64, 20000, 300     # 150 blocks of rows: all keys of most are one CTA's
    seqs = [(N + new, new)]
    c = make(int(below), seqs, n_q, 1, dim, page, act)
    scale = 0.125
    c["q"].fill_(1.0)
    c["k"].zero_()
    c["v"].fill_(1.0)
    c["ks"][0].zero_()
    c["vs"][0].fill_(1.0)
    pg = int(c["table"][0, 0])
    size = below * math.log(2.0) / (scale * dim)          # the key's dimensions, in f16
    c["k"][pg, 0, 3], c["ks"][0][0, 3] = size, size
    c["v"][pg, 0, 3], c["vs"][0][0, 3] = 2.0 ** -12, 2.0 ** -12
    attn(ctx, c, n_q, 1, dim, page, scale)
    assert ctx.status() == 0
    k3 = float(c["ks"][0][0, 3, 0])
    A = scale * dim * k3
    for tok in (0, 7, new - 1):
        keys = N + tok + 1
        small = math.exp(-A) * (keys - 1)
        want = (2.0 ** -12 + small) / (1 + small)
        tol = (A + 1) * 2.0 ** -18 * want + keys * 2.0 ** -36
        if act == "f16":
            tol += 2 * 2.0 ** -11 * want + 2.0 ** -25
        got = c["out"].double().view(-1, n_q, dim)[tok]
        assert ((got - want).abs() <= tol).all(), ((got - want).abs().max().item(), tol, want)


@pytest.mark.parametrize("act", ["f32", "f16"])
def test_rows_of_a_million_keys(ctx, act):
    """Long sums, which tensor memory truncates at every instruction, in pieces of thousands of tiles: values of one come back as one. The sums
    of 2^13 tiles round to f32 at every tile (4 deviations: 4 2^-24 2^6.5 3^-1 for steps of a growing sum, numerator and denominator: 2^-17.1); f16: up to
    2^-13 cut off sums in tensor memory, the
    probabilities' roundings, 2^-11 at most and of either sign (over 2^20 keys 4 2^-11 3^-0.5 2^-10: 2^-19.8), and the result's half step."""
    from fast_llm_b200 import paged
    n_q, dim, page, N, new = 128, 64, 256, 1 << 20, 300   # 150 blocks of rows: all keys of most are one CTA's
    g = torch.Generator(device="cuda").manual_seed(20)
    k, v = torch.zeros((N // page, 1, page, dim), device="cuda", dtype=torch.float16), torch.ones((N // page, 1, page, dim), device="cuda", dtype=torch.float16)
    k[..., 0] = 8 * torch.rand((N // page, 1, page), generator=g, device="cuda")
    q = torch.ones((new, n_q * dim), device="cuda", dtype=DT[act])
    out = torch.full_like(q, CANARY)
    cache = paged.PagedCache(ctx, k, v, N // page, page, 1, dim)
    torch.cuda.synchronize()
    cache.attn(q, torch.arange(N // page, dtype=torch.int32, device="cuda").view(1, -1), ints([0, new]), ints([N]), new, 0.125, out)
    ctx.sync()
    assert ctx.status() == 0
    assert ((out.double() - 1).abs() <= 2.0 ** -17 + (2.0 ** -13 + 2.0 ** -19 + 2.0 ** -11 if act == "f16" else 0)).all(), (out.double() - 1).abs().max().item()


@pytest.mark.parametrize("seqs", [[(200, 3), (77, 1)], [(130, 70)]])
@pytest.mark.parametrize("q_size,k_size", [(1e35, 1e-4), (3e37, 1e-4), (1e-34, 1.0), (1e-37, 1.0)])
def test_rows_of_q_at_the_ends_of_f32(ctx, q_size, k_size, seqs):
    c = make(9, seqs, 8, 2, 128, 16, "f32", kv_scale=k_size)
    c["q"].mul_(q_size)
    scale = 1.0 / (q_size * k_size * math.sqrt(128))
    assert torch.isfinite(c["q"]).all()
    attn(ctx, c, 8, 2, 128, 16, scale)
    check(ctx, c, seqs, 8, 2, 128, scale, "f32")


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("n_q,n_kv,dim,seqs", [(8, 2, 128, [(900, 1), (3000, 3), (0, 1), (2, 4)]), (8, 2, 64, [(1500, 90), (700, 1), (3, 40)]), (32, 8, 128, [(1200, 600), (1000, 1000)])])
@pytest.mark.parametrize("rising", [False, True])
def test_lse_is_the_maximum_and_the_sum(ctx, n_q, n_kv, dim, seqs, act, rising):
    """Each of the two for itself, which what merges parts of a sequence needs. rising: the maximum grows by 0.3 exponents per 64 keys, so that references
    lag it. A score is off by 2^-19 A (see above), the maximum's product by 2^-23 of it, the sum by twice the scores', 2^-21 of the probabilities and 2^-18 for its roundings."""
    page = 16
    c = make(len(seqs) + dim, seqs, n_q, n_kv, dim, page, act)
    scale = 1.0 / math.sqrt(dim)
    if rising:
        c["q"].fill_(1.0)
        for s, (L, _) in enumerate(seqs):
            j = torch.arange(L, device="cuda")
            c["ks"][s].zero_()
            c["ks"][s][:, :, 0] = ((j // 64) * 0.2 / scale * (j % 64 == 17)).half()
            c["k"][c["table"][s].long()[j // page], :, j % page] = c["ks"][s].transpose(0, 1)
    attn(ctx, c, n_q, n_kv, dim, page, scale)
    assert ctx.status() == 0
    _, _, want = expect(c, seqs, n_q, n_kv, dim, scale, act)
    q = c["q"].double().abs().view(-1, n_q, dim)
    for s, (L, m) in enumerate(seqs):
        if not m:
            continue
        a = slice(c["start"][s], c["start"][s] + m)
        A = torch.zeros((m, n_q), dtype=torch.float64, device="cuda")
        for h in range(n_q):
            if L:
                A[:, h] = (q[a, h] @ c["ks"][s][h * n_kv // n_q].double().abs().t() * scale).amax(-1)
        got = c["lse"][a].double()
        none = want[a, :, 0] == -math.inf
        assert (got[none] == want[a][none]).all()
        m_off, s_off = (got[..., 0] - want[a, :, 0]).abs(), (got[..., 1] - want[a, :, 1]).abs()
        assert (m_off <= A * 2.0 ** -19 + 2.0 ** -22 * want[a, :, 0].abs())[~none].all()
        assert (s_off <= (2 * A * 2.0 ** -19 + 2.0 ** -18 + 2.0 ** -21) * want[a, :, 1])[~none].all()


@pytest.mark.parametrize("n_seq,new,kv_len", [(66, 1, 1 << 22), (1, 1, (1 << 22) + 64), (33, 17, 1 << 24), (32, 17, 1 << 24)])
def test_lines_that_32_bits_do_not_hold(ctx, n_seq, new, kv_len):
    """Sequences of together 2^32 tiles or more over all KV heads (one: 2^26), which can share their pages: reported, nothing is written."""
    from fast_llm_b200 import paged
    n_kv, dim, page = 1024, 64, 256
    k = torch.zeros((1, n_kv, page, dim), device="cuda", dtype=torch.float16)
    table = torch.zeros((n_seq, -(-kv_len // page)), dtype=torch.int32, device="cuda")
    q = torch.ones((n_seq * new, n_kv * dim), device="cuda", dtype=torch.float16)
    out = torch.full_like(q, CANARY)
    cache = paged.PagedCache(ctx, k, k, 1, page, n_kv, dim)
    torch.cuda.synchronize()
    cache.attn(q, table, ints([i * new for i in range(n_seq + 1)]), ints([kv_len] * n_seq), new, 0.125, out)
    ctx.sync()
    assert ctx.status() == 4
    assert (out == CANARY).all()


def test_plan_without_tokens(ctx):
    """A step in which requests only end or are rewound."""
    got = run_plan(ctx, [40, 17], [0, 5], [0, 0], [[0, 1, 2], [3, 4, -1]], [-1] * 5, 0, 16, 0)
    assert ctx.status() == 0
    assert got == dict(table=[[0, 1, 2], [3, 4, -1]], free=[0, 1, 2, 4, -1], count=4, pos=[], slot=[], start=[0, 0, 0], length=[0, 5])


@pytest.mark.parametrize("act,dim", [("f32", 128), ("f16", 128), ("f16", 64)])
@pytest.mark.parametrize("seqs,wide,max_new", [
    ([(700, 1)] * 2 + [(500, 30)], 0, None),                     # the table's width bounds the single tokens' work: one kernel takes all
    ([(700, 1)] * 2 + [(500, 30), (90, 90)], 4000, None),        # it does not, but the lengths are short: the same, after the other one looked at them
    ([(9000, 1), (8000, 2)] * 6 + [(500, 30)], 0, None),         # each by its rows
    ([(900, 1)] * 3 + [(900, 4)], 4000, 200),                    # a call that allows chunks and has none
    ([(900, 1)] * 3 + [(900, 4)], 0, 200),                       # the same under a narrow table
    ([(700, 1)] * 40 + [(500, 30), (64, 5)], 0, None)])          # more than 32 sequences
def test_sequences_of_few_rows_beside_chunks(ctx, seqs, wide, max_new, act, dim):
    n_q, n_kv, page = 16, 4, 16
    c = make(len(seqs) + wide, seqs, n_q, n_kv, dim, page, act)
    if wide:
        c["table"] = torch.cat([c["table"], torch.full((len(seqs), wide), -7, dtype=torch.int32, device="cuda")], 1).contiguous()
    if max_new:
        more = max_new + 2 - c["q"].shape[0]                     # (n_tokens bounds max_new)
        c["q"] = torch.cat([c["q"], c["q"].new_zeros((more, n_q * dim))])
        c["out_all"] = torch.full((max_new + 2, n_q * dim + 8), CANARY, device="cuda", dtype=DT[act])
        c["out"] = c["out_all"][:, :n_q * dim]
        c["lse"] = torch.full((max_new + 2, n_q, 2), CANARY, device="cuda")
    attn(ctx, c, n_q, n_kv, dim, page, 1.0 / math.sqrt(dim), max_new=max_new)
    check(ctx, c, seqs, n_q, n_kv, dim, 1.0 / math.sqrt(dim), act)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("seqs", [[(300, 1), (70, 2)], [(300, 100)]])
def test_scores_of_millions(ctx, seqs, act):
    """Rows whose scores reach 2^23: the largest takes all (the next one is 1000 below at least), its value comes back."""
    n_q, n_kv, dim, page = 8, 2, 128, 16
    c = make(41, seqs, n_q, n_kv, dim, page, act)
    c["q"].fill_(16.0)
    for s, (L, _) in enumerate(seqs):
        j = torch.arange(L, device="cuda")
        c["ks"][s].zero_()
        c["ks"][s][:, :, 1] = 32 * ((j * 37) % L).half()       # whole numbers below 2^14, all different
        c["k"][c["table"][s].long()[j // page], :, j % page] = c["ks"][s].transpose(0, 1)
    attn(ctx, c, n_q, n_kv, dim, page, 50.0)                    # 16 * 32 * 50 = 25600 a step, up to 7.7e6
    assert ctx.status() == 0
    got = c["out"].double().view(-1, n_q, dim)
    for s, (L, m) in enumerate(seqs):
        for i in range(m):
            best = int(((torch.arange(L - m + i + 1) * 37) % L).argmax())
            want = c["vs"][s][:, best].double().repeat_interleave(n_q // n_kv, 0)
            assert ((got[c["start"][s] + i] - want).abs() <= (2.0 ** -20 + (2.0 ** -10 if act == "f16" else 0)) * want.abs()).all()
