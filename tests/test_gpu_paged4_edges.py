"""The 4-bit paged cache and the verification of drafts at the ends of what their numbers may be: probabilities and picks that are none, value scales far apart or near fp16's last bits, far positions."""
import math

import numpy as np
import pytest
import torch

from paged4_ref import TYPES, Problem4, quantise, values
from xalm_b200 import paged

pytestmark = pytest.mark.gpu


# ---- drafts ------------------------------------------------------------------------------------------------------------------------------
def weight(x):
    return float(x) if float(x) > 0 else 0.0  # NaN too


def by_definition(starts, tokens, target, accept, pick, draft=None):
    """Tokens and how many drafts are taken; what is negative or no number is a zero before anything is done with it."""
    V, out, taken = target.shape[1], [None] * len(tokens), []
    for s in range(len(starts) - 1):
        at, end = starts[s], starts[s + 1]
        while at + 1 < end:
            x = int(tokens[at + 1])
            if not 0 <= x < V or not float(accept[at]) * (1.0 if draft is None else weight(draft[at, x])) < weight(target[at, x]):
                break
            out[at], at = x, at + 1
        taken.append(max(at - starts[s], 0))
        if starts[s] == end:
            continue
        p = [weight(w) for w in target[at].tolist()]
        left = p
        if at + 1 < end:
            if draft is None:
                left = [w if v != int(tokens[at + 1]) else 0.0 for v, w in enumerate(p)]
            else:
                left = [max(w - weight(d), 0.0) for w, d in zip(p, draft[at].tolist())]
        if not any(left):
            left = p
        some = [v for v, w in enumerate(left) if w > 0]
        r = float(pick[s])
        out[at] = -1
        if some:
            out[at] = some[-1]
            if r < 1:
                goal, total = max(r, 0.0) * math.fsum(left), 0.0
                for v in some:
                    total += left[v]
                    if total > goal:
                        out[at] = v
                        break
        for i in range(at + 1, end):
            out[i] = -1
    return out, taken


def check_verify(starts, tokens, target, accept, pick, draft=None):
    dev = lambda x: None if x is None else x.cuda()
    left = torch.full((tokens.shape[0],), 77, dtype=torch.int32, device="cuda")
    out, taken = paged.verify(torch.tensor(starts, dtype=torch.int32, device="cuda"), dev(tokens), dev(target), dev(accept), dev(pick), draft=dev(draft), out=left)
    want, want_taken = by_definition(starts, tokens, target, accept, pick, draft)
    assert taken.tolist() == want_taken
    assert out.tolist() == [77 if w is None else w for w in want]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [33, 3000])
def test_a_draft_of_no_probability_is_taken_as_one_of_zero(V, type):
    """The drafted token's own numbers, of target and draft: a sequence of two drafts for each pair, the second an ordinary one that is always taken."""
    odd = [-2.0, -0.0, 0.0, 0.5, 1.0, math.nan, -math.inf, -math.nan]
    cases = [(q, p, u) for q in odd for p in odd for u in (0.0, 0.25, 0.75)] + [(math.inf, p, u) for p in odd for u in (0.25, 0.75)]
    B, x = len(cases), 7
    g = torch.Generator().manual_seed(11)
    target, draft = (torch.randint(0, 8, (3 * B, V), generator=g) / 1024 for _ in range(2))  # sums are exact
    accept = torch.full((3 * B,), 0.5)
    tokens = torch.full((3 * B,), x, dtype=torch.int32)
    for i, (q, p, u) in enumerate(cases):
        draft[3 * i, x], target[3 * i, x], accept[3 * i] = q, p, u
        draft[3 * i + 1, x], target[3 * i + 1, x] = 0.25, 0.5
    pick = torch.rand(B, generator=g)
    t = TYPES[type]
    check_verify(list(range(0, 3 * B + 1, 3)), tokens, target.to(t), accept, pick, draft.to(t))


@pytest.mark.parametrize("known", [None, True, False])
@pytest.mark.parametrize("type", ["f32", "f16"])
@pytest.mark.parametrize("V", [1, 5, 1000, 40000])
def test_a_pick_that_is_not_below_1_draws_the_last_weight(V, type, known):
    """And one below 0 the first, as 0 does; behind refused drafts and without any."""
    g = torch.Generator().manual_seed(V)
    picks = [math.nan, -math.nan, 1.0, 1.0, 1.5, 2.0, 1e30, math.inf, 1 - 2.0 ** -24, 0.0, -0.0, -1.0, -math.inf]
    B, n = len(picks), 1 if known is None else 2
    target, draft = (torch.randn(n * B, V, generator=g).mul(3).softmax(dim=1) for _ in range(2))
    target[:, V - V // 3:] = 0  # the last weight is not the last token, and parts of the vocabulary have none
    target[:, :V // 4] = 0
    tokens = torch.full((n * B,), V // 2, dtype=torch.int32)
    accept = torch.full((n * B,), 1.0)
    target[0::n, V // 2] = 0  # refused
    if V == 1:
        target[:] = 0.5
        accept[:] = 2.0
    t = TYPES[type]
    check_verify(list(range(0, n * B + 1, n)), tokens, target.to(t), accept, torch.tensor(picks), draft.to(t) if known else None)


# ---- attention --------------------------------------------------------------------------------------------------------------------------
def near(got, want, tol, what=""):
    over = (got.double().cpu() - want).abs() - tol
    assert float(over.max()) <= 0, f"{what}: {float(over.max())} over the tolerance at {int((over > 0).sum())} of {over.numel()}"


def check_as_few(p):
    """attend4 against 64 bits by the tolerances of few rows (Problem4.attend), however many there are: p d enters the second product as one fp16 number for bf16, as two for fp16 and fp32.  In units where
    the largest scale that the row sees, D, is 2^11 at least, fp16's last place is off by 2^-25: by 2^-36 D in p d, by 8 times that in a value's part, for each key, where the largest p is 1."""
    cache, batch = p.on_gpu()
    out, lse = paged.attend4(cache, batch, p.gq, p.scale, want_lse=True)
    cache.check()
    p.many = lambda s: False
    want, want_lse, tol, tol_lse = p.attend()
    if p.type != "f32":
        for n in range(p.rows):
            s, last = p.row(n)
            at = torch.arange(last + 1)
            pages = p.table[s].long()[at // p.page]
            score = torch.einsum("grd,jgd->grj", p.q[n].double().unflatten(0, (p.G, p.rep)), p.k[pages, :, at % p.page]) * p.scale
            total = torch.exp(want_lse[n] - score.amax(dim=-1).flatten())  # the sum of p
            scales = p.pool_scales(1)[pages, :, at % p.page].double().abs().max()
            tol[n] += (8 * (last + 1) * 2.0 ** -36 * float(scales) / total)[:, None]
    near(out, want, tol, "out")
    near(lse, want_lse, tol_lse, "lse")


MANY = [dict(new=[1], rep=70), dict(new=[20], rep=4), dict(new=[1] * 20, rep=4, groups=([0, 20], [128]))]  # more than 64 rows that read the same keys


@pytest.mark.parametrize("power", [-8, -14, -20, -24, 12])
@pytest.mark.parametrize("kind", range(len(MANY)))
@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_many_rows_keep_small_probabilities_of_small_and_large_scales(type, kind, power):
    """Of 64 keys 63 lie e^14 to e^19 below the first: they count with all the bits that the result has, at scales of 2^power."""
    n = 135
    p = Problem4(type, lens=[n] * len(MANY[kind]["new"]), G=1, d=32, page=64, seed=66, **MANY[kind])
    k, v = torch.zeros(p.pages, 1, 64, 32), torch.zeros(p.pages, 1, 64, 32)
    k[..., 0] = -8.0
    v[..., 1] = -8.0 * 2.0 ** power
    k[:, 0, 0] = 0
    v[:, 0, 0] = 0
    v[:, 0, 0, 0] = -8.0 * 2.0 ** power
    p.fill(k, v)
    p.q[:] = 0
    p.q[..., 0] = (14 + 5 * torch.rand(p.rows, p.H, generator=p.gen)).to(p.t) / 8
    p.scale = 1.0
    check_as_few(p)


@pytest.mark.parametrize("kind", range(len(MANY)))
@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_many_rows_have_the_bits_of_few(type, kind):
    """All keys but the first of each page alike, each row with a probability of its own for them: the numbers that fp16 rounds are the same for all of them, and so are its errors."""
    p = Problem4(type, lens=[135] * len(MANY[kind]["new"]), G=1, d=32, page=64, seed=67, **MANY[kind])
    k, v = torch.zeros(p.pages, 1, 64, 32), torch.zeros(p.pages, 1, 64, 32)
    k[..., 0] = -8.0
    v[..., :] = -8.0 * (1 + torch.arange(32) // 4 / 8) * 1.2822265625  # scales of 11 bits
    k[:, 0, 0] = 0
    v[:, 0, 0] = 0
    p.fill(k, v)
    p.q[:] = 0
    p.q[..., 0] = (2 * torch.rand(p.rows, p.H, generator=p.gen)).to(p.t) / 8
    p.scale = 1.0
    check_as_few(p)


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_long_prompts_have_the_bits_of_few_rows(type):
    for groups in (None, ([0, 3], [256])):
        check_as_few(Problem4(type, [90, 1, 200], [900, 300, 456], rep=4, d=128, dv=64, page=64, seed=68, groups=groups))


@pytest.mark.parametrize("power", [12, 18, 24, 30])
@pytest.mark.parametrize("where", [0, 5, 150, 299])
@pytest.mark.parametrize("rep", [1, 4, 6, 16])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_a_large_scale_of_next_to_no_weight_takes_no_bits_from_fp32_rows(type, rep, where, power):
    """A value 2^power times the others', e^-90 below their scores (the largest of the first keys, where it is the first): fp32 rows are as exact as without it, others lose what is below 2^-36 of it."""
    p = Problem4(type, [1, 3], [300, 310], G=2, rep=rep, d=64, page=16, seed=69)
    k, v = torch.randn(p.pages, 2, 16, 64, generator=p.gen), torch.randn(p.pages, 2, 16, 64, generator=p.gen) * 2.0 ** -14
    p.q[..., 0] = 12.0
    k[..., 0] = 7.5
    for s in range(2):
        for at in range(where + 1 if where < 6 else 0):  # those before it as far below
            k[p.table[s, at // 16], :, at % 16, 0] = -7.5
        k[p.table[s, where // 16], :, where % 16, 0] = -7.5
        v[p.table[s, where // 16], :, where % 16] *= 2.0 ** power
    p.fill(k, v)
    p.scale = 0.5
    check_as_few(p)


@pytest.mark.parametrize("rep", [1, 4, 6, 16])
def test_fp32_rows_whose_scores_grow_as_their_scales_shrink(rep):
    """Every key some e^3 above the one before it, its value 2^-0.5 as large: the unit of the sums follows the products, down as well as up."""
    p = Problem4("f32", [1, 3], [70, 64], G=2, rep=rep, d=64, page=16, seed=70)
    k, v = torch.randn(p.pages, 2, 16, 64, generator=p.gen) * 0.1, torch.randn(p.pages, 2, 16, 64, generator=p.gen)
    for s in range(2):
        for at in range(p.lens[s]):
            k[p.table[s, at // 16], :, at % 16, 0] = 0.15 * at - 5
            v[p.table[s, at // 16], :, at % 16] *= 2.0 ** (12 - 0.5 * at)
    p.fill(k, v)
    p.q[..., 0] = 20.0
    p.scale = 1.0
    check_as_few(p)


# ---- appending --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("last", [1 << 30, (1 << 29) + 77])
def test_keys_at_the_farthest_positions_are_the_definitions(last, neighbours):
    """Keys whose turned entries lie next to borders between two codes, at positions of 30 bits and angles to a turn for every position: the product of position and frequency has more than 53 bits."""
    P, G, n, rot = 256, 8, 32, 1024 // 32
    g = torch.Generator().manual_seed(12)
    freq = (0.5 + 0.5 * torch.rand(rot, generator=g)).float()
    pages = (last + P - 1) // P
    pos = np.arange(last - n, last)
    angle = pos.astype(np.longdouble)[:, None] * freq.numpy().astype(np.longdouble)  # 54 bits
    assert np.finfo(np.longdouble).nmant >= 63
    cs, sn = np.cos(angle)[:, None], np.sin(angle)[:, None]
    i = np.arange(rot)
    a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + rot)
    aim = (torch.randint(-7, 7, (n, G, 64), generator=g) + 0.5).numpy().astype(np.longdouble)
    aim[..., 0], aim[..., 32] = -8, -8
    k = np.zeros((n, G, 64), dtype=np.float32)
    k[..., a], k[..., b] = aim[..., a] * cs + aim[..., b] * sn, aim[..., b] * cs - aim[..., a] * sn  # turned back
    x, y = k[..., a].astype(np.longdouble), k[..., b].astype(np.longdouble)
    turned = np.zeros((n, G, 64), dtype=np.float32)
    turned[..., a], turned[..., b] = x * cs - y * sn, y * cs + x * sn
    want = values(*quantise(torch.from_numpy(turned)), 64)

    pool = torch.zeros(2, G, paged.page4_bytes(P, 64), dtype=torch.uint8, device="cuda")
    table = torch.zeros(1, pages, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    cache = paged.PagedCache4(pool, P, 64)
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")
    batch = paged.Batch(i32([0, n]), i32([last]), table)
    rows = torch.from_numpy(k).cuda()
    q = paged.append4(cache, batch, rows, rows, q=rows, freq=freq.cuda(), neighbours=neighbours)
    got = paged.read4(cache, batch, n)[0].double().cpu()
    cache.check()
    assert torch.equal(got, want), f"{int((got != want).sum())} of {got.numel()} numbers"
    # queries: cos and sin within 2^-22, three roundings of fp32
    assert float((q.double().cpu() - torch.from_numpy(turned).double()).abs().max()) <= 2.0 ** -21 * float(rows.abs().max())
