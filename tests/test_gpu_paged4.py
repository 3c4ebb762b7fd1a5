"""The 4-bit paged cache and the verification of drafts on a GPU, against a plain restatement in 64 bits (paged4_ref.py, which also derives the tolerances)."""
import math
import threading

import pytest
import torch

from paged4_ref import BLOCKS, HALF, TYPES, Problem4, pack, quantise, turned, unpack, values, verify
from xalm_b200 import capi, paged

pytestmark = pytest.mark.gpu


def near(got, want, tol, what=""):
    """NaN where that is, within tol elsewhere."""
    got = got.double().cpu()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got[~fin]), torch.isnan(want[~fin])) and torch.equal(got[~fin].nan_to_num(), want[~fin].nan_to_num()), what
    over = ((got - want).abs() - tol)[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {float(over.max())} over the tolerance at {int((over > 0).sum())} of {over.numel()}"


def check_attend(p, only=None):
    cache, batch = p.on_gpu()
    left = torch.full((p.rows, p.H, p.dv), 7.0, dtype=p.t, device="cuda")
    out, lse = paged.attend4(cache, batch, p.gq, p.scale, out=left, want_lse=True)
    cache.check()
    want, want_lse, tol, tol_lse = p.attend(only)
    rows = [n for n in range(p.rows) if p.row(n) is not None] if only is None else only
    near(out[rows], want[rows], tol[rows], "out")
    near(lse[rows], want_lse[rows], tol_lse[rows], "lse")
    outside = [n for n in range(p.rows) if p.row(n) is None]
    assert (out[outside] == 7.0).all(), "rows outside every sequence"
    return out, lse


SHAPES = {
    "one": dict(new=[1], lens=[1]),
    "one_long": dict(new=[1], lens=[1000]),
    "ragged": dict(new=[1, 1, 1, 1], lens=[1, 63, 64, 65]),
    "many": dict(new=[1] * 37, lens=[(17 * i) % 301 + 1 for i in range(37)]),
    "empty": dict(new=[0, 1, 0, 3, 0], lens=[0, 5, 40, 3, 17], pad_rows=3, offset=2),
    "drafts": dict(new=[5, 3, 1, 6, 2], lens=[105, 200, 77, 6, 400]),
    "prompt": dict(new=[70], lens=[70]),
    "chunk": dict(new=[33, 1, 150], lens=[133, 200, 151], pad_rows=1),
    "shared": dict(new=[1] * 9, lens=[256 + 7 * i for i in range(9)], groups=([0, 9], [256])),
    "two_groups": dict(new=[1] * 12, lens=[129] * 5 + [300 + i for i in range(7)], groups=([0, 5, 12], [128, 256])),
    "group_and_alone": dict(new=[1, 2, 3, 1, 1], lens=[70, 130, 131, 132, 9], groups=([1, 4], [64])),
    "shared_chunks": dict(new=[40, 25, 60], lens=[256 + 40, 256 + 30, 256 + 200], groups=([0, 3], [256])),
}


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_attend(shape, type):
    check_attend(Problem4(type, d=64, page=64, seed=1, **SHAPES[shape]))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,dv", [(8, 8), (16, 128), (40, 72), (64, 256), (80, 80), (96, 64), (128, 64), (128, 128), (192, 128), (256, 64), (128, 256), (256, 256)])
def test_attend_of_any_head_size(d, dv, type):
    check_attend(Problem4(type, [1, 20, 1], [90, 150, 64], d=d, dv=dv, page=32, seed=2))
    check_attend(Problem4(type, [1, 5, 40], [130, 140, 170], d=d, dv=dv, page=32, seed=3, groups=([0, 3], [128])))


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("order", ["head", "page", "layer"])
def test_attend_of_any_page(page, order, type):
    check_attend(Problem4(type, [1, 1, 40, 1], [page, page + 1, 3 * page - 1, 700], d=64, page=page, order=order, seed=4))


@pytest.mark.parametrize("type", ["f32", "f16"])
@pytest.mark.parametrize("G,rep", [(1, 1), (3, 1), (2, 5), (1, 8), (1, 16), (1, 20), (5, 8), (1, 71)])
def test_attend_of_any_heads(G, rep, type):
    check_attend(Problem4(type, [1, 7, 1], [50, 60, 300], G=G, rep=rep, d=32, page=16, seed=5))
    check_attend(Problem4(type, [1, 7, 1], [250, 260, 300], G=G, rep=rep, d=32, page=16, seed=6, groups=([0, 3], [240])))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3, 3.0])
def test_attend_of_any_scale(scale, type):
    """Scores' signs turned, all equal, nearly equal, and so far apart that one key has nearly everything."""
    for groups in (None, ([0, 3], [192])):
        p = Problem4(type, [1, 9, 40], [193, 260, 300], d=64, page=64, seed=46, groups=groups)
        p.scale = scale
        check_attend(p)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,rep,d,dv,page", [(8, 4, 64, 64, 16), (8, 4, 128, 128, 64), (6, 5, 80, 72, 32), (16, 1, 128, 64, 256), (4, 16, 128, 128, 128), (2, 3, 192, 256, 64)])
def test_long_prompts(G, rep, d, dv, page, type):
    """Prompts of many units, whose pieces a block meets several of, with and without pages in common; some rows of every sequence are looked at."""
    new, lens = [700, 1, 37, 300, 1, 513], [1900, 1500, 1061, 1324, 1025, 1537]
    for groups in (None, ([0, 2, 6], [1024, 1024])):
        p = Problem4(type, new, lens, G=G, rep=rep, d=d, dv=dv, page=page, seed=47, groups=groups, pad_rows=5)
        check_attend(p, sorted({min(p.starts[s] + x, p.starts[s + 1] - 1) for s in range(len(new)) for x in (0, 1, 31, 32, 63, 64, 128, 255, 400, new[s] - 1)}))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,rep", [(1, 1), (2, 4), (3, 5)])
def test_groups_of_several_tokens_to_a_sequence(G, rep, type):
    new, lens = [16, 20, 0, 9, 31, 1, 3, 17, 2, 25], [290, 276, 256, 300, 287, 70, 67, 150, 66, 600]
    check_attend(Problem4(type, new, lens, G=G, rep=rep, d=64, page=64, seed=50, groups=([0, 5, 6, 9], [256, 64, 64]), pad_rows=2, offset=1))


@pytest.mark.parametrize("type", ["f32", "f16"])
def test_thousands_of_sequences(type):
    check_attend(Problem4(type, [1] * 4000, [i % 19 + 1 for i in range(4000)], G=1, rep=1, d=256, page=16, seed=48), only=list(range(0, 4000, 37)) + [3999])


def magnitudes(p, low, high):
    """Keys and values of all sizes, alike within a token's head."""
    g = torch.Generator().manual_seed(60)
    shape = (p.pages, p.G, p.page)
    size = lambda: torch.exp2(torch.rand(*shape, 1, generator=g) * (high - low) + low)
    return torch.randn(*shape, p.d, generator=g) * size(), torch.randn(*shape, p.dv, generator=g) * size()


@pytest.mark.parametrize("rep", [4, 8, 16, 30, 70])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_scales_of_all_sizes(type, rep):
    """Tokens whose scales differ by up to 2^12, the largest ones anywhere: the unit of the sums grows as they come."""
    p = Problem4(type, [1, 3], [600, 333], rep=rep, d=64, page=16, seed=61)
    p.fill(*magnitudes(p, -8, 4))
    check_attend(p)


@pytest.mark.parametrize("rep", [1, 4, 8, 16, 30])
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_what_a_row_does_not_see_may_be_no_number_or_of_any_size(type, rep):
    """Behind a row's own position lie blocks that are no numbers and scales 2^30 above its own; what nobody sees is all ones already."""
    p = Problem4(type, [12, 30], [200, 47], rep=rep, d=64, page=16, seed=62)
    want, want_lse, tol, tol_lse = p.attend()
    for s, first in ((0, 195), (1, 40)):  # these positions and all behind them
        for at in range(first, p.lens[s]):
            pg, sl = int(p.table[s, at // 16]), at % 16
            k, v = torch.full((1, p.G, 16, 64), 3.0e5 if at % 2 else math.nan), torch.full((1, p.G, 16, 64), -5.0e5 if at % 3 else math.inf)
            one = pack(k, v)
            o = 0
            for size in (32, 4, 32, 4):
                p.pool[pg, :, o + sl * size:o + (sl + 1) * size] = one[0, :, o + sl * size:o + (sl + 1) * size]
                o += 16 * size
    cache, batch = p.on_gpu()
    out, lse = paged.attend4(cache, batch, p.gq, p.scale, want_lse=True)
    rows = [n for n in range(p.rows) if p.row(n)[1] < (195, 40)[p.row(n)[0]]]
    near(out[rows], want[rows], tol[rows])
    near(lse[rows], want_lse[rows], tol_lse[rows])


@pytest.mark.parametrize("rep", [1, 4, 8, 16, 30])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_a_block_that_is_no_number_stays_in_its_block_and_its_rows(type, rep):
    p = Problem4(type, [10], [150], rep=rep, d=96, page=16, seed=63)
    k, v = torch.randn(p.pages, p.G, 16, 96, generator=p.gen), torch.randn(p.pages, p.G, 16, 96, generator=p.gen)
    v[p.table[0, 9], 0, 2, 40] = math.nan  # position 146, the second block
    p.fill(k, v)
    cache, batch = p.on_gpu()
    out = paged.attend4(cache, batch, p.gq, p.scale).cpu()
    bad = torch.isnan(out)
    seen = torch.tensor([p.row(n)[1] >= 146 for n in range(10)])
    head = torch.arange(p.H) < rep
    entry = (torch.arange(96) >= 32) & (torch.arange(96) < 64)
    assert torch.equal(bad, seen[:, None, None] & head[:, None] & entry)
    k[p.table[0, 9], 1, 2, 0] = math.inf
    p.fill(k, v.nan_to_num())
    cache, batch = p.on_gpu()
    out, lse = paged.attend4(cache, batch, p.gq, p.scale, want_lse=True)
    assert torch.equal(torch.isnan(lse.cpu()), seen[:, None] & ~head) and torch.equal(torch.isnan(out.cpu()), (seen[:, None] & ~head)[..., None].expand(-1, -1, 96))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_queries_of_any_size(type):
    """Rows whose largest entries are far from 1, zeros, and a row that is no number beside others."""
    p = Problem4(type, [1, 6], [99, 300], rep=6, d=64, page=16, seed=64)
    sizes = [1.0, 2.0 ** -13, 0.0, 2.0 ** 12, 1.0, 2.0 ** -9, 30.0] if type == "f16" else [1.0, 2.0 ** -100, 0.0, 2.0 ** 40, 1e-30, 2.0 ** -126, 30.0]
    p.q *= torch.tensor(sizes, dtype=p.t)[:, None, None]
    p.scale = 0.05
    check_attend(p)
    p.q[4, 3, 5] = math.nan
    p.q[4, 7, 0] = math.inf
    cache, batch = p.on_gpu()
    out = paged.attend4(cache, batch, p.gq, p.scale).cpu()
    bad = torch.isnan(out).any(dim=2)
    assert bad[4, 3] and bad[4, 7] and int(bad.sum()) == 2


@pytest.mark.parametrize("rep", [1, 8, 16, 70])
@pytest.mark.parametrize("type", ["f16", "bf16", "f32"])
def test_an_infinite_query_gives_no_number_whatever_the_keys(type, rep):
    """All keys of one sign: their scores are all the same infinity."""
    p = Problem4(type, [2], [40], G=1, rep=rep, d=64, page=16, seed=74)
    p.fill(-torch.rand(p.pages, 1, 16, 64, generator=p.gen) - 0.5, torch.randn(p.pages, 1, 16, 64, generator=p.gen))
    p.q[0, 0, 7], p.q[1, rep - 1, 9] = math.inf, -math.inf
    cache, batch = p.on_gpu()
    out, lse = paged.attend4(cache, batch, p.gq, p.scale, want_lse=True)
    bad = torch.zeros(2, rep, dtype=torch.bool)
    bad[0, 0], bad[1, rep - 1] = True, True
    assert torch.equal(torch.isnan(lse.cpu()), bad) and torch.equal(torch.isnan(out.cpu()), bad[..., None].expand(2, rep, 64))


@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("rep", [1, 8, 16, 70])
@pytest.mark.parametrize("type", ["f16", "bf16", "f32"])
def test_scores_that_fp32_holds_to_a_few_units_give_finite_results(type, rep, rows):
    """Scores around 2^26, where neighbouring fp32 numbers are more than the running maximum's slack apart."""
    p = Problem4(type, [rows], [400], G=1, rep=rep, d=64, page=16, seed=65)
    p.q = (p.q.abs() + 1).to(p.t)
    p.scale = 2.0 ** 20
    cache, batch = p.on_gpu()
    out, lse = paged.attend4(cache, batch, p.gq, p.scale, want_lse=True)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    assert (out.abs().double().cpu().amax() <= p.v.nan_to_num().abs().max() * 1.01)


@pytest.mark.parametrize("rep", [1, 8, 16, 70])
@pytest.mark.parametrize("type", ["f16", "bf16", "f32"])
def test_scores_too_large_for_fp32_to_tell_apart_count_alike(type, rep):
    """All keys the same and scores around 2^30: the mean of the values, wherever the largest scale is among them."""
    p = Problem4(type, [1], [500], G=1, rep=rep, d=64, page=16, seed=75)
    g = torch.Generator().manual_seed(76)
    size = torch.exp2(torch.randint(-6, 7, (p.pages, 1, 16, 1), generator=g).float())
    p.fill(torch.full((p.pages, 1, 16, 64), -8.0), torch.randn(p.pages, 1, 16, 64, generator=g) * size)
    p.q[:] = -(2.0 ** 10)
    p.scale = 2.0 ** 11
    cache, batch = p.on_gpu()
    out, lse = paged.attend4(cache, batch, p.gq, p.scale, want_lse=True)
    used = p.v.nan_to_num().flatten(0, 2)[~torch.isnan(p.v).flatten(0, 2).any(dim=1)]
    want = used.mean(dim=0)
    # equal probabilities: sums of 500 numbers in fp32, and of products of two fp16 roundings where there are many rows; then the type's own rounding
    tol = want.abs() * HALF[type] + used.abs().mean(dim=0) * (2.0 ** -13 if type == "f32" else 2.0 ** -10)
    near(out.double().cpu(), want.expand(1, rep, 64), tol.expand(1, rep, 64))
    assert torch.allclose(lse.cpu(), torch.full_like(lse.cpu(), 64 * 8 * 2.0 ** 21), rtol=2 ** -20)


@pytest.mark.parametrize("rep", [4, 8, 16, 40, 70])
@pytest.mark.parametrize("type", ["f16", "bf16", "f32"])
def test_many_small_probabilities_beside_a_large_one(type, rep):
    """8192 keys e^-14 below the first, with values that add up beside its own: they count with all the bits that the result has."""
    n = 8193
    p = Problem4(type, [1], [n], G=1, rep=rep, d=32, page=64, seed=66)
    k, v = torch.zeros(p.pages, 1, 64, 32), torch.zeros(p.pages, 1, 64, 32)
    k[..., 0] = -8.0
    v[..., 1] = -800.0
    first = int(p.table[0, 0])
    k[first, 0, 0] = 0
    v[first, 0, 0] = 0
    v[first, 0, 0, 0] = -8.0
    p.fill(k, v)
    p.q[:] = 0
    p.q[..., 0] = 14.0 / 8
    p.scale = 1.0
    check_attend(p)


def test_rows_before_the_first_token_see_nothing():
    """More rows than the sequence has tokens: the first two are zeros, the others as they should be, and the arrays are reported."""
    p = Problem4("bf16", [6], [4], d=64, page=16, seed=67)
    cache, batch = p.on_gpu()
    out, lse = paged.attend4(cache, batch, p.gq, p.scale, want_lse=True)
    with pytest.raises(capi.XalmError, match="do not fit"):
        cache.check()
    assert (out[:2] == 0).all() and (lse[:2] == -math.inf).all()
    want, want_lse, tol, tol_lse = p.attend()
    near(out[2:], want[2:], tol[2:])
    near(lse[2:], want_lse[2:], tol_lse[2:])


@pytest.mark.parametrize("type", ["f32", "f16"])
def test_pages_outside_the_pool_read_as_zeros_and_are_reported(type):
    p = Problem4(type, [1, 20], [100, 90], d=64, page=16, seed=68)
    cache, batch = p.on_gpu()
    for bad in (-1, p.pages, 2 ** 31 - 1, -2 ** 31):
        batch.tensors[2][0, 2] = bad
        batch.tensors[2][1, 1] = bad
        k, v = p.k.clone(), p.v.clone()
        out, lse = paged.attend4(cache, batch, p.gq, p.scale, want_lse=True)
        got = paged.read4(cache, batch, p.rows)
        with pytest.raises(capi.XalmError, match="outside the pool"):
            cache.check()
        cache.check()
        p.k[p.table[0, 2]], p.v[p.table[0, 2]], p.k[p.table[1, 1]], p.v[p.table[1, 1]] = 0, 0, 0, 0
        want, want_lse, tol, tol_lse = p.attend()
        near(out, want, tol)
        near(lse, want_lse, tol_lse)
        for n in range(p.rows):
            s, at = p.row(n)
            assert torch.equal(got[0][n].double().cpu(), p.k[p.table[s, at // 16], :, at % 16])
        p.k, p.v = k, v


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_arrays_that_do_not_fit_stay_in_bounds_and_are_reported(type):
    p = Problem4(type, [1, 5, 3], [40, 70, 33], d=64, page=16, seed=69)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    big = 2 ** 31 - 1
    k = torch.randn(p.rows, p.G, 64, device="cuda").to(p.t)
    for starts, lens in (([0, 1, 6, 9], [big, 70, 33]), ([0, 1, 6, 9], [40, -5, 33]), ([0, 1, 6, big], [40, 70, 33]), ([-3, 1, 6, 9], [40, 70, 33]), ([0, 6, 1, 9], [40, 70, 33]), ([0, 1, 6, 9], [0, 2, 33])):
        cache, batch = p.on_gpu()
        batch = paged.Batch(i32(starts), i32(lens), batch.tensors[2])
        for call in (lambda: paged.attend4(cache, batch, p.gq, p.scale), lambda: paged.read4(cache, batch, p.rows), lambda: paged.append4(cache, batch, k, k)):
            call()
            with pytest.raises(capi.XalmError, match="do not fit"):
                cache.check()
        del cache
    cache, batch = p.on_gpu()
    for groups, shared in (([0, big], [16]), ([-5, 2], [big]), ([2, 1], [16]), ([0, 3], [-7])):
        paged.attend4(cache, paged.Batch(i32(p.starts), i32(p.lens), batch.tensors[2], groups=i32(groups), shared=i32(shared)), p.gq, p.scale)
    torch.cuda.synchronize()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_rows_of_a_wider_array(type):
    p = Problem4(type, [1, 3, 30], [40, 70, 90], d=64, dv=128, page=16, seed=70)
    cache, batch = p.on_gpu()
    wide = torch.full((p.rows, p.H * 64 + 24), 3.0, dtype=p.t, device="cuda")
    q = wide[:, 8:8 + p.H * 64].unflatten(1, (p.H, 64))
    q.copy_(p.gq)
    room = torch.full((p.rows, p.H * 128 + 16), 5.0, dtype=p.t, device="cuda")
    out = room[:, 8:8 + p.H * 128].unflatten(1, (p.H, 128))
    paged.attend4(cache, batch, q, p.scale, out=out)
    want, _, tol, _ = p.attend()
    near(out, want, tol)
    assert (room[:, :8] == 5).all() and (room[:, -8:] == 5).all()


def test_offsets_past_32_bits():
    """A pool of more than 4 GB: the last pages are as good as the first."""
    P, G, d = 64, 8, 128
    n = paged.page4_bytes(P, d)
    pages = (5 << 30) // (G * n)
    pool = torch.zeros(pages, G, n, dtype=torch.uint8, device="cuda")
    p = Problem4("bf16", [1, 4], [200, 300], G=G, d=d, page=P, seed=71)
    far = p.table.clone()
    where = {}
    for s in range(2):
        for j in range(-(-p.lens[s] // P)):
            at = pages - 1 - len(where)
            where[int(p.table[s, j])] = at
            far[s, j] = at
    for a, b in where.items():
        pool[b] = p.pool[a].cuda()
    cache = paged.PagedCache4(pool, P, d)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    batch = paged.Batch(i32(p.starts), i32(p.lens), far.cuda())
    out = paged.attend4(cache, batch, p.q.cuda(), p.scale)
    want, _, tol, _ = p.attend()
    near(out, want, tol)
    k = torch.randn(5, G, d, device="cuda")
    paged.append4(cache, batch, k, k)
    got = paged.read4(cache, batch, 5)
    assert torch.equal(got[0].double().cpu(), values(*quantise(k.cpu()), d)) and torch.equal(got[0], got[1])
    cache.check()


def test_groups_change_nothing_but_the_order_of_sums():
    p = Problem4("bf16", [1] * 20, [1024 + 13 * i for i in range(20)], d=128, page=64, seed=72, groups=([0, 20], [1024]))
    got = check_attend(p)
    cache, batch = p.on_gpu()
    alone = paged.attend4(cache, paged.Batch(*batch.tensors[:3]), p.gq, p.scale)
    tol = p.attend()[2]
    near(alone, got[0].double().cpu(), 2 * tol)


def test_calls_repeat_themselves_bit_for_bit():
    for kw in (dict(new=[1] * 30, lens=[100 + 31 * i for i in range(30)]), dict(new=[5] * 9, lens=[500] * 9, groups=([0, 9], [448])), dict(new=[300, 20], lens=[400, 900])):
        for type in ("f32", "f16"):
            p = Problem4(type, d=64, page=64, seed=73, **kw)
            cache, batch = p.on_gpu()
            first = paged.attend4(cache, batch, p.gq, p.scale)
            for _ in range(5):
                assert torch.equal(paged.attend4(cache, batch, p.gq, p.scale), first)


# ---- appending and reading -----------------------------------------------------------------------------------------------------------------------
def stored(p, x, freq, mag, neighbours, turn):
    """Scales and codes of rows x (rows, G, n) as the cache keeps them."""
    y = x.double().clone()
    if turn:
        for n in range(p.rows):
            if p.row(n) is not None:
                y[n] = turned(x[n], p.row(n)[1], freq, mag, neighbours)
    return quantise(y.float())


def check_append(p, in_type, freq=None, mag=1.0, neighbours=False, with_q=True, size=1.0, x=None):
    g = torch.Generator().manual_seed(80)
    t = TYPES[in_type]
    k, v = (torch.randn(p.rows, p.G, n, generator=g).mul(size).to(t) for n in (p.d, p.dv)) if x is None else x
    q = torch.randn(p.rows, p.H, p.d, generator=g).to(t)
    cache, batch = p.on_gpu()
    before = p.gpool.cpu()
    q_out = torch.full((p.rows, p.H, p.d), 7.0, dtype=t, device="cuda")
    gf = None if freq is None else freq.cuda()
    got = paged.append4(cache, batch, k.cuda(), v.cuda(), q=q.cuda() if with_q else None, freq=gf, mag=mag, neighbours=neighbours, q_out=q_out if with_q else None)
    cache.check()
    kd, kc = stored(p, k, freq, mag, neighbours, True)
    vd, vc = stored(p, v, freq, mag, neighbours, False)
    want_k, want_v = unpack(before, p.page, p.d, p.dv)
    rows = [n for n in range(p.rows) if p.row(n) is not None]
    for n in rows:
        s, at = p.row(n)
        want_k[p.table[s, at // p.page], :, at % p.page] = values(kd[n], kc[n], p.d)
        want_v[p.table[s, at // p.page], :, at % p.page] = values(vd[n], vc[n], p.dv)
    after = p.gpool.cpu()
    for have, want in zip(unpack(after, p.page, p.d, p.dv), (want_k, want_v)):
        assert torch.equal(torch.isnan(have), torch.isnan(want)) and torch.equal(have.nan_to_num(), want.nan_to_num())
    touched = torch.zeros(p.pages, p.page, dtype=torch.bool)
    for n in rows:
        s, at = p.row(n)
        touched[p.table[s, at // p.page], at % p.page] = True
    at = 0
    for b in (BLOCKS(p.d), BLOCKS(p.dv)):
        for size in (16 * b, 2 * b):
            a, c = (z[:, :, at:at + p.page * size].unflatten(2, (p.page, size)).transpose(1, 2)[~touched] for z in (before, after))
            assert torch.equal(a, c), "slots of other tokens"
            at += p.page * size
    if with_q:
        half = HALF[in_type]
        for n in range(p.rows):
            if n not in rows:
                assert (got[n] == 7).all()
                continue
            want = turned(q[n], p.row(n)[1], freq, mag, neighbours)
            # cos and sin are within 2^-22 of the angle's, as are three roundings of fp32; then the type's own
            tol = want.abs() * half + 2.0 ** -21 * q[n].abs().double().max() * max(abs(mag), 1) + (2.0 ** -25 if in_type == "f16" else 0)
            near(got[n], want, tol, "q")
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        rk, rv = paged.read4(cache, batch, p.rows, dtype=dtype)
        for n in rows:
            for have, d, c, w in ((rk, kd, kc, p.d), (rv, vd, vc, p.dv)):
                want = values(d[n], c[n], w).to(dtype)
                assert torch.equal(have[n].cpu().nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))
    return cache, batch, k, v


@pytest.mark.parametrize("in_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("neighbours", [False, True])
def test_append(in_type, neighbours):
    freq = 10000.0 ** (-torch.arange(32) / 32)
    check_append(Problem4("f16", [3, 0, 1, 40, 1], [70, 0, 1, 90, 16], d=64, page=16, seed=81, offset=2, pad_rows=3), in_type, freq, 1.25, neighbours)


@pytest.mark.parametrize("order", ["head", "page", "layer"])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("d,dv,rot", [(8, 16, 4), (40, 72, 5), (64, 64, 0), (80, 96, 20), (96, 64, 16), (128, 256, 64), (256, 128, 100), (192, 192, 96), (256, 256, 128)])
def test_append_of_any_head_size(d, dv, rot, neighbours, order):
    freq = 10000.0 ** (-torch.arange(rot) / max(rot, 1))
    check_append(Problem4("f16", [3, 1, 21], [70, 1, 33], G=3, rep=2, d=d, dv=dv, page=32, order=order, seed=82), "bf16", freq if rot else None, 1.0, neighbours)


@pytest.mark.parametrize("in_type", ["f32", "bf16", "f16"])
def test_append_of_any_size(in_type):
    """Numbers below and above what fp16 scales have, halves between two codes, both signs alike, zeros, and what is no number."""
    p = Problem4("f16", [12], [12], G=1, rep=1, d=64, page=16, seed=83)
    k = torch.randn(12, 1, 64, generator=torch.Generator().manual_seed(84))
    k[1] *= 2.0 ** -22
    k[2] *= 2.0 ** -16
    k[3] = 0
    k[4] = (torch.arange(64) % 16 - 8) * 0.5 + 0.25  # between two codes of 1/2
    k[4, 0, 0], k[4, 0, 32] = -4, -4
    k[5] = torch.where(torch.arange(64) % 2 == 0, 3.0, -3.0)
    k[6] *= 60000.0 if in_type == "f16" else 1e30
    k[6].clamp_(-65504, 65504) if in_type == "f16" else None
    k[7, 0, 3], k[8, 0, 40], k[9, 0, 63] = math.nan, math.inf, -math.inf
    k[10] = 1e-45 if in_type == "f32" else 0
    k[11, 0, :32] = torch.linspace(0, 7.5, 32)  # one sign
    k = k.to(TYPES[in_type])
    check_append(p, in_type, x=(k, k.flip(0)), with_q=False)


@pytest.mark.parametrize("in_type", ["f32", "bf16"])
def test_append_where_scales_have_few_bits_or_all(in_type):
    """Rows of sizes 2^-26 to 2^18 (scales below fp16's normal numbers are far from -M / 8), and rows whose quotients lie on borders between two codes."""
    p = Problem4("f16", [90], [90], G=1, rep=1, d=64, page=16, seed=77)
    g = torch.Generator().manual_seed(78)
    k = torch.randn(90, 1, 64, generator=g) * torch.exp2(torch.arange(90) / 2 - 26)[:, None, None]
    d = torch.exp2(torch.randint(-10, 8, (90, 1, 2), generator=g).float()) * (1 + torch.randint(0, 1024, (90, 1, 2), generator=g) / 1024)
    half = torch.randint(-17, 16, (90, 1, 64), generator=g) / 2
    half[..., 0], half[..., 32] = -8, -8
    v = half.clamp_min(-8) * d.repeat_interleave(32, dim=2)
    check_append(p, in_type, x=(k.to(TYPES[in_type]), v.to(TYPES[in_type])), with_q=False)


def test_append_far_positions_and_many_rows():
    freq = 1e6 ** (-torch.arange(32) / 32)
    p = Problem4("f16", [2, 1], [200000, 131073], G=1, rep=1, d=64, page=256, seed=85, k=torch.zeros(1300, 1, 256, 64), v=torch.zeros(1300, 1, 256, 64), spare=1300 - 782 - 513)
    check_append(p, "bf16", freq)
    check_append(Problem4("f16", [500, 1, 300], [520, 1, 1000], G=2, rep=2, d=64, page=64, seed=86), "f16", freq)


def test_append_leaves_out_what_has_no_slot():
    p = Problem4("f16", [5, 3], [40, 20], G=2, d=64, page=16, seed=87)
    cache, batch = p.on_gpu()
    before = p.gpool.clone()
    k = torch.randn(8, 2, 64, device="cuda")
    batch.tensors[2].fill_(-1)
    paged.append4(cache, batch, k, k)
    with pytest.raises(capi.XalmError, match="outside the pool"):
        cache.check()
    assert torch.equal(p.gpool, before)
    batch.tensors[2].copy_(p.table)
    batch.tensors[1].copy_(torch.tensor([p.table.shape[1] * 16 + 5, 2], dtype=torch.int32))  # behind the table; before the first token
    paged.append4(cache, batch, k, k)
    with pytest.raises(capi.XalmError, match="do not fit"):
        cache.check()
    now, was = p.gpool.view(p.pages, -1), before.view(p.pages, -1)
    changed = {int(x) for x in torch.nonzero((now != was).any(dim=1)).flatten()}
    assert changed == {int(p.table[1, 0])}


def test_results_that_overlap_what_a_call_is_given_are_refused():
    p = Problem4("f16", [4], [40], d=64, page=16, seed=88)
    cache, batch = p.on_gpu()
    k = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda")
    q = torch.zeros(4, 8, 64, dtype=torch.float16, device="cuda")
    for call in (lambda: paged.append4(cache, batch, k, k, q=q, q_out=q), lambda: paged.attend4(cache, batch, q, 1.0, out=q), lambda: paged.read4(cache, batch, 4, dtype=torch.float16, k=k, v=k),
                 lambda: paged.append4(cache, batch, k, k.float()), lambda: paged.append4(cache, batch, k[:3], k), lambda: paged.attend4(cache, batch, q[:, :, :32], 1.0),
                 lambda: paged.attend4(cache, batch, q.double(), 1.0), lambda: paged.attend4(cache, batch, q, 1.0, out=q.float()), lambda: paged.attend4(cache, batch, q, math.nan),
                 lambda: paged.append4(cache, batch, k, k, freq=torch.zeros(33, device="cuda")), lambda: paged.append4(cache, batch, k, k, q_out=q), lambda: paged.attend4(cache, batch, q[:, :3], 1.0)):
        with pytest.raises(capi.XalmError):
            call()
    raw = p.gpool.view(-1)[:4 * 8 * 64 * 2].view(torch.float16).view(4, 8, 64)
    with pytest.raises(capi.XalmError, match="overlaps the pool"):
        paged.attend4(cache, batch, q, 1.0, out=raw)
    L, need = capi.lib(), 10 ** 7
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    for at, room in ((p.gpool.data_ptr() // 256 * 256, need), (work.data_ptr(), 100)):
        (bp, held) = batch.of(4)
        assert L.xalm_cuda_paged4_attend(cache.p, bp, q.data_ptr(), 512, 8, 1, 1.0, torch.empty_like(q).data_ptr(), 512, None, at, room, None) in (1, 2)


# ---- streams, graphs, threads ----------------------------------------------------------------------------------------------------------------------
def test_a_captured_step_follows_its_arrays_and_other_streams_do_not_meet():
    p = Problem4("bf16", [1, 1, 1], [50, 64, 130], d=128, page=16, seed=90)
    longer = Problem4("bf16", [1, 1, 1], [20, 100, 99], d=128, page=16, seed=91)
    cache, batch = p.on_gpu()
    lens, table = batch.tensors[1], batch.tensors[2]
    k, v = torch.randn(3, 2, 128, device="cuda").bfloat16(), torch.randn(3, 2, 128, device="cuda").bfloat16()
    freq = (1e4 ** (-torch.arange(64) / 64)).cuda()

    def step():
        q = paged.append4(cache, batch, k, v, q=p.gq, freq=freq)
        return paged.attend4(cache, batch, q, p.scale)

    pool = p.gpool.clone()
    want = step()
    p.gpool.copy_(pool)
    side = [torch.cuda.Stream() for _ in range(3)]
    graphs, outs = [], []
    for s in side[:2]:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(step())
        graphs.append(g)
    p.gpool.copy_(pool)
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(side[2]):
            other = paged.attend4(cache, batch, p.gq, p.scale)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want) and torch.isfinite(other).all()
    lens.copy_(torch.tensor([49, 60, 131], dtype=torch.int32))
    table[2, 8] = p.table[2, 8]
    want = step()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want)
    del longer


def test_calls_of_different_sizes_in_several_threads():
    p = Problem4("f16", [1, 6, 30, 2], [77, 200, 95, 16], d=64, page=16, seed=92)
    cache, batch = p.on_gpu()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    want = paged.attend4(cache, batch, p.gq, p.scale)
    few = paged.Batch(i32([0, 1, 2, 3, 4]), batch.tensors[1], batch.tensors[2])
    q4 = p.gq[:4].contiguous()
    want4 = paged.attend4(cache, few, q4, p.scale)
    bad = []

    def work(b, q, w):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(100):
                if not torch.equal(paged.attend4(cache, b, q, p.scale), w):
                    bad.append(1)

    threads = [threading.Thread(target=work, args=x) for x in ((batch, p.gq, want), (few, q4, want4), (batch, p.gq, want), (few, q4, want4))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


# ---- drafts ----------------------------------------------------------------------------------------------------------------------------------------
def draft_problem(B, drafts, V, type="f32", known=True, seed=0, offset=0, pad=0, peak=2.0):
    g = torch.Generator().manual_seed(seed)
    starts = [offset]
    for s in range(B):
        n = int(torch.randint(drafts[0], drafts[1] + 1, (1,), generator=g))
        starts.append(starts[-1] + (n + 1 if n >= 0 else 0))
    N = starts[-1] + pad
    logits = torch.randn(N, V, generator=g) * peak
    target, draft = logits.softmax(dim=1), (logits + torch.randn(N, V, generator=g)).softmax(dim=1)
    drawn = torch.multinomial(draft, 1, generator=g).squeeze(1) if known else draft.argmax(dim=1)
    tokens = torch.cat((drawn[:1], drawn[:-1])).to(torch.int32)
    t = TYPES[type]
    return starts, tokens, target.to(t), torch.rand(N, generator=g), torch.rand(B, generator=g), draft.to(t) if known else None


def check_verify(starts, tokens, target, accept, pick, draft=None):
    dev = lambda x: None if x is None else x.cuda()
    left = torch.full((tokens.shape[0],), 77, dtype=torch.int32, device="cuda")
    out, taken = paged.verify(torch.tensor(starts, dtype=torch.int32, device="cuda"), dev(tokens), target if target.is_cuda else dev(target), dev(accept), dev(pick),
                              draft=draft if draft is None or draft.is_cuda else dev(draft), out=left)
    want, want_taken = verify(starts, tokens, target.cpu(), accept, pick, None if draft is None else draft.cpu())
    assert taken.tolist() == want_taken
    assert out.tolist() == [77 if w is None else w for w in want]
    return want_taken


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("V", [1, 2, 31, 128, 1000, 4097, 32003])
def test_verify(V, known, type):
    problem = list(draft_problem(9, (-1, 5), V, type, known and V > 1, seed=V, offset=2, pad=3))
    check_verify(*problem)
    problem[3] = problem[3] * 0.02  # nearly every draft is taken
    check_verify(*problem)


@pytest.mark.parametrize("B,drafts,V", [(1, (0, 0), 50000), (1, (70, 70), 300), (200, (0, 2), 515), (3, (8, 8), 131072)])
def test_verify_of_any_size(B, drafts, V):
    check_verify(*draft_problem(B, drafts, V, seed=5))


def test_verify_picks_at_both_ends_and_on_every_border():
    """Weights of whole parts of 2^-10: sums are exact, and each border belongs to the token behind it."""
    V = 1 << 10
    w = torch.zeros(V)
    w[5:900:7] = 1.0
    w = w / 1024
    n = int((w > 0).sum())
    picks = torch.tensor([0.0, 1 - 2.0 ** -24] + [i / n for i in range(0, n, 3)], dtype=torch.float32)
    B = len(picks)
    check_verify(list(range(B + 1)), torch.zeros(B, dtype=torch.int32), w.expand(B, V).contiguous(), torch.zeros(B), picks)


def test_verify_counts_what_is_no_probability_as_nothing():
    V = 700
    starts, tokens, target, accept, pick, draft = draft_problem(8, (3, 3), V, seed=9)
    target[0] = draft[0]  # nothing is left of it
    accept[0] = 1.0
    target[4:8] = 0  # nothing at all
    target[9, ::2], target[9, 1::4], draft[9, 3::5] = math.nan, -1.0, -2.0
    target[13, 5:], draft[13] = 0, 1.0
    tokens[17], tokens[21] = -1, V
    tokens[26] = 2 ** 31 - 1
    check_verify(starts, tokens, target, accept, pick, draft)
    check_verify(starts, tokens, target, accept, pick)
    late = pick.clone()
    late[:4] = torch.tensor([1.0, 2.0, -1.0, math.inf])
    dev = lambda x: x.cuda()
    out, taken = paged.verify(torch.tensor(starts, dtype=torch.int32, device="cuda"), *map(dev, (tokens, target, accept, late)), draft=dev(draft))
    assert ((out >= -1) & (out < V)).all() and ((taken >= 0) & (taken <= 3)).all()


def test_verify_rows_of_wider_arrays_and_bad_starts():
    starts, tokens, target, accept, pick, draft = draft_problem(6, (2, 5), 1001, seed=10)
    N = len(tokens)
    for width, at in ((1001, 0), (1024, 0), (1030, 3), (1028, 4)):
        wide_p, wide_q = torch.full((N, width + 8), 9.0, device="cuda"), torch.full((N, width + 8), 9.0, device="cuda")
        a, b = wide_p[:, at:at + 1001], wide_q[:, at:at + 1001]
        a.copy_(target), b.copy_(draft)
        check_verify(starts, tokens, a, accept, pick, b)
    big = 2 ** 31 - 1
    dev = lambda x: x.cuda()
    for bad in ([0, 3, 2, 9, big, big, N], [-5, -3, 0, 4, 5, 6, N + 100], [big] * 7):
        out, taken = paged.verify(torch.tensor(bad, dtype=torch.int32, device="cuda"), *map(dev, (tokens, target, accept, pick)), draft=dev(draft))
        torch.cuda.synchronize()
    for call in (lambda: paged.verify(out[:3], dev(tokens), dev(target), dev(accept), dev(pick)), lambda: paged.verify(out, dev(tokens), dev(target).double(), dev(accept), dev(pick)),
                 lambda: paged.verify(out[:7], dev(tokens).long(), dev(target), dev(accept), dev(pick)), lambda: paged.verify(out[:7], dev(tokens), dev(target), dev(accept), dev(pick), draft=dev(draft)[:, :5]),
                 lambda: paged.verify(out[:7], dev(tokens), dev(target).T, dev(accept), dev(pick)), lambda: paged.verify(out[:7], dev(tokens), dev(target), dev(accept)[:3], dev(pick))):
        with pytest.raises(capi.XalmError):
            call()


# ---- a run of them -----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_serving_with_drafts(type):
    """Two sequences of a one-layer model over a 4-bit cache: prompts, then steps of a token and three drafts; what the drafts wrote is overwritten where they are not taken.  After every step the
    cache holds what appending the tokens taken one by one would have left, and attention over it is the definition's."""
    t, V, G, rep, d, P = TYPES[type], 50, 2, 4, 64, 16
    g = torch.Generator().manual_seed(95)
    H = G * rep
    emb = {n: torch.randn(V, h, d, generator=g).to(t) for n, h in (("q", H), ("k", G), ("v", G))}
    head = torch.randn(H * d, V, generator=g) / 8
    freq = 1e4 ** (-torch.arange(32) / 32)
    text = [[3, 7, 1, 44, 20, 9, 9, 13, 2], [5] * 20 + [6, 7]]
    pages = 12
    pool = torch.full((pages, G, paged.page4_bytes(P, d)), 255, dtype=torch.uint8, device="cuda")
    cache = paged.PagedCache4(pool, P, d)
    table = torch.arange(pages, dtype=torch.int32).flip(0).view(2, 6)
    kept = [[], []]  # tokens whose keys and values the cache holds for good
    fresh = [list(x) for x in text]  # tokens of the next call that are certain
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for step in range(6):
        guess = [[int(x) for x in torch.randint(V, (3,), generator=g)] if step else [] for _ in range(2)]
        rows = [fresh[s] + guess[s] for s in range(2)]
        starts = [0, len(rows[0]), len(rows[0]) + len(rows[1])]
        lens = [len(kept[s]) + len(rows[s]) for s in range(2)]
        flat = rows[0] + rows[1]
        batch = paged.Batch(i32(starts), i32(lens), table.cuda())
        q = paged.append4(cache, batch, emb["k"][flat].cuda(), emb["v"][flat].cuda(), q=emb["q"][flat].cuda(), freq=freq.cuda())
        out = paged.attend4(cache, batch, q, d ** -0.5)
        cache.check()
        p = Problem4(type, [len(r) for r in rows], lens, G=G, rep=rep, d=d, page=P, seed=0)
        p.table, p.q, p.scale = table, q.cpu(), d ** -0.5
        p.pool = pool.cpu()
        p.pages = pages
        p.k, p.v = unpack(p.pool, P, d, d)
        for s in range(2):  # what the cache holds is the tokens' own, one by one
            for at, x in enumerate(kept[s] + rows[s]):
                want = values(*quantise(turned(emb["k"][x], at, freq, 1.0, False).float()), d)
                assert torch.equal(p.k[table[s, at // P], :, at % P], want)
                assert torch.equal(p.v[table[s, at // P], :, at % P], values(*quantise(emb["v"][x].float()), d))
        want, _, tol, _ = p.attend()
        near(out, want, tol)
        target = (out.float().flatten(1).cpu() @ head).softmax(dim=1)
        draft = torch.full_like(target, 1.0 / V)
        accept, pick = torch.rand(len(flat), generator=g), torch.rand(2, generator=g)
        # behind a prompt only its last row counts: what it has certain is no draft
        vstarts, vrows = [0], []
        for s in range(2):
            vrows += range(starts[s] + len(fresh[s]) - 1, starts[s + 1])
            vstarts.append(len(vrows))
        args = torch.tensor(flat, dtype=torch.int32)[vrows], target[vrows], accept[vrows], pick, draft[vrows]
        check_verify(vstarts, *args)
        got, taken = paged.verify(i32(vstarts), *(x.cuda() for x in args[:4]), draft=args[4].cuda())
        for s in range(2):
            n = int(taken[s])
            kept[s] += fresh[s] + guess[s][:n]
            fresh[s] = [int(got[vstarts[s] + n])]


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("new,rep,groups", [([64] * 40, 1, None), ([65] * 40, 1, None), ([16] * 60, 4, ([0, 30, 60], [16, 16])), ([1] * 300, 7, ([0, 100, 300], [16, 32])), ([17, 3] * 30, 4, ([0, 60], [32])),
                                            ([400] + [1] * 50, 4, None)])
def test_as_many_units_as_there_is_room_for(new, rep, groups, type):
    """Segments that just are, or just are not, the kernel's of many rows, in numbers that fill the workspace's places."""
    lens = [n + 32 + (7 * i) % 40 for i, n in enumerate(new)]
    p = Problem4(type, new, lens, G=3, rep=rep, d=64, page=16, seed=93, groups=groups)
    check_attend(p, only=list(range(0, p.rows, max(1, p.rows // 150))) + [p.rows - 1])
