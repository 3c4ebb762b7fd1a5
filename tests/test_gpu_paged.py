"""The paged cache's operators on a GPU, against a plain restatement in 64 bits (paged_ref.py, which also derives the tolerances)."""
import math

import pytest
import torch

from paged_ref import HALF, F32, TYPES, Problem
from xalm_b200 import capi, paged

pytestmark = pytest.mark.gpu


def near(got, want, tol, what=""):
    """Equal where it is not finite, within tol elsewhere."""
    got = got.double().cpu()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got[~fin]), torch.isnan(want[~fin])) and torch.equal(got[~fin].nan_to_num(), want[~fin].nan_to_num()), what
    over = ((got - want).abs() - tol)[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {float(over.max())} over the tolerance at {int((over > 0).sum())} of {over.numel()}"


def check_attend(p, lists=None, groups=True):
    cache, batch = p.on_gpu()
    left = torch.full((p.rows, p.H, p.dv), 7.0, dtype=p.t, device="cuda")
    if lists is None:
        out, lse = paged.attend(cache, batch, p.gq, p.scale, out=left, want_lse=True)
    else:
        out, lse = paged.attend_selected(cache, batch, p.gq, lists.to("cuda"), p.scale, out=left, want_lse=True)
    want, want_lse, tol, tol_lse = p.attend(lists)
    inside = ~torch.isnan(want).all(dim=2).all(dim=1) | torch.tensor([p.row(n) is not None for n in range(p.rows)])
    near(out[inside.to("cuda")], want[inside], tol[inside], "out")
    near(lse[inside.to("cuda")], want_lse[inside], tol_lse[inside], "lse")
    assert (out[~inside.to("cuda")] == 7.0).all(), "rows outside every sequence"
    cache.check()
    return out, lse


SHAPES = {
    "one": dict(new=[1], lens=[1]),
    "one_long": dict(new=[1], lens=[1000]),
    "ragged": dict(new=[1, 1, 1, 1], lens=[1, 63, 64, 65]),
    "many": dict(new=[1] * 37, lens=[(17 * i) % 301 + 1 for i in range(37)]),
    "empty": dict(new=[0, 1, 0, 3, 0], lens=[0, 5, 40, 3, 17], pad_rows=3, offset=2),
    "prompt": dict(new=[70], lens=[70]),
    "chunk": dict(new=[33, 1, 150], lens=[133, 200, 151], pad_rows=1),
    "shared": dict(new=[1] * 9, lens=[256 + 7 * i for i in range(9)], groups=([0, 9], [256])),
    "two_groups": dict(new=[1] * 12, lens=[128] * 0 + [129] * 5 + [300 + i for i in range(7)], groups=([0, 5, 12], [128, 256])),
    "group_and_alone": dict(new=[1, 2, 3, 1, 1], lens=[70, 130, 131, 132, 9], groups=([1, 4], [64])),
    "shared_chunks": dict(new=[40, 25, 60], lens=[256 + 40, 256 + 30, 256 + 200], groups=([0, 3], [256])),
}


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_attend(shape, type):
    check_attend(Problem(type, d=64, page=64, seed=1, **SHAPES[shape]))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,dv", [(8, 8), (16, 128), (40, 72), (80, 80), (128, 64), (128, 128), (192, 128), (256, 256)])
def test_attend_of_any_head_size(d, dv, type):
    check_attend(Problem(type, [1, 20, 1], [90, 150, 64], d=d, dv=dv, page=32, seed=2))
    check_attend(Problem(type, [1, 5, 70], [130, 140, 200], d=d, dv=dv, page=32, seed=3, groups=([0, 3], [128])))


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["position", "head"])
def test_attend_of_any_page(page, layout, type):
    check_attend(Problem(type, [1, 1, 40, 1], [page, page + 1, 3 * page - 1, 700], d=64, page=page, layout=layout, seed=4))


@pytest.mark.parametrize("type", ["f32", "f16"])
@pytest.mark.parametrize("G,rep", [(1, 1), (3, 1), (2, 5), (1, 16), (1, 20), (5, 8), (1, 71)])
def test_attend_of_any_heads(G, rep, type):
    check_attend(Problem(type, [1, 7, 1], [50, 60, 300], G=G, rep=rep, d=32, page=16, seed=5))
    check_attend(Problem(type, [1, 7, 1], [250, 260, 300], G=G, rep=rep, d=32, page=16, seed=6, groups=([0, 3], [240])))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3, 3.0])
def test_attend_of_any_scale(scale, type):
    """Scores' signs turned, all equal, nearly equal, and so far apart that one key has nearly everything."""
    for groups in (None, ([0, 3], [192])):
        p = Problem(type, [1, 9, 40], [193, 260, 300], d=64, page=64, seed=46, groups=groups)
        p.scale = scale
        check_attend(p)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,rep,d,dv,page", [(8, 4, 64, 64, 16), (8, 4, 128, 128, 64), (6, 5, 80, 72, 32), (16, 1, 128, 64, 256), (4, 16, 128, 128, 128), (2, 3, 192, 256, 64)])
def test_long_prompts(G, rep, d, dv, page, type):
    """Prompts of many units, whose pieces a block meets several of, with and without pages in common; some rows of every sequence are looked at."""
    new, lens = [700, 1, 37, 300, 1, 513], [1900, 1500, 1061, 1324, 1025, 1537]
    for groups in (None, ([0, 2, 6], [1024, 1024])):
        p = Problem(type, new, lens, G=G, rep=rep, d=d, dv=dv, page=page, seed=47, groups=groups, pad_rows=5)
        some = sorted({min(p.starts[s] + x, p.starts[s + 1] - 1) for s in range(len(new)) for x in (0, 1, 31, 32, 63, 64, 127, 128, 255, 256, 400, new[s] - 1)})
        cache, batch = p.on_gpu()
        out, lse = paged.attend(cache, batch, p.gq, p.scale, want_lse=True)
        cache.check()
        want, want_lse, tol, tol_lse = p.attend(only=some)
        near(out[some], want[some], tol[some], "out")
        near(lse[some], want_lse[some], tol_lse[some], "lse")


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,rep", [(1, 1), (2, 4), (8, 2), (3, 5)])
def test_groups_of_several_tokens_to_a_sequence(G, rep, type):
    """Many rows that each have shared pages and pages of their own, groups of one sequence and sequences without new tokens among them."""
    new, lens = [16, 20, 0, 9, 31, 1, 3, 17, 2, 25], [290, 276, 256, 300, 287, 70, 67, 150, 66, 600]
    check_attend(Problem(type, new, lens, G=G, rep=rep, d=64, page=64, seed=50, groups=([0, 5, 6, 9], [256, 64, 64]), pad_rows=2, offset=1))


def test_thousands_of_sequences_with_the_largest_heads():
    """So many that shared memory has room for one tile of keys and values beside them only."""
    check_attend(Problem("f32", [1] * 4000, [i % 19 + 1 for i in range(4000)], G=1, rep=1, d=256, page=16, seed=48))


def test_calls_in_two_threads_do_not_meet():
    """One cache and one batch, calls of different numbers of rows at the same time."""
    import threading
    p = Problem("bf16", [3, 5], [300, 400], G=2, d=64, page=64, seed=49, pad_rows=4)
    cache, batch = p.on_gpu()
    want = {n: paged.attend(cache, batch, p.gq[:n], p.scale) for n in (8, 12)}
    wrong = []

    def serve(n):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(200):
                out = paged.attend(cache, batch, p.gq[:n], p.scale)
                stream.synchronize()
                if not torch.equal(out[:8], want[n][:8]):
                    wrong.append(n)

    threads = [threading.Thread(target=serve, args=(n,)) for n in (8, 12)]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    cache.check()
    assert not wrong


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_groups_change_nothing_but_the_order_of_sums(type):
    """More shared tokens than the sequences have, parts of pages, overlong groups, groups of one: the annotation is cut to what holds."""
    for groups in (([0, 4], [10 ** 9]), ([0, 4], [70]), ([0, 1, 4], [64, 64]), ([0, 4], [0]), ([0, 4], [-5]), ([1, 3], [128])):
        p = Problem(type, [1, 3, 1, 2], [200, 203, 201, 130], d=64, page=64, seed=7)
        for s in range(1, 4):
            p.table[s, :2] = p.table[0, :2]
        p.groups = groups
        check_attend(p)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_unwritten_slots_and_later_tokens_may_hold_anything(type):
    for fill in (math.nan, math.inf):
        for new, lens in (([1, 1, 1], [1, 50, 65]), ([9, 30], [20, 100])):
            p = Problem(type, new, lens, d=64, page=64, seed=8)
            p.written_only(fill)
            check_attend(p)
    # a NaN in the last token stays with the rows that see it
    p = Problem(type, [20, 150], [20, 170], d=64, page=16, rep=2, seed=9)
    for s in range(2):
        pg, sl = p.slots(s, p.lens[s] - 1)
        p.k[pg, sl], p.v[pg, sl, :, 3] = math.nan, math.inf
    cache, batch = p.on_gpu()
    out = paged.attend(cache, batch, p.gq, p.scale).double().cpu()
    for s in range(2):
        p.v[p.slots(s, p.lens[s] - 1)] = 0
        p.k[p.slots(s, p.lens[s] - 1)] = 0
    want, _, tol, _ = p.attend()
    seen = torch.ones(p.rows, dtype=torch.bool)
    for s in range(2):
        seen[p.starts[s + 1] - 1] = False
    near(out[seen], want[seen], tol[seen])
    assert torch.isnan(out[~seen]).all()


@pytest.mark.parametrize("type", ["f16", "bf16", "f32"])
def test_a_value_that_is_not_finite_stays_in_its_column_and_its_rows(type):
    p = Problem(type, [40], [140], d=64, page=16, rep=2, seed=10)
    pg, sl = p.slots(0, 120)
    p.v[pg, sl, 0, 5] = math.inf
    cache, batch = p.on_gpu()
    out = paged.attend(cache, batch, p.gq, p.scale).double().cpu()
    assert torch.isinf(out[20:, :2, 5]).all() and torch.isfinite(out[:20]).all() and torch.isfinite(out[20:, 2:]).all()
    rest = [c for c in range(64) if c != 5]
    assert torch.isfinite(out[:, :, rest]).all()


@pytest.mark.parametrize("type", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rep", [1, 4, 8, 9, 16])
@pytest.mark.parametrize("what", ["all", "shared", "lists"])
def test_infinite_values_of_few_rows_stay_in_their_column(what, rep, type):
    groups = ([0, 2], [64]) if what == "shared" else None
    p = Problem(type, [1, 1, 1], [140, 150, 31], d=64, page=16, G=2, rep=rep, seed=11, groups=groups)
    for s, at, c, x in ((0, 3, 5, math.inf), (0, 60, 6, -math.inf), (1, 149, 7, math.inf), (2, 30, 63, -math.inf), (0, 100, 9, math.nan)):
        pg, sl = p.slots(s, at)
        p.v[pg, sl, 1, c] = x
    check_attend(p, lists=torch.arange(p.max_pages, dtype=torch.int32).repeat(p.rows, p.G, 1) if what == "lists" else None)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_large_and_equal_scores(type):
    p = Problem(type, [1, 8], [300, 200], d=64, page=32, seed=11, key_scale=30.0)  # one key takes all
    check_attend(p)
    p = Problem(type, [1, 8], [300, 200], d=64, page=32, seed=12)
    p.k.zero_()  # the mean of the values
    check_attend(p)


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_pages_outside_the_pool_read_as_zeros_and_are_reported(type):
    p = Problem(type, [1, 3], [150, 100], d=64, page=16, seed=13, spare=4)
    cache, batch = p.on_gpu()
    table = p.table.clone()
    for bad in (-1, p.pages, 2 ** 31 - 1, -2 ** 31):
        table[0, 3], table[1, 5] = bad, bad
        batch.tensors[2].copy_(table)
        out = paged.attend(cache, batch, p.gq, p.scale)
        with pytest.raises(capi.XalmError):
            cache.check()
        cache.check()
        q = Problem(type, [1, 3], [150, 100], d=64, page=16, seed=13, spare=4)
        for s, j in ((0, 3), (1, 5)):
            q.k[q.table[s, j].long()] = 0
            q.v[q.table[s, j].long()] = 0
        want, _, tol, _ = q.attend()
        near(out, want, tol)


@pytest.mark.parametrize("type", ["f32", "f16"])
def test_arrays_that_do_not_fit_stay_in_bounds_and_are_reported(type):
    """Lengths beyond the table are cut; rows out of order and out of range belong to nobody."""
    p = Problem(type, [1, 2], [40, 60], d=64, page=16, seed=14)
    cache, batch = p.on_gpu()
    batch.tensors[1].copy_(torch.tensor([40, 10 ** 9], dtype=torch.int32))
    q = Problem(type, [1, 2], [40, 64], d=64, page=16, seed=14)
    q.table = p.table
    out = paged.attend(cache, batch, p.gq, p.scale)
    with pytest.raises(capi.XalmError):
        cache.check()
    want, _, tol, _ = q.attend()
    near(out, want, tol)
    for starts in ([0, 5, 3], [-4, 1, 3], [3, 2, 1], [0, 2 ** 31 - 1, 3], [0, 0, 2 ** 31 - 1]):
        batch.tensors[0].copy_(torch.tensor(starts, dtype=torch.int32))
        for lists in (None, torch.zeros(3, 2, 2, dtype=torch.int32, device="cuda")):
            out = paged.attend(cache, batch, p.gq, p.scale) if lists is None else paged.attend_selected(cache, batch, p.gq, lists, p.scale)
            torch.cuda.synchronize()
    batch.tensors[0].copy_(torch.tensor([0, 1, 3], dtype=torch.int32))
    batch.tensors[1].copy_(torch.tensor([-7, 1], dtype=torch.int32))  # the second has two new tokens and one in all: its first row sees nothing
    out = paged.attend(cache, batch, p.gq, p.scale)
    assert (out[:2] == 0).all() and (out[2] != 0).any()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_rows_of_a_wider_array(type):
    p = Problem(type, [1, 5, 1], [70, 80, 90], d=64, page=32, seed=15)
    cache, batch = p.on_gpu()
    want = paged.attend(cache, batch, p.gq, p.scale)
    wide = torch.randn(p.rows, p.H * 64 + 24, device="cuda").to(p.t)
    wide[:, 16:16 + p.H * 64] = p.gq.flatten(1)
    out = torch.zeros(p.rows, p.H * 64 + 40, device="cuda").to(p.t)
    paged.attend(cache, batch, wide[:, 16:16 + p.H * 64].view(p.rows, p.H, 64), p.scale, out=out[:, 8:8 + p.H * 64].view(p.rows, p.H, 64))
    assert torch.equal(out[:, 8:8 + p.H * 64].view_as(want), want) and (out[:, :8] == 0).all() and (out[:, 8 + p.H * 64:] == 0).all()


def test_pools_inside_larger_ones():
    for type in ("f32", "bf16"):
        p = Problem(type, [1, 5, 1], [70, 80, 90], d=64, page=16, G=2, seed=16)
        cache, batch = p.on_gpu()
        want = paged.attend(cache, batch, p.gq, p.scale)
        both = torch.full((p.pages, 16, 3, 2, 64), math.nan, device="cuda").to(p.t)  # layers, keys and values of a slot side by side
        k, v = both[:, :, 0], both[:, :, 2]
        k.copy_(p.gk)
        v.copy_(p.gv)
        assert torch.equal(paged.attend(paged.PagedCache(k, v), batch, p.gq, p.scale), want)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements: the pages at its end."""
    pages = (1 << 32) // (64 * 8 * 128) + 40
    k = torch.zeros(pages, 64, 8, 128, dtype=torch.float16, device="cuda")
    p = Problem("f16", [1, 1], [250, 100], G=8, rep=4, d=128, page=64, seed=17)
    at = torch.arange(p.pages) + pages - p.pages
    k[at.to("cuda")] = p.k.to("cuda")
    vals = p.v.to("cuda")
    v = k  # values where the keys are
    p.v = p.k
    p.on_gpu()
    cache = paged.PagedCache(k, v)
    table = torch.where(p.table >= 0, p.table + pages - p.pages, -1).to(torch.int32).to("cuda")
    batch = paged.Batch(torch.tensor(p.starts, dtype=torch.int32, device="cuda"), torch.tensor(p.lens, dtype=torch.int32, device="cuda"), table)
    want, _, tol, _ = p.attend()
    near(paged.attend(cache, batch, p.gq, p.scale), want, tol)
    kk = torch.randn(2, 8, 128, device="cuda").half()
    paged.append(cache, batch, kk, kk)
    for s in range(2):
        page = int(table[s, (p.lens[s] - 1) // 64])
        assert torch.equal(k[page, (p.lens[s] - 1) % 64], kk[s])
    del vals


# ---- selected pages --------------------------------------------------------------------------------------------------------------------------
def some_lists(p, n, seed, own=True, shuffle=False):
    g = torch.Generator().manual_seed(seed)
    out = torch.full((p.rows, p.G, n), -1, dtype=torch.int32)
    for r in range(p.rows):
        w = p.row(r)
        if w is None or w[1] < 0:
            continue
        last = w[1] // p.page
        for h in range(p.G):
            pick = torch.randperm(last + 1, generator=g)[:n].tolist()
            if own and last not in pick:
                pick[-1] = last
            pick = pick if shuffle else sorted(pick)
            out[r, h, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    return out


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("n", [1, 3, 8, 40])
def test_attend_selected(n, page, type):
    p = Problem(type, [1, 1, 6, 0, 1], [700, 300, 260, 33, 1], d=64, page=page, seed=18, pad_rows=2, offset=1)
    check_attend(p, some_lists(p, n, 1))
    check_attend(p, some_lists(p, n, 2, own=False))


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_lists_in_any_order_with_repetitions_and_strangers(type):
    p = Problem(type, [1, 1, 3], [700, 300, 260], d=64, page=16, seed=19)
    tidy = some_lists(p, 9, 3)
    want = check_attend(p, tidy)
    g = torch.Generator().manual_seed(4)
    messy = torch.cat([tidy, tidy[:, :, 2:5], torch.full((p.rows, p.G, 4), -1, dtype=torch.int32), torch.full((p.rows, p.G, 3), 44, dtype=torch.int32),
                       torch.full((p.rows, p.G, 2), 2 ** 31 - 1, dtype=torch.int32), torch.full((p.rows, p.G, 2), -2 ** 31, dtype=torch.int32)], dim=2)
    for r in range(p.rows):
        for h in range(p.G):
            messy[r, h] = messy[r, h, torch.randperm(messy.shape[2], generator=g)]
    messy[messy == 44] = 45  # beyond every row's own page
    out, lse = check_attend(p, messy)
    tol = p.attend(tidy)[2]
    near(out, want[0].double().cpu(), 2 * tol)
    none = torch.full((p.rows, p.G, 5), -1, dtype=torch.int32)
    check_attend(p, none)  # rows that see nothing
    long = torch.full((p.rows, p.G, 1024), -1, dtype=torch.int32)
    long[:, :, 1000:1009] = tidy
    check_attend(p, long)


@pytest.mark.parametrize("G,rep", [(1, 1), (2, 5), (1, 20), (3, 16)])
@pytest.mark.parametrize("d,dv", [(32, 32), (80, 64), (256, 256)])
def test_attend_selected_of_any_heads(G, rep, d, dv):
    p = Problem("f16", [1, 4], [400, 150], G=G, rep=rep, d=d, dv=dv, page=32, seed=20)
    check_attend(p, some_lists(p, 6, 5))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_selected_unwritten_slots(type):
    p = Problem(type, [1, 9], [77, 100], d=64, page=16, seed=21)
    p.written_only()
    p.v[p.slots(1, 99)] = math.nan  # only the last row sees it
    lists = some_lists(p, 4, 6)
    cache, batch = p.on_gpu()
    out = paged.attend_selected(cache, batch, p.gq, lists.to("cuda"), p.scale).double().cpu()
    assert torch.isnan(out[9]).all()
    p.v[p.slots(1, 99)] = 0
    want, _, tol, _ = p.attend(lists)
    near(out[:9], want[:9], tol[:9])


# ---- choosing pages ----------------------------------------------------------------------------------------------------------------------------
def with_means(p, seed=30):
    g = torch.Generator().manual_seed(seed)
    p.means = torch.randn(p.pages, p.G, p.d, generator=g).to(p.t)
    return p


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("top,first,recent", [(1, 0, 0), (4, 1, 1), (8, 0, 0), (8, 3, 4), (17, 2, 0), (64, 1, 1)])
def test_select(top, first, recent, type):
    p = with_means(Problem(type, [1, 1, 7, 0, 1, 1], [2000, 300, 260, 33, 1, 16], d=64, page=16, seed=22, pad_rows=2, offset=1))
    cache, batch = p.on_gpu()
    left = torch.full((p.rows, p.G, top), 7, dtype=torch.int32, device="cuda")
    got = paged.select(cache, batch, p.gq, top, first, recent, out=left).cpu()
    want = p.select(p.means, top, first, recent)
    inside = torch.tensor([p.row(n) is not None for n in range(p.rows)])
    assert torch.equal(got[inside], want[inside])
    assert (got[~inside] == 7).all()
    cache.check()


def test_select_equal_scores_and_scores_that_are_not_finite():
    p = with_means(Problem("f32", [1, 3], [2000, 1000], d=64, page=16, seed=23))
    p.means = torch.randint(-1, 2, p.means.shape, generator=p.gen).float()
    p.q = torch.randint(-1, 2, p.q.shape, generator=p.gen).float()
    p.q[:, :, 3:] = 0  # few different scores
    cache, batch = p.on_gpu()
    for top in (3, 10, 33, 100):
        assert torch.equal(paged.select(cache, batch, p.gq, top).cpu(), p.select(p.means, top, 1, 1))
    p.means[::3, 0, 0] = math.nan
    p.means[1::5, 1, 1] = math.inf
    p.means[2::5, :, 2] = -math.inf
    p.q[:, :, :3] = 1
    p.q[1] = -1
    cache, batch = p.on_gpu()
    for top in (3, 10, 33, 100):
        assert torch.equal(paged.select(cache, batch, p.gq, top).cpu(), p.select(p.means, top, 1, 1))
    p.means.zero_()
    cache, batch = p.on_gpu()
    got = paged.select(cache, batch, p.gq, 6, 2, 1).cpu()
    assert got[0, 0].tolist() == [0, 1, 2, 3, 123, 124]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,rep,d", [(1, 1, 8), (3, 5, 40), (2, 16, 256), (1, 71, 136)])
def test_select_of_any_heads(G, rep, d, type):
    p = with_means(Problem(type, [1, 3], [1500, 400], G=G, rep=rep, d=d, page=32, seed=24))
    cache, batch = p.on_gpu()
    assert torch.equal(paged.select(cache, batch, p.gq, 9, 1, 2).cpu(), p.select(p.means, 9, 1, 2))


@pytest.mark.parametrize("new", [[1, 1, 1], [0, 1, 0], [1, 37, 16], [2, 1, 100]])
@pytest.mark.parametrize("pages", [3, 100, 1500, 2100])
def test_select_of_steps_and_prompts(pages, new):
    """Every way of the rows: one to a block, and blocks of 16 and 8."""
    p = with_means(Problem("f16", new, [new[0] + 5, 900, 700], d=64, page=16, G=2, seed=26, pad_rows=1))
    width = p.table.shape[1]
    p.table = torch.cat([p.table.clamp_min(0)] * (pages // width + 1), dim=1)[:, :pages].contiguous()
    p.max_pages, p.lens = pages, [min(n, pages * 16) for n in (new[0] + 5, pages * 16, pages * 16 - 9)]
    for a in (p.means, -p.means):
        p.means = a
        cache, batch = p.on_gpu()
        got, want = paged.select(cache, batch, p.gq, 7).cpu(), p.select(p.means, 7, 1, 1)
        inside = torch.tensor([p.row(n) is not None for n in range(p.rows)])
        assert torch.equal(got[inside], want[inside])


@pytest.mark.parametrize("new", [[3, 1, 190], [160, 0, 33]])
@pytest.mark.parametrize("pages", [60, 512, 520])
def test_select_of_more_rows_than_multiprocessors(pages, new):
    """Blocks of 16 and of 8 rows."""
    p = with_means(Problem("bf16", new, [new[0] + 5, 900, 700], d=64, page=16, G=2, seed=51, pad_rows=1))
    width = p.table.shape[1]
    p.table = torch.cat([p.table.clamp_min(0)] * (pages // width + 1), dim=1)[:, :pages].contiguous()
    p.max_pages, p.lens = pages, [min(n, pages * 16) for n in (new[0] + 5, pages * 16, pages * 16 - 9)]
    for a in (p.means, -p.means):
        p.means = a
        cache, batch = p.on_gpu()
        got, want = paged.select(cache, batch, p.gq, 7).cpu(), p.select(p.means, 7, 1, 1)
        inside = torch.tensor([p.row(n) is not None for n in range(p.rows)])
        assert torch.equal(got[inside], want[inside])


def test_select_of_a_long_sequence():
    """20000 pages, most of them the same few of the pool."""
    p = with_means(Problem("bf16", [1, 2], [900, 900], d=128, page=16, G=2, seed=25))
    p.table = torch.cat([p.table[:, :50].repeat(1, 400), p.table[:, 50:57]], dim=1).contiguous()
    p.max_pages, p.lens = p.table.shape[1], [20000 * 16 + 100, 19000 * 16 + 1]
    cache, batch = p.on_gpu()
    got, want = paged.select(cache, batch, p.gq, 40).cpu(), p.select(p.means, 40, 1, 1)
    assert torch.equal(got, want)


# ---- appending -----------------------------------------------------------------------------------------------------------------------------------
def check_append(p, in_type, rot, neighbours, mag=1.0, means=True, queries=True):
    cast = TYPES[in_type]
    kn, vn, qn = p.normal(p.rows, p.G, p.d, dtype=cast), p.normal(p.rows, p.G, p.dv, dtype=cast), p.normal(p.rows, p.H, p.d, dtype=cast)
    freq = 10000.0 ** (-torch.arange(rot, dtype=torch.float32) / max(rot, 1))
    if means:
        p.means = p.normal(p.pages, p.G, p.d)
    cache, batch = p.on_gpu()
    q_out = torch.full((p.rows, p.H, p.d), 7.0, dtype=p.t, device="cuda")
    out = paged.append(cache, batch, kn.to("cuda"), vn.to("cuda"), q=qn.to("cuda") if queries else None, freq=freq.to("cuda") if rot else None, mag=mag, neighbours=neighbours,
                       q_out=q_out if queries else None)
    # turned entries: two products and a sum in fp32, sine and cosine each off by 2^-23 and the reduced angle by 2^-24 pi; then one rounding
    half = HALF[p.type]
    turned_err = 8 * F32 * abs(mag)
    tiny = 2.0 ** -25 if p.type == "f16" else 0.0

    def close(got, want, big):
        near(got, want, want.abs() * half + big * turned_err + tiny)

    kt, qt = p.turned(kn, rot, freq, mag, neighbours), p.turned(qn, rot, freq, mag, neighbours)
    size = lambda x: x.double().abs().amax(dim=-1, keepdim=True) * 2
    rows = [n for n in range(p.rows) if p.row(n) is not None]
    k, v = p.k.double().clone(), p.v.double().clone()
    big = torch.zeros_like(k)
    for n in rows:
        pg, sl = p.slots(*p.row(n))
        k[pg, sl], v[pg, sl], big[pg, sl] = kt[n], vn[n].double(), size(kn[n])
    untouched = big.amax(dim=(2, 3)) == 0
    assert torch.equal(p.gk.cpu()[untouched], p.k[untouched])
    close(p.gk, torch.where(big > 0, k, p.k.double()), big)
    near(p.gv, v, v.abs() * half + tiny)
    if queries:
        inside = torch.tensor([n in rows for n in range(p.rows)])
        close(out[inside.to("cuda")], qt[inside], size(qn)[inside].expand_as(qt[inside]))
        assert (out[~inside.to("cuda")] == 7.0).all()
    else:
        assert out is None
    if means:
        got, keys = cache.means.double().cpu(), p.gk.double().cpu()
        full = set()
        for n in rows:
            s, pos = p.row(n)
            if pos % p.page == p.page - 1:
                full.add(int(p.table[s, pos // p.page]))
        for page in range(p.pages):
            if page in full:
                want = keys[page].mean(dim=0)
                near(got[page], want, want.abs() * half + keys[page].abs().mean(dim=0) * (p.page + 2) * F32 + tiny)
            else:
                assert torch.equal(got[page], p.means[page].double())
    cache.check()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("in_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("neighbours", [False, True])
def test_append(in_type, type, neighbours):
    check_append(Problem(type, [1, 40, 0, 16, 1, 1], [33, 140, 7, 32, 64, 1], d=64, page=16, seed=31, pad_rows=2, offset=1), in_type, 32, neighbours)


@pytest.mark.parametrize("d,dv,rot", [(8, 16, 4), (40, 8, 20), (64, 64, 0), (64, 64, 5), (72, 80, 12), (128, 128, 32), (256, 256, 128), (136, 24, 67)])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("layout", ["position", "head"])
def test_append_of_any_head_size(d, dv, rot, neighbours, layout):
    check_append(Problem("bf16", [1, 70, 3], [64, 100, 131], G=3, rep=2, d=d, dv=dv, page=32, layout=layout, seed=32), "f32", rot, neighbours, mag=1.25)
    check_append(Problem("f32", [20], [64], G=1, rep=1, d=d, dv=dv, page=64, layout=layout, seed=33), "f32", rot, neighbours, queries=False)


def test_results_that_overlap_their_queries_are_refused():
    p = Problem("f16", [1, 4], [30, 40], d=64, page=16, seed=53)
    cache, batch = p.on_gpu()
    k = torch.zeros(p.rows, p.G, 64, dtype=p.t, device="cuda")
    rows, heads = p.rows, p.H
    room = torch.zeros(4 * rows * heads * 64, dtype=p.t, device="cuda")
    dense = lambda at: room[at:at + rows * heads * 64].view(rows, heads, 64)
    wide = room[:rows * 3 * heads * 64].view(rows, 3 * heads, 64)
    pages = torch.zeros(rows, p.G, 1, dtype=torch.int32, device="cuda")
    freq = torch.ones(12, device="cuda")
    one = heads * 64
    for q, out, meets in ((dense(0), dense(8), True), (dense(8), dense(0), True), (dense(0), dense(rows * one - 8), True), (dense(0), dense(rows * one), False), (dense(rows * one), dense(0), False),
                          (wide[:, :heads], wide[:, heads:2 * heads], False), (wide[:, heads:2 * heads], wide[:, :heads], False), (wide[:, :heads], wide[:, heads - 1:2 * heads - 1], True),
                          (wide[:, heads:2 * heads], wide[:, 1:heads + 1], True), (dense(0), wide[:, heads:2 * heads], True), (dense(0), dense(0), True)):
        for call in (lambda: paged.attend(cache, batch, q, 1.0, out=out), lambda: paged.attend_selected(cache, batch, q, pages, 1.0, out=out),
                     lambda: paged.append(cache, batch, k, k, q=q, freq=freq, q_out=out)):
            if meets:
                with pytest.raises(capi.XalmError, match="overlaps"):
                    call()
            else:
                call()
    cache.check()


@pytest.mark.parametrize("neighbours,rot", [(False, 32), (False, 8), (True, 5), (True, 32), (False, 0)])
def test_append_turns_queries_in_place(neighbours, rot):
    p = Problem("bf16", [1, 40, 700], [9, 90, 701], d=64, page=16, seed=52, pad_rows=2)
    cache, batch = p.on_gpu()
    k, v = (torch.randn(p.rows, p.G, 64, generator=p.gen).to(p.t).cuda() for _ in range(2))
    freq = torch.rand(rot, generator=p.gen).cuda() if rot else None
    want = paged.append(cache, batch, k, v, q=p.gq, freq=freq, neighbours=neighbours)
    inside = [n for n in range(p.rows) if p.row(n) is not None]
    wide = torch.zeros(p.rows, p.H + 3, 64, dtype=p.t, device="cuda")
    wide[:, :p.H] = p.gq
    q = wide[:, :p.H]
    assert paged.append(cache, batch, k, v, q=q, freq=freq, neighbours=neighbours, q_out=q) is q
    assert torch.equal(q[inside], want[inside]) and (wide[:, p.H:] == 0).all()


def test_append_far_positions():
    """Position 1000000: the angle in 32 bits would be 0.03 off."""
    p = Problem("f32", [1, 2], [100, 90], d=64, page=256, seed=34)
    p.table = p.table.repeat(1, 4000).contiguous()
    p.max_pages, p.lens = 4000, [1000001, 777778]
    check_append(p, "f32", 32, False)


def test_append_without_means_or_queries_and_of_one_token():
    check_append(Problem("f16", [1], [1], d=64, page=16, seed=35), "f16", 32, False, means=False)
    check_append(Problem("f16", [1], [16], d=64, page=16, seed=35), "f16", 32, False, queries=False)


def test_append_to_pages_outside_the_pool_is_left_out_and_reported():
    p = Problem("bf16", [1, 2, 40], [40, 60, 40], d=64, page=16, seed=36, spare=2)
    p.means = p.normal(p.pages, p.G, p.d)
    cache, batch = p.on_gpu()
    for bad in (-1, p.pages, 2 ** 31 - 1):
        table = p.table.clone()
        table[1, 3] = table[2, 1] = bad
        batch.tensors[2].copy_(table)
        before = p.gk.clone()
        rows = torch.randn(p.rows, 2, 64, device="cuda").to(p.t)
        paged.append(cache, batch, rows, rows)
        with pytest.raises(capi.XalmError):
            cache.check()
        for s in range(3):
            for j in range(4):
                page = int(p.table[s, j]) if j < p.max_pages else -1
                if (s, j) in ((1, 3), (2, 1)) and page >= 0:
                    assert torch.equal(p.gk[page], before[page])
        assert torch.equal(p.gk[int(p.table[0, 2]), 39 - 32], rows[0])


def test_append_arrays_that_do_not_fit():
    p = Problem("f32", [1, 2], [40, 60], d=64, page=16, seed=37)
    p.means = p.normal(p.pages, p.G, p.d)
    cache, batch = p.on_gpu()
    rows = torch.randn(3, 2, 64, device="cuda")
    for starts, lens in (([0, 5, 3], [40, 60]), ([-4, 1, 3], [40, 60]), ([3, 2, 1], [40, 60]), ([0, 2 ** 31 - 1, 3], [40, 60]), ([0, 1, 3], [40, 2 ** 31 - 1]), ([0, 1, 3], [0, 1]),
                         ([0, 1, 3], [-2 ** 31, 5])):
        batch.tensors[0].copy_(torch.tensor(starts, dtype=torch.int32))
        batch.tensors[1].copy_(torch.tensor(lens, dtype=torch.int32))
        paged.append(cache, batch, rows, rows)
        paged.select(cache, batch, p.gq, 3)
        with pytest.raises(capi.XalmError):
            cache.check()


# ---- together ------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_a_batch_served_step_by_step_equals_one_pass(type):
    """Three prompts behind a shared one, then single tokens, keys appended as they come: every step's rows against the restatement over all tokens."""
    page, G, rep, d, steps = 16, 2, 4, 64, 9
    lens = [64 + 30, 64 + 1, 64 + 77]
    final = [n + steps for n in lens]
    p = Problem(type, [1, 1, 1], final, G=G, rep=rep, d=d, page=page, seed=40, groups=([0, 3], [64]))
    p.means = torch.zeros(p.pages, G, d, dtype=p.t)
    freq = (10000.0 ** (-torch.arange(d // 2, dtype=torch.float32) / (d // 2))).to("cuda")
    cache, batch = p.on_gpu()
    starts, length, table = batch.tensors[:3]
    g = torch.Generator(device="cuda").manual_seed(5)
    rows = lambda n, h: torch.randn(n, h, d, generator=g, device="cuda").to(p.t)

    def step(new, now):
        starts.copy_(torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32))
        length.copy_(torch.tensor(now, dtype=torch.int32))
        n = sum(new)
        q = paged.append(cache, batch, rows(n, G), rows(n, G), q=rows(n, G * rep), freq=freq)
        dense = paged.attend(cache, batch, q, p.scale)
        lists = paged.select(cache, batch, q, 4)
        some = paged.attend_selected(cache, batch, q, lists, p.scale)
        cache.check()
        r = Problem(type, new, now, G=G, rep=rep, d=d, page=page, seed=0)
        r.table, r.max_pages, r.pages = p.table, p.max_pages, p.pages
        r.k, r.v, r.q = p.gk.cpu(), p.gv.cpu(), q.cpu()
        want, _, tol, _ = r.attend()
        near(dense, want, tol)
        assert torch.equal(lists.cpu(), r.select(cache.means.cpu(), 4, 1, 1))
        want, _, tol, _ = r.attend(lists.cpu())
        near(some, want, tol)

    only = paged.Batch(torch.tensor([0, 64], dtype=torch.int32, device="cuda"), torch.tensor([64], dtype=torch.int32, device="cuda"), table[:1])
    paged.append(cache, only, rows(64, G), rows(64, G), freq=freq)  # the shared prompt, once
    step([n - 64 for n in lens], lens)
    for i in range(steps):
        step([1, 1, 1], [n + i + 1 for n in lens])


def test_a_captured_step_follows_its_arrays_and_other_streams_do_not_meet():
    p = Problem("bf16", [1] * 5, [100, 200, 40, 5, 300], d=64, page=16, seed=41, groups=([0, 2], [64]))
    p.table[1, :4] = p.table[0, :4]
    p.means = p.normal(p.pages, p.G, p.d)
    cache, batch = p.on_gpu()
    length = batch.tensors[1]
    q = p.gq.clone()

    def serve():
        lists = paged.select(cache, batch, q, 3)
        return paged.attend(cache, batch, q, p.scale), paged.attend_selected(cache, batch, q, lists, p.scale)

    serve()
    side = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                outs = serve()
            graphs.append((gr, outs))
    for lens in ([100, 200, 40, 5, 300], [99, 150, 33, 1, 257], [70, 65, 1, 2, 3]):
        length.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        one, two = torch.cuda.Stream(), torch.cuda.Stream()
        for (gr, _), st in zip(graphs, (one, two)):
            with torch.cuda.stream(st):
                for _ in range(3):
                    gr.replay()
        with torch.cuda.stream(torch.cuda.Stream()):
            plain = serve()
        torch.cuda.synchronize()
        r = Problem("bf16", [1] * 5, lens, d=64, page=16, seed=41)
        r.table, r.k, r.v, r.q = p.table, p.k, p.v, p.q
        want, _, tol, _ = r.attend()
        near(plain[0], want, tol)
        for _, outs in graphs:
            assert torch.equal(outs[0], plain[0]) and torch.equal(outs[1], plain[1])


def test_calls_repeat_themselves_bit_for_bit():
    p = Problem("bf16", [1] * 30, [500 + 13 * i for i in range(30)], G=4, d=128, page=64, seed=42, groups=([0, 30], [448]))
    cache, batch = p.on_gpu()
    first = paged.attend(cache, batch, p.gq, p.scale, want_lse=True)
    for _ in range(5):
        again = paged.attend(cache, batch, p.gq, p.scale, want_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_many_rows_many_times(type):
    """Groups of all sizes around the tensor-core units' halves, long enough for several pieces to a CTA; every repetition the same, and no wait that gave up."""
    g = torch.Generator().manual_seed(44)
    sizes = [64, 33, 5, 31, 70]
    bounds = [0]
    for n in sizes:
        bounds.append(bounds[-1] + n)
    shared = [64 * n for n in (90, 31, 200, 64, 17)]
    lens = [shared[i] + int(torch.randint(1, 400, (1,), generator=g)) for i, n in enumerate(sizes) for _ in range(n)]
    B, G, d, page = bounds[-1], 4, 128, 64
    width, pages = max(-(-n // page) for n in lens), 2000
    gg = torch.Generator(device="cuda").manual_seed(45)
    k, v = (torch.randn(pages, page, G, d, generator=gg, device="cuda").to(TYPES[type]) for _ in range(2))
    table = torch.randint(0, pages, (B, width), generator=gg, device="cuda", dtype=torch.int32)
    for i in range(len(sizes)):
        table[bounds[i]:bounds[i + 1], :shared[i] // page] = table[bounds[i], :shared[i] // page]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cache = paged.PagedCache(k, v)
    q = torch.randn(B, 4 * G, d, generator=gg, device="cuda").to(TYPES[type])
    alone = paged.Batch(i32(range(B + 1)), i32(lens), table)
    together = paged.Batch(i32(range(B + 1)), i32(lens), table, groups=i32(bounds), shared=i32(shared))
    want, want_lse = paged.attend(cache, alone, q, d ** -0.5, want_lse=True)
    first, first_lse = paged.attend(cache, together, q, d ** -0.5, want_lse=True)
    cache.check()
    # two ways of the same sums: each rounds every probability once and the result once
    spread = 2 * HALF[type] * float(v.abs().max())
    assert float((first.float() - want.float()).abs().max()) < spread and float((first_lse - want_lse).abs().max()) < 1e-4
    for _ in range(300):
        out, lse = paged.attend(cache, together, q, d ** -0.5, want_lse=True)
        assert torch.equal(out, first) and torch.equal(lse, first_lse)
    cache.check()


def test_a_workspace_too_small_is_refused():
    import ctypes as C
    p = Problem("bf16", [1], [100], d=64, page=16, seed=43)
    cache, batch = p.on_gpu()
    batch.c.rows = 1
    need = C.c_size_t(0)
    L = capi.lib()
    capi.check(L.xalm_cuda_paged_workspace(cache.p, batch.p, p.H, 0, C.byref(need)))
    work = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(p.gq)
    args = lambda n: (cache.p, batch.p, p.gq.data_ptr(), p.H * 64, p.H, p.scale, out.data_ptr(), p.H * 64, None, work.data_ptr(), n, None)
    assert L.xalm_cuda_paged_attend(*args(need.value - 1)) == 1
    assert L.xalm_cuda_paged_attend(*args(need.value)) == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits,words", [(1, "names a page"), (2, "do not fit"), (4, "gave up a wait"), (5, "names a page outside the pool and a kernel gave up")])
def test_what_kernels_report_is_raised_once(bits, words):
    cache, _ = Problem("bf16", [1], [20], d=64, page=16, seed=54).on_gpu()
    cache.status.fill_(bits)
    with pytest.raises(capi.XalmError, match=words):
        cache.check()
    cache.check()
