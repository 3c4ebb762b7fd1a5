"""The paged cache's operators where a number, a length or a caller comes to the edge of what they take, against the restatement in 64 bits (paged_ref.py, which derives the tolerances)."""
import math

import pytest
import torch

from paged_ref import F32, HALF, Problem
from test_gpu_paged import near
from xalm_b200 import capi, paged

pytestmark = pytest.mark.gpu


# ---- probabilities far below a row's largest one ---------------------------------------------------------------------------------------------
def sink(type, new, lens, below, rep, page=64, groups=None, wave=0.0):
    """Key 0 of every sequence has a score `below` above all others' and a value of 0; the others' values are 1, their scores equal, or `wave` apart."""
    p = Problem(type, new, lens, G=1, rep=rep, d=64, page=page, seed=60, groups=groups)
    p.q.zero_()
    p.q[:, :, 0], p.q[:, :, 1] = 4.0, 1.0
    p.k.zero_()
    if wave:
        p.k[..., 1] = (torch.rand(p.k.shape[:-1], generator=p.gen) * 2 - 1).mul_(wave * 8).to(p.t)
    p.v.fill_(1.0)
    for s in range(len(new)):
        at = p.slots(s, 0)
        p.k[at], p.v[at] = 0.0, 0.0
        p.k[at + (0, 0)] = 2.0 * below  # times 4, times the scale 1 / 8
    return p


def looked_at(p, n=9):
    rows = [r for r in range(p.rows) if p.row(r) is not None]
    return sorted(set(rows[:: max(1, len(rows) // n)] + rows[-1:]))


def check(p, lists=None, round_p=True):
    cache, batch = p.on_gpu()
    some = looked_at(p)
    args = dict(want_lse=True)
    out, lse = paged.attend(cache, batch, p.gq, p.scale, **args) if lists is None else paged.attend_selected(cache, batch, p.gq, lists.to("cuda"), p.scale, **args)
    cache.check()
    want, want_lse, tol, tol_lse = p.attend(lists, round_p=round_p, only=some)
    near(out[some], want[some], tol[some], "out")
    near(lse[some], want_lse[some], tol_lse[some], "lse")


# tokens and query heads to a kv head: 1, 8, 9, 16 and 256 rows
ROWS = {1: (1, 1), 8: (1, 8), 9: (1, 9), 16: (1, 16), 256: (64, 4)}


@pytest.mark.parametrize("type", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("n,below", [(4096, 12), (8192, 20), (32768, 14), (32768, 20)])
@pytest.mark.parametrize("where", ["own", "shared", "lists"])
def test_many_small_probabilities_beside_a_large_one(where, n, below, rows, type):
    tokens, rep = ROWS[rows]
    if where == "shared":  # the rows are those of two or more sequences
        if rows == 9:
            p = sink(type, [1] * 9, [n + 64 + i for i in range(9)], below, 1, groups=([0, 9], [n]))
        elif rows == 1:
            p = sink(type, [1, 0], [n + 64, n], below, 1, groups=([0, 2], [n]))
        elif rows == 256:
            p = sink(type, [1] * 16, [n + 1] * 16, below, 16, groups=([0, 16], [n]))
        else:
            p = sink(type, [1, 1], [n + 64, n + 7], below, rep // 2, groups=([0, 2], [n]))
        return check(p)
    if where == "lists" and rows == 256:
        tokens = 3  # a unit has one token's rows there
    p = sink(type, [tokens], [n], below, rep)
    check(p, torch.arange(p.max_pages, dtype=torch.int32).repeat(p.rows, p.G, 1) if where == "lists" else None)


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 4, 8, 9, 16])
@pytest.mark.parametrize("where", ["own", "lists", "shared", "wide"])
def test_probabilities_of_few_rows_keep_more_bits_than_their_type(where, rows, type):
    """The tolerance has no rounding of the probabilities in it, and the results are near 0 beside the values that they are sums of."""
    d = 256 if where == "wide" else 64
    groups = ([0, 2], [192]) if where == "shared" else None
    p = Problem(type, [1, 1], [260, 290], G=2, rep=rows, d=d, page=64, seed=61, groups=groups)
    p.v = (p.v.float() + 3 * torch.sign(p.v.float())).to(p.t)  # results near 0 from values that are not
    check(p, torch.arange(p.max_pages, dtype=torch.int32).repeat(p.rows, p.G, 1) if where == "lists" else None, round_p=False)


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("rep", [1, 8, 9, 16])
@pytest.mark.parametrize("below", [5, 20, 40, 60])
def test_an_infinite_value_of_a_small_probability_gives_an_infinity(below, rep, type):
    """Also where the probability is far below what fp16 holds beside the row's largest."""
    for bad in (math.inf, -math.inf):
        p = sink(type, [1], [300], below, rep)
        p.v[p.slots(0, 200) + (0, 7)] = bad
        cache, batch = p.on_gpu()
        out = paged.attend(cache, batch, p.gq, p.scale)
        assert (out[:, :, 7] == bad).all() and torch.isfinite(out[:, :, :7]).all() and torch.isfinite(out[:, :, 8:]).all()


# ---- calls from several threads ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_calls_of_different_sizes_in_several_threads(type):
    """Each thread has a batch of its own number of sequences, length of lists and width of tables, so that no two calls want the same shared memory."""
    from concurrent.futures import ThreadPoolExecutor
    rounds, jobs = 150, []
    for seqs, top, width in ((3, 4, 900), (400, 40, 1500), (1500, 200, 3000), (2500, 600, 700)):
        p = Problem(type, [1] * seqs, [i % 200 + 1 for i in range(seqs)], G=2, rep=3, d=64, page=16, seed=62)
        p.means = p.normal(p.pages, p.G, p.d)
        p.table = torch.cat([p.table, torch.full((seqs, width - p.max_pages), -1, dtype=torch.int32)], dim=1)
        p.max_pages = width
        cache, batch = p.on_gpu()

        def serve(cache=cache, batch=batch, q=p.gq, top=top, scale=p.scale):
            lists = paged.select(cache, batch, q, top)
            return lists, paged.attend(cache, batch, q, scale), paged.attend_selected(cache, batch, q, lists, scale)

        jobs.append((serve, serve(), cache))
    torch.cuda.synchronize()

    def thread(job):
        serve, want, _ = job
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for n in range(rounds):
                got = serve()
                stream.synchronize()
                assert all(torch.equal(x, y) for x, y in zip(got, want)), n
        return rounds

    with ThreadPoolExecutor(len(jobs)) as pool:
        assert list(pool.map(thread, jobs)) == [rounds] * len(jobs)
    for *_, cache in jobs:
        cache.check()


def test_no_call_takes_shared_memory_from_another():
    """The same kernel launched from two threads with more and with less shared memory, as fast as the calls go."""
    from concurrent.futures import ThreadPoolExecutor
    L, jobs = capi.lib(), []
    for width in (24000, 7000):
        p = Problem("bf16", [1], [40], G=1, rep=1, d=64, page=16, seed=63, max_pages=width)
        p.means = p.normal(p.pages, p.G, p.d)
        cache, batch = p.on_gpu()
        batch.c.rows = 1
        jobs.append((cache, batch, p.gq, torch.empty(1, 1, 4, dtype=torch.int32, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()

    def thread(job):
        cache, batch, q, out, stream = job
        args = cache.p, batch.p, q.data_ptr(), 64, 1, 4, 1, 1, out.data_ptr(), stream.cuda_stream
        refused = sum(L.xalm_cuda_paged_select(*args) != 0 for _ in range(20000))
        stream.synchronize()
        return refused

    with ThreadPoolExecutor(2) as pool:
        assert list(pool.map(thread, jobs)) == [0, 0]
    for cache, _, _, out, _ in jobs:
        assert out.flatten().tolist() == [0, 1, 2, -1]
        cache.check()


# ---- what kernels report -----------------------------------------------------------------------------------------------------------------------
def test_check_waits_for_every_stream():
    p = Problem("bf16", [1], [20], d=64, page=16, seed=64)
    cache, batch = p.on_gpu()
    batch.tensors[2][0, 1] = p.pages
    rows = torch.zeros(1, p.G, 64, dtype=p.t, device="cuda")
    paged.append(cache, batch, rows, rows)  # the kernel is in memory before it has to run late
    with pytest.raises(capi.XalmError, match="names a page"):
        cache.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # a tenth of a second
        paged.append(cache, batch, rows, rows)
    with pytest.raises(capi.XalmError, match="names a page"):
        cache.check()
    cache.check()


def test_no_report_is_lost_while_others_are_read():
    """One thread keeps reading the word, another keeps reporting: every report is in what was read or still there."""
    import threading
    p = Problem("bf16", [1], [20], d=64, page=16, seed=65)
    cache, batch = p.on_gpu()
    batch.tensors[2][0, 1] = p.pages
    rows = torch.zeros(1, p.G, 64, dtype=p.t, device="cuda")
    done, raised = threading.Event(), []

    def read():
        with torch.cuda.stream(torch.cuda.Stream()):
            while not done.is_set():
                try:
                    cache.check()
                except capi.XalmError:
                    raised.append(1)

    torch.cuda.synchronize()
    reader = threading.Thread(target=read)
    reader.start()
    seen = 0
    for n in range(300):
        before = len(raised)
        paged.append(cache, batch, rows, rows)
        for _ in range(2000):  # a report appears in at most a check that is under way and the one after it
            if len(raised) > before:
                break
            done.wait(0.001)
        seen += len(raised) > before
        if seen <= n:
            break
    done.set()
    reader.join()
    assert seen == 300


# ---- lengths beyond the table ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,over", [([1, 1], [1, 0]), ([40, 3], [2, 0]), ([20, 700], [0, 650]), ([5, 2], [5, 2 ** 31 - 1 - 64])])
def test_append_writes_nothing_behind_the_table_and_no_other_slots_instead(new, over, type):
    """Tokens that the table has no page for are reported and left out; the others go where they belong, and every query is turned by its own position."""
    page, cap = 16, 64
    p = Problem(type, new, [cap, cap], d=64, page=page, seed=66)
    p.means = p.normal(p.pages, p.G, p.d)
    cache, batch = p.on_gpu()
    lens = [cap + x for x in over]
    batch.tensors[1].copy_(torch.tensor(lens, dtype=torch.int32))
    kn, vn, qn = p.normal(p.rows, p.G, 64), p.normal(p.rows, p.G, 64), p.normal(p.rows, p.H, 64)
    freq = torch.zeros(32)  # no turn but for the first pair's
    freq[0] = 2.0 ** -9
    out = paged.append(cache, batch, kn.cuda(), vn.cuda(), q=qn.cuda(), freq=freq.cuda())
    with pytest.raises(capi.XalmError, match="do not fit"):
        cache.check()
    cache.check()
    k, v, full = p.k.clone(), p.v.clone(), set()
    angle = torch.zeros(p.rows, dtype=torch.float64)
    for s in range(2):
        for i in range(new[s]):
            pos = lens[s] - new[s] + i
            angle[p.starts[s] + i] = pos * 2.0 ** -9
            if pos < cap:
                at = p.slots(s, pos)
                k[at], v[at] = kn[p.starts[s] + i], vn[p.starts[s] + i]
                k[at + (slice(None), 0)] = math.nan  # turned: looked at below only
                k[at + (slice(None), 32)] = math.nan
                if pos % page == page - 1:
                    full.add(int(p.table[s, pos // page]))
    got, same = p.gk.cpu(), ~torch.isnan(k)
    assert torch.equal(got[same], k[same]) and torch.equal(p.gv.cpu(), v)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    x, y = qn[:, :, 0].double(), qn[:, :, 32].double()
    want = torch.stack([x * c - y * s, y * c + x * s], dim=-1)
    near(out[:, :, [0, 32]], want, want.abs() * HALF[type] + 8 * F32 * (x.abs() + y.abs())[..., None] + 2.0 ** -25)
    means = cache.means.cpu()
    for n in range(p.pages):
        if n in full:
            exact = got[n].double().mean(dim=0)
            near(means[n], exact, exact.abs() * HALF[type] + (page + 2) * F32 * got[n].double().abs().mean(dim=0) + 2.0 ** -25)
        else:
            assert torch.equal(means[n], p.means[n])


# ---- scores at the ends of fp32 ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("new,pages", [([1, 1], 40), ([1, 1], 700), ([150, 3], 40), ([150, 3], 300)])
def test_select_where_sums_leave_the_range_of_fp32(new, pages, type):
    """Sums that overflow on their way to an ordinary number, and numbers whose products fp32 rounds to 0, are in the order of 64 bits."""
    p = Problem(type, new, [new[0] + 600, new[1] + 550], G=2, rep=1, d=64, page=16, seed=67)
    p.table = torch.cat([p.table.clamp_min(0)] * (pages // p.max_pages + 1), dim=1)[:, :pages].contiguous()
    p.max_pages = pages
    p.lens = [pages * 16, pages * 16 - 9]

    def same(means, q, tops):
        p.means, p.q = means.to(p.t), q.to(p.t)
        cache, batch = p.on_gpu()
        for top in tops:
            assert torch.equal(paged.select(cache, batch, p.gq, top).cpu(), p.select(p.means, top, 1, 1))

    rand = lambda *s: torch.randn(*s, generator=p.gen)
    means, q = rand(p.pages, p.G, 64), torch.ones(p.rows, p.H, 64)
    means[::7], means[3::7] = 0.0, 0.0  # scores of 0, whatever the order of the sum
    means[::7, :, :4] = torch.tensor([2.0e38, 2.0e38, -2.0e38, -2.0e38])
    means[3::7, :, 8:12] = torch.tensor([-2.0e38, -2.0e38, 2.0e38, 2.0e38])
    same(means, q, (3, 20))
    same(means, -q, (9,))
    # 2^-75 times 2^-80, and sums just above the smallest number
    same(rand(p.pages, p.G, 64) * 2.0 ** -75, rand(p.rows, p.H, 64) * 2.0 ** -80, (9,))
    same(rand(p.pages, p.G, 64) * 2.0 ** -70, rand(p.rows, p.H, 64) * 2.0 ** -76, (9,))


# ---- arrays that lie in one another ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_results_that_overlap_what_a_call_is_given_are_refused(type):
    """Nothing is launched for them; rows side by side in one array are taken."""
    p = Problem(type, [1, 4], [30, 40], d=64, page=16, seed=68, groups=([0, 2], [16]))
    p.means = p.normal(p.pages, p.G, p.d)
    cache, batch = p.on_gpu()
    L, n, H, G, row = capi.lib(), p.rows, p.H, p.G, p.H * 64
    new = lambda *s, dtype=p.t: torch.zeros(*s, dtype=dtype, device="cuda")
    k, v, q, out, freq, lse, lists = new(n, G, 64), new(n, G, 64), new(n, H, 64), new(n, H, 64), new(32, dtype=torch.float32), new(n, H, dtype=torch.float32), new(n, G, 4, dtype=torch.int32)
    work = new(1 << 27, dtype=torch.uint8)
    bp = batch.of(n)[0]
    at = lambda t: t.data_ptr()

    def append(q_out):
        return L.xalm_cuda_paged_append(cache.p, bp, at(k), G * 64, at(v), G * 64, at(q), row, H, cache.c.type, q_out, row, at(freq), 32, 1.0, 0, None)

    def attend(out, lse, work):
        return L.xalm_cuda_paged_attend(cache.p, bp, at(q), row, H, 0.1, out, row, lse, work, 1 << 26, None)

    def selected(out, lse, work):
        return L.xalm_cuda_paged_attend_selected(cache.p, bp, at(q), row, H, at(lists), 4, 0.1, out, row, lse, work, 1 << 26, None)

    def select(out):
        return L.xalm_cuda_paged_select(cache.p, bp, at(q), row, H, 4, 1, 1, out, None)

    fixed = [p.gk, p.gv, cache.means, cache.status, *batch.tensors]
    for x in fixed + [q]:
        low, end = at(x) // 256 * 256, at(x) + (x.numel() - 1) * x.element_size()
        for here in (at(x), low, end // 16 * 16):
            calls = [attend(here, at(lse), at(work)), selected(here, at(lse), at(work)), attend(at(out), here, at(work)), selected(at(out), here, at(work)), select(here)]
            assert calls == [1] * 5 and (x is q or append(here) == 1), (x.shape, calls)
        assert attend(at(out), at(lse), low) == 1 and selected(at(out), at(lse), low) == 1
    for here in (at(k), at(v) + 16, at(freq)):
        assert append(here) == 1
    assert selected(at(lists), at(lse), at(work)) == 1 and selected(at(out), at(lists), at(work)) == 1 and attend(at(out), at(out), at(work)) == 1
    assert attend(at(work), at(lse), at(work)) == 1 and attend(at(out), at(work) + 4096, at(work)) == 1
    assert b"overlaps" in L.xalm_cuda_last_error()
    torch.cuda.synchronize()
    assert torch.equal(p.gk.cpu(), p.k) and torch.equal(p.gv.cpu(), p.v)
    assert append(at(out)) == attend(at(out), at(lse), at(work)) == select(at(lists)) == selected(at(out), at(lse), at(work)) == 0
    # one projection's rows, queries turned where they are
    qkv = torch.randn(n, H + 2 * G, 64, generator=p.gen).to(p.t).cuda()
    qs, ks, vs = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    want = paged.append(cache, batch, ks.clone(), vs.clone(), q=qs.clone(), freq=freq)
    assert torch.equal(paged.append(cache, batch, ks, vs, q=qs, freq=freq, q_out=qs), want)
    with pytest.raises(capi.XalmError, match="overlaps k or v"):
        paged.append(cache, batch, ks, vs, q=q, freq=freq, q_out=qkv[:, 1:H + 1])
    cache.check()


# ---- idle places of a group --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rep", [2, 20])
@pytest.mark.parametrize("new,lens", [([0, 1, 0, 1, 1, 0], [0, 200, 0, 131, 300, 0]), ([0, 0, 3, 0, 2], [0, 0, 190, 0, 140]), ([1, 0, 0, 0, 1], [129, 0, 7, 0, 140]), ([0, 1, 0], [0, 150, 0]),
                                      ([0, 0, 0], [0, 0, 0])])
def test_idle_places_neither_end_the_sharing_nor_lend_their_pages(new, lens, rep, type):
    p = Problem(type, new, lens, G=2, rep=rep, d=64, page=16, seed=69, pad_rows=1, offset=1)
    live = [s for s in range(len(new)) if new[s]]
    for s in live:
        p.table[s, :8] = p.table[live[0], :8]
    p.groups = [0, len(new)], [128]
    cache, batch = p.on_gpu()
    inside = [r for r in range(p.rows) if p.row(r) is not None]
    out, lse = paged.attend(cache, batch, p.gq, p.scale, want_lse=True)
    cache.check()
    want, want_lse, tol, tol_lse = p.attend()
    near(out[inside], want[inside], tol[inside], "out")
    near(lse[inside], want_lse[inside], tol_lse[inside], "lse")
    if len(live) < 2:
        return
    # What is read once is read by the first live sequence's table: where the others' name other pages, and the first's are what counts, the common part was shared
    table = p.table.clone()
    for s in live[1:]:
        table[s, :8] = table[live[0], 8:9]
    batch.tensors[2].copy_(table)
    again, _ = paged.attend(cache, batch, p.gq, p.scale, want_lse=True)
    cache.check()
    assert torch.equal(again[inside], out[inside])


# ---- values that are not finite ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("below", [5, 20, 40, 60])
@pytest.mark.parametrize("where", ["own", "shared", "divided", "long"])
def test_infinite_values_of_many_rows_stay_in_their_columns(where, below, type):
    """Beside probabilities far below what fp16 holds too; of both signs and a NaN in one column; seen by all rows, and by the later ones only."""
    if where in ("shared", "long"):
        n = 512 if where == "shared" else 32768  # a tile to a block, several
        p = sink(type, [1] * 16, [n + 88 + i for i in range(16)], below, 16, groups=([0, 16], [n]))
        places = [(0, 100, 7, math.inf), (0, 101, 8, math.inf), (0, 300, 8, -math.inf), (0, 5, 63, math.nan), (3, n + 88, 9, -math.inf)]
    else:
        n = 70 if where == "own" else 700
        p = sink(type, [n], [n + 500], below, 4)
        places = [(0, 100, 7, math.inf), (0, 101, 8, math.inf), (0, 520, 8, -math.inf), (0, 5, 63, math.nan), (0, 515, 9, -math.inf), (0, 560, 10, math.inf)]
    for s, at, c, x in places:
        p.v[p.slots(s, at) + (0, c)] = x
    cache, batch = p.on_gpu()
    out, lse = paged.attend(cache, batch, p.gq, p.scale, want_lse=True)
    cache.check()
    some = list(range(p.rows)) if where != "divided" else looked_at(p, 40) + [14, 15, 16, 18, 19, 20, 21, 59, 60, 61]
    want, want_lse, tol, tol_lse = p.attend(only=some)
    near(out[some], want[some], tol[some], "out")
    near(lse[some], want_lse[some], tol_lse[some], "lse")


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("rep", [1, 4])
def test_a_query_that_is_not_finite_makes_no_other_row_wait(rep, type):
    """Rows of NaN are what they are: no row is done again key by key."""
    p = Problem(type, [2000, 9], [3000, 2000], G=2, rep=rep, d=64, page=64, seed=70)
    cache, batch = p.on_gpu()
    bad = p.gq.clone()
    bad[5:2005:100] = math.nan

    def time(q):
        best = math.inf
        for _ in range(5):
            ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            ends[0].record()
            out = paged.attend(cache, batch, q, p.scale)
            ends[1].record()
            torch.cuda.synchronize()
            best = min(best, ends[0].elapsed_time(ends[1]))
        return best, out

    plain, want = time(p.gq)
    spoilt, got = time(bad)
    assert torch.isnan(got[5:2005:100]).all()
    fine = torch.ones(p.rows, dtype=torch.bool)
    fine[5:2005:100] = False
    assert torch.equal(got[fine], want[fine])
    assert spoilt < 5 * plain, (spoilt, plain)


# ---- workspaces --------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seqs,groups,most", [(128, 2, 80), (1000, 3, 400), (4000, 1, 1500)])
def test_a_batch_of_single_tokens_needs_no_room_for_long_ones(seqs, groups, most):
    """In MiB; 32 heads of 128 over 8, some sequences of which share pages."""
    import ctypes as C
    k = torch.zeros(4, 64, 8, 128, dtype=torch.bfloat16, device="cuda")
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    cache, batch = paged.PagedCache(k, k), paged.Batch(i(seqs + 1), i(seqs), i(seqs, 100), i(groups + 1), i(groups))
    need = C.c_size_t(0)
    capi.check(capi.lib().xalm_cuda_paged_workspace(cache.p, batch.of(seqs)[0], 32, 0, C.byref(need)))
    assert need.value < most << 20, need.value / 2 ** 20


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("new,rep,groups", [([1] * 40, 17, ([0, 20, 40], [64, 128])), ([1] * 40, 17, ([0, 40], [64])), ([17] * 30, 1, ([0, 30], [64])), ([1, 0, 17, 2, 0, 33] * 6, 1, ([0, 18, 36], [64, 64])),
                                            ([9] * 20, 2, ([2, 4, 6, 8, 19], [64, 64, 128, 64])), ([257, 1, 255, 256], 1, ([0, 4], [128]))])
def test_as_many_units_as_there_is_room_for(new, rep, groups, type):
    """Segments of just more rows than the short ones' kernel takes, each a unit of its own, in the smallest workspace."""
    lens = [190 + n + 7 * i % 40 for i, n in enumerate(new)]
    p = Problem(type, new, lens, G=3, rep=rep, d=64, page=64, seed=71, groups=groups)
    cache, batch = p.on_gpu()
    out, lse = paged.attend(cache, batch, p.gq, p.scale, want_lse=True)
    cache.check()
    some = looked_at(p, 60)
    want, want_lse, tol, tol_lse = p.attend(only=some)
    near(out[some], want[some], tol[some], "out")
    near(lse[some], want_lse[some], tol_lse[some], "lse")


# ---- scores of millions ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 8, 16, 256])
def test_scores_that_fp32_holds_to_half_a_unit_give_finite_results(rows, type):
    """Scores of some 5 million with differences that fp32 rounds: what a probability is may be off by much, but it is no infinity, and sums to one."""
    tokens, rep = ROWS[rows]
    n = 65536  # several tiles to a block
    for step in (8, 16, 20):
        p = sink(type, [tokens], [n], 0, rep)
        p.q[:, :, 0] = 2048.0
        p.q[:, :, 0] += (torch.arange(p.rows * p.H) % 97).view(p.rows, p.H).to(p.t) * (2.0 if type != "bf16" else 16.0)
        p.k[..., 0], p.v = 20000.0, torch.ones_like(p.v)
        at = torch.arange(n)
        p.k[p.slots(0, at) + (0, 1)] = (step * (at // 128 % 2)).to(p.t)  # the larger ones come after the first that a row sees
        cache, batch = p.on_gpu()
        out = paged.attend(cache, batch, p.gq, p.scale)
        assert torch.isfinite(out).all() and float((out - 1).abs().max()) < 0.5, step
        if rows < 256:
            out = paged.attend_selected(cache, batch, p.gq, torch.arange(p.max_pages, dtype=torch.int32).repeat(p.rows, 1, 1).cuda(), p.scale)
            assert torch.isfinite(out).all() and float((out - 1).abs().max()) < 0.5, step


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("new,lens,bad", [([1000, 750, 1], [2000, 1500, 1000], 1600), ([1500, 20, 1], [3000, 1500, 1000], 2983), ([3, 2], [40000, 300], 39999), ([300, 300], [30000, 300], 29850)])
def test_rows_that_take_long_end_no_wait(new, lens, bad, type):
    """A token of NaN inside a prompt: the rows before it are done again key by key, and the warps that wait for that meanwhile do not give up."""
    p = Problem(type, new, lens, G=8 if lens[0] < 10000 else 1, rep=4, d=128, page=64, seed=72)
    at = p.slots(0, bad)
    p.k[at], p.v[at] = math.nan, math.nan
    cache, batch = p.on_gpu()
    out = paged.attend(cache, batch, p.gq, p.scale)
    cache.check()
    first = bad - (lens[0] - new[0])  # row of the token
    assert torch.isnan(out[first:new[0]]).all() and torch.isfinite(out[:first]).all() and torch.isfinite(out[new[0]:]).all()
    p.k[at], p.v[at] = 0.0, 0.0
    some = sorted({max(first - i, 0) for i in (1, 2, 3, 17, 33, 50, 64, 65, 130)} - {first}) + [p.rows - 1]
    want, _, tol, _ = p.attend(only=some)
    near(out[some], want[some], tol[some])
