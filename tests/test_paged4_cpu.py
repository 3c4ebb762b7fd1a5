"""The 4-bit paged cache and the verification of drafts without a GPU: the host's checks refuse what does not fit before anything is launched, and the restatement agrees with itself."""
import ctypes as C
import math

import pytest
import torch

from paged4_ref import BLOCKS, Problem4, pack, place, quantise, unpack, values, verify
from xalm_b200 import capi, paged
from xalm_b200 import types as T

A = 1 << 20  # an address at a 16-byte boundary that no check reads from
RUN = 16 * 18 * 4


def cache(**over):
    c = dict(device=0, pages=4, page_size=16, kv_heads=2, dim=64, vdim=64, pool=A, page=2 * RUN, head=RUN, status=0)
    c.update(over)
    return paged._Cache4(**c)


def batch(**over):
    b = dict(rows=3, seqs=2, max_pages=5, groups=0, starts=A, lens=A, table=A, table_row=5, group_bounds=0, group_shared=0)
    b.update(over)
    return paged._Batch(**b)


def calls(c, b, q=A, q_row=512, heads=8, out=4 * A, out_row=512, scale=0.1, k=2 * A, k_row=128, v=3 * A, v_row=128, type=T.BF16.id, freq=A, rot=32, work=8 * A, room=1 << 40, lse=None):
    L, p, w = capi.lib(), C.byref(c), C.byref(b)
    return {"append": lambda: L.xalm_cuda_paged4_append(p, w, k, k_row, v, v_row, q, q_row, heads, type, out, out_row, freq, rot, 1.0, 0, None),
            "attend": lambda: L.xalm_cuda_paged4_attend(p, w, q, q_row, heads, type, scale, out, out_row, lse, work, room, None),
            "read": lambda: L.xalm_cuda_paged4_read(p, w, type, k, k_row, v, v_row, None)}


ALL = ["append", "attend", "read"]


@pytest.mark.parametrize("bad", [dict(pages=0), dict(page_size=8), dict(page_size=24), dict(page_size=512), dict(kv_heads=0), dict(kv_heads=65536), dict(dim=0), dict(dim=12), dict(dim=264),
                                 dict(vdim=4), dict(vdim=-8), dict(pool=0), dict(pool=A + 8), dict(page=RUN), dict(head=RUN - 16), dict(head=RUN + 8), dict(page=2 * RUN + 4), dict(page=0),
                                 dict(head=-RUN), dict(page=1 << 41), dict(dim=128), dict(page_size=32), dict(status=A + 2)])
def test_a_cache_that_does_not_fit_is_refused(bad):
    for name in ALL:
        assert calls(cache(**bad), batch())[name]() == 1, name


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(seqs=-1), dict(max_pages=-1), dict(groups=-1), dict(table_row=4), dict(starts=0), dict(lens=0), dict(table=0), dict(seqs=4097),
                                 dict(seqs=4000, groups=97, group_bounds=A, group_shared=A), dict(groups=1), dict(groups=1, group_bounds=A), dict(lens=A + 2)])
def test_a_batch_that_does_not_fit_is_refused(bad):
    for name in ALL:
        assert calls(cache(), batch(**bad))[name]() == 1, name


@pytest.mark.parametrize("bad,names", [
    (dict(q=0), ["attend"]), (dict(q=A + 2), ["append", "attend"]), (dict(q_row=511), ["append", "attend"]), (dict(q_row=504), ["append", "attend"]), (dict(out=0), ["append", "attend"]),
    (dict(out=4 * A + 4), ["append", "attend"]), (dict(out_row=500), ["append", "attend"]), (dict(heads=0), ["append", "attend"]), (dict(heads=7), ["attend"]), (dict(heads=-8), ["append", "attend"]),
    (dict(heads=65536, q_row=1 << 23, out_row=1 << 23), ["append", "attend"]), (dict(scale=math.nan), ["attend"]), (dict(scale=math.inf), ["attend"]), (dict(work=0), ["attend"]),
    (dict(work=A + 128), ["attend"]), (dict(lse=A + 2), ["attend"]), (dict(k=0), ["append", "read"]), (dict(v=0), ["append", "read"]), (dict(k_row=120), ["append", "read"]),
    (dict(v_row=100), ["append", "read"]), (dict(type=T.U8.id), ALL), (dict(rot=33), ["append"]), (dict(rot=-1), ["append"]), (dict(freq=0), ["append"]), (dict(freq=A + 2), ["append"]),
    (dict(out=A), ["append", "attend"]), (dict(out=A + 512), ["append", "attend"]), (dict(v=2 * A), ["read"]), (dict(out=2 * A), ["append"]), (dict(lse=4 * A), ["attend"]), (dict(lse=A), ["attend"])])
def test_rows_that_do_not_fit_are_refused(bad, names):
    for name in names:
        assert calls(cache(), batch(), **bad)[name]() in (1, 2), name
        assert capi.lib().xalm_cuda_last_error()


def test_nothing_to_do_is_no_error_and_launches_nothing():
    for b in (batch(rows=0), batch(seqs=0, starts=0, lens=0, table=0, max_pages=0)):
        for name, call in calls(cache(), b).items():
            assert call() == 0, name


def test_either_order_of_pages_and_heads_is_taken():
    """As far as the checks go: without a device the call then fails for want of one."""
    if capi.device_count_or_zero():
        pytest.skip("made-up addresses are for a box without a GPU")
    for c in (cache(), cache(page=RUN, head=4 * RUN), cache(page=1 << 20, head=RUN + 16), cache(dim=40, vdim=8)):
        for name, call in calls(c, batch(), q=16 * A, k=17 * A, v=18 * A, out=19 * A, work=32 * A, freq=20 * A, rot=16).items():
            assert call() == 3, name


def test_python_refuses_tensors_that_do_not_fit():
    n = paged.page4_bytes(16, 64)
    for args in ((torch.zeros(4, 2, n), 16, 64), (torch.zeros(4, 2, n, dtype=torch.uint8), 32, 64), (torch.zeros(4, n, dtype=torch.uint8), 16, 64), (torch.zeros(4, 2, n, dtype=torch.uint8), 16, 64, 128),
                 (torch.zeros(4, 2, 2 * n, dtype=torch.uint8)[:, :, ::2], 16, 64), (torch.zeros(4, 2, n, dtype=torch.uint8), 16, 64)):
        with pytest.raises(capi.XalmError):
            paged.PagedCache4(*args)
    assert paged.page4_bytes(64, 128) == 64 * 144 and paged.page4_bytes(16, 80, 256) == 16 * 18 * 12


def drafts(**over):
    a = dict(device=0, type=T.F32.id, seqs=2, rows=6, vocab=100, starts=A, tokens=2 * A, target=3 * A, target_row=100, draft=4 * A, draft_row=104, accept=5 * A, pick=6 * A, out=7 * A, taken=8 * A)
    a.update(over)
    return capi.lib().xalm_cuda_verify_drafts(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(type=T.U8.id), dict(seqs=-1), dict(seqs=65536), dict(rows=-1), dict(vocab=0), dict(vocab=-5), dict(vocab=(1 << 30) + 1, target_row=1 << 31, draft_row=1 << 31), dict(target_row=99),
                                 dict(draft_row=99), dict(target_row=1 << 41), dict(starts=0), dict(tokens=0), dict(target=0), dict(accept=0), dict(pick=0), dict(out=0), dict(taken=0),
                                 dict(tokens=A + 1), dict(target=3 * A + 2), dict(draft=4 * A + 1), dict(out=2 * A), dict(out=3 * A + 2000), dict(taken=A + 8), dict(taken=7 * A + 20), dict(out=5 * A)])
def test_drafts_that_do_not_fit_are_refused(bad):
    assert drafts(**bad) in (1, 2)
    assert capi.lib().xalm_cuda_last_error()


def test_no_sequences_to_verify_is_no_error():
    assert drafts(seqs=0) == 0


def test_python_refuses_drafts_that_do_not_fit():
    i, f = lambda *s: torch.zeros(*s, dtype=torch.int32), lambda *s: torch.zeros(*s)
    with pytest.raises(capi.XalmError):
        paged.verify(i(3), i(6), f(6, 100), f(6), f(2))  # on no GPU


def test_the_format_is_what_its_definition_says():
    x = torch.randn(3, 2, 16, 96, generator=torch.Generator().manual_seed(1)) * torch.tensor([1e-9, 1.0, 1e4])[:, None, None, None]
    d, c = quantise(x)
    assert d.dtype == torch.float16 and (c[..., 3, :] == 8).all() and (d[..., 3] == 0).all()
    y = values(d, c, 96)
    top = x.unflatten(-1, (-1, 32)).abs().amax(dim=-1, keepdim=True).expand(*x.shape[:-1], 3, 32).flatten(-2)
    # half a step, d being off by half a unit of its own, and one step where 8 d has the other sign
    assert ((y - x.double()).abs()[1:] <= top.double()[1:] / 8 * (1 + 2.0 ** -9)).all()
    assert ((y - x.double()).abs()[1:] <= top.double()[1:] / 16 * (1 + 2.0 ** -9)).double().mean() > 0.95
    assert (y[0] == 0).all()  # below what fp16 has
    back = unpack(pack(x, x[..., :40]), 16, 96, 40)
    assert torch.equal(back[0], y) and torch.equal(back[1], values(*quantise(x[..., :40]), 40))
    both = torch.zeros(1, 1, 16, 32)
    both[0, 0, 0, :2] = torch.tensor([-2.0, 2.0])  # the positive one
    assert float(quantise(both)[0][0, 0, 0, 0]) == -0.25 and quantise(both)[1][0, 0, 0, 0, :3].tolist() == [15, 0, 8]
    seen = {place(e, lanes, 4) for lanes in (4,) for e in range(128)}
    assert len(seen) == 128 and {b for b, _ in seen} == set(range(64)) and len({place(e, 8, 8) for e in range(256)}) == 256


def test_the_restatement_of_attention_sees_what_it_should():
    p = Problem4("f16", [3, 1, 0], [19, 5, 0], pad_rows=2, offset=1)
    out, lse, tol, _ = p.attend()
    assert torch.isnan(out[0]).all() and torch.isnan(out[5:]).all() and torch.isfinite(out[1:5]).all()
    assert torch.isnan(p.k[p.table[0, 1], :, 3:]).all() and BLOCKS(64) == 2
    assert float(tol[1:5].max()) < 0.02 * float(out[1:5].abs().max())


def test_the_restatement_of_verification_keeps_the_targets_distribution():
    g = torch.Generator().manual_seed(2)
    V, n = 5, 20000
    p, q = torch.tensor([0.5, 0.2, 0.1, 0.15, 0.05]), torch.tensor([0.1, 0.4, 0.3, 0.1, 0.1])
    x = torch.multinomial(q, n, replacement=True, generator=g).tolist()
    u, r = torch.rand(n, generator=g), torch.rand(n, generator=g)
    count = torch.zeros(V)
    for i in range(n):
        out, taken = verify([0, 2], [0, x[i]], p.expand(2, V), [u[i], 0.5], [r[i]], q.expand(2, V))
        count[out[0]] += 1
    # five standard deviations of a count
    assert ((count / n - p).abs() < 5 * (p * (1 - p) / n).sqrt()).all()
