"""The paged cache without a GPU: the host's checks refuse what does not fit before anything is launched, and the restatement that the GPU tests use agrees with itself."""
import ctypes as C
import math

import pytest
import torch

from paged_ref import Problem
from xalm_b200 import capi, paged
from xalm_b200 import types as T

A = 1 << 20  # an address at a 16-byte boundary that no check reads from


def cache(**over):
    c = dict(type=T.BF16.id, device=0, pages=4, page_size=16, kv_heads=2, dim=64, vdim=64, k=A, v=A, k_page=2048, k_slot=128, k_head=64, v_page=2048, v_slot=128, v_head=64,
             means=A, status=0)
    c.update(over)
    return paged._Cache(**c)


def batch(**over):
    b = dict(rows=3, seqs=2, max_pages=5, groups=0, starts=A, lens=A, table=A, table_row=5, group_bounds=0, group_shared=0)
    b.update(over)
    return paged._Batch(**b)


def calls(c, b, q=A, q_row=512, heads=8, out=A, out_row=512, scale=0.1, lists=A, n=4, top=4, first=1, recent=1, k=A, k_row=128, v=A, v_row=128, in_type=T.BF16.id, freq=A,
          rot=32, work=A, room=1 << 40):
    L, p, w = capi.lib(), C.byref(c), C.byref(b)
    return {"append": lambda: L.xalm_cuda_paged_append(p, w, k, k_row, v, v_row, q, q_row, heads, in_type, out, out_row, freq, rot, 1.0, 0, None),
            "attend": lambda: L.xalm_cuda_paged_attend(p, w, q, q_row, heads, scale, out, out_row, None, work, room, None),
            "select": lambda: L.xalm_cuda_paged_select(p, w, q, q_row, heads, top, first, recent, out, None),
            "attend_selected": lambda: L.xalm_cuda_paged_attend_selected(p, w, q, q_row, heads, lists, n, scale, out, out_row, None, work, room, None)}


ALL = ["append", "attend", "select", "attend_selected"]


@pytest.mark.parametrize("bad", [dict(type=T.Q8.id), dict(pages=0), dict(page_size=8), dict(page_size=24), dict(page_size=512), dict(kv_heads=0), dict(dim=0), dict(dim=12),
                                 dict(dim=264, k_head=264), dict(vdim=4), dict(k=0), dict(v=0), dict(k=A + 8), dict(v=A + 2), dict(means=A + 4), dict(k_slot=0),
                                 dict(k_slot=-128), dict(v_page=2044), dict(k_slot=64), dict(v_head=32), dict(k_page=1024), dict(v_page=1 << 41)])
def test_a_cache_that_does_not_fit_is_refused(bad):
    for name in ALL:
        assert calls(cache(**bad), batch())[name]() in (1, 2), name


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(seqs=-1), dict(max_pages=-1), dict(groups=-1), dict(table_row=4), dict(starts=0), dict(lens=0), dict(table=0), dict(seqs=4097),
                                 dict(seqs=4000, groups=97, group_bounds=A, group_shared=A), dict(groups=1), dict(groups=1, group_bounds=A)])
def test_a_batch_that_does_not_fit_is_refused(bad):
    for name in ALL:
        assert calls(cache(), batch(**bad))[name]() == 1, name


@pytest.mark.parametrize("bad,names", [
    (dict(q=0), ALL[1:]), (dict(q=A + 2), ALL), (dict(q_row=511), ALL), (dict(q_row=504), ALL), (dict(out=0), ALL), (dict(out=A + 4), ["append", "attend", "attend_selected"]),
    (dict(out_row=500), ["append", "attend", "attend_selected"]), (dict(heads=0), ALL), (dict(heads=7), ALL[1:]), (dict(heads=-8), ALL), (dict(scale=math.nan), ["attend", "attend_selected"]),
    (dict(scale=math.inf), ["attend", "attend_selected"]), (dict(work=0), ["attend", "attend_selected"]), (dict(work=A + 128), ["attend", "attend_selected"]),
    (dict(lists=0), ["attend_selected"]), (dict(n=0), ["attend_selected"]), (dict(n=-3), ["attend_selected"]), (dict(n=1025), ["attend_selected"]),
    (dict(top=0), ["select"]), (dict(top=2), ["select"]), (dict(top=1025), ["select"]), (dict(first=-1), ["select"]), (dict(recent=-1), ["select"]), (dict(recent=3), ["select"]),
    (dict(first=2 ** 31 - 1), ["select"]), (dict(k=0), ["append"]), (dict(v=0), ["append"]), (dict(k_row=120), ["append"]), (dict(v_row=100), ["append"]), (dict(in_type=T.U8.id), ["append"]),
    (dict(rot=33), ["append"]), (dict(rot=-1), ["append"]), (dict(freq=0), ["append"])])
def test_rows_that_do_not_fit_are_refused(bad, names):
    for name in names:
        assert calls(cache(), batch(), **bad)[name]() in (1, 2), name
        assert capi.lib().xalm_cuda_last_error()


def test_select_needs_mean_keys_and_room_for_the_scores():
    assert calls(cache(means=0), batch())["select"]() == 4
    assert calls(cache(), batch(max_pages=24577, table_row=24577))["select"]() == 1


def test_tables_of_more_tokens_than_positions_are_refused():
    for op in calls(cache(page_size=16), batch(max_pages=(1 << 26) + 1, table_row=1 << 27)).values():
        assert op() == 1


def test_nothing_to_do_is_no_error_and_launches_nothing():
    for b in (batch(rows=0), batch(seqs=0, starts=0, lens=0, table=0, max_pages=0)):
        for name, call in calls(cache(), b).items():
            assert call() == 0, name


def test_a_head_major_pool_and_a_sliced_one_are_taken():
    """As far as the checks go: without a device the call then fails for want of one."""
    if capi.device_count_or_zero():
        pytest.skip("made-up addresses are for a box without a GPU")
    for c in (cache(k_slot=64, k_head=1024, v_slot=64, v_head=1024), cache(k_page=1 << 20, k_slot=4096, k_head=512)):
        for name, call in calls(c, batch()).items():
            assert call() == 3, name


def test_python_refuses_tensors_that_do_not_fit():
    k = torch.zeros(4, 16, 2, 64)
    for args in ((k, k), (k, k.half()), (k, k[:3]), (k[0], k[0]), (k.transpose(2, 3), k.transpose(2, 3)), (k, k, torch.zeros(4, 2, 32))):
        with pytest.raises(capi.XalmError):
            paged.PagedCache(*args)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    for args in ((i(3), i(3), i(2, 5)), (i(2), i(2), i(2, 5)), (i(3).long(), i(2), i(2, 5)), (i(3), i(2), i(5, 2).T), (i(3), i(2), i(2)), (i(3), i(2), i(2, 5), i(2)), (i(3), i(2), i(2, 5), i(2), i(2))):
        with pytest.raises(capi.XalmError):
            paged.Batch(*args)
    assert paged.Batch(i(3), i(2), i(2, 5), i(3), i(2)).c.groups == 2


def test_the_restatement_sees_what_it_should():
    p = Problem("f32", [3, 1, 0], [19, 5, 0], pad_rows=2, offset=1)
    out, lse, tol, _ = p.attend()
    assert torch.isnan(out[0]).all() and torch.isnan(out[5:]).all() and not torch.isnan(out[1:5]).any()
    everything = torch.arange(p.max_pages).repeat(p.rows, p.G, 1)
    again = p.attend(lists=everything)
    assert torch.equal(again[0][1:5], out[1:5])
    q = p.turned(p.q, 16, torch.ones(16), 1.0, False)
    assert torch.allclose(q[1:5].norm(dim=-1), p.q[1:5].double().norm(dim=-1))
