"""Pages taken, shared, given back and copied, slots that move together: tables, counts, codes and scales against plain forms, all of them whole numbers or equal bits."""
import numpy as np
import pytest

from powerserve_b200 import capi
from tests import _paged as P
from tests.test_gpu_serve_attention import be  # noqa: F401

pytestmark = pytest.mark.gpu


def run(be, c, edits, held=True):  # noqa: F811
    """edits: (table number, from number or None, n_old, n_new); checks everything"""
    rec = np.zeros(len(edits), capi.PAGE_EDIT)
    for e, (t, f, old, new) in enumerate(edits):
        rec[e] = (c.dev[t].ptr, 0 if f is None else c.dev[f].ptr, old, new, len(c.tables[t]), 0)
    h = be.upload(np.full(len(edits), -7, np.int32))
    be.paged_edit(c.cache, rec, h if held else None)
    want, copies = P.edit(c.refs, c.P, [(c.tables[t], None if f is None else c.tables[f], old, new) for t, f, old, new in edits])
    was_codes, was_scales = c.codes.copy(), c.scales.copy()
    B = c.P // P.BLOCK
    for src, dst, n in copies:
        shape = (*c.codes.shape[:4], B, -1)
        c.codes.reshape(shape)[:, dst, :, :, :n] = was_codes.reshape(shape)[:, src, :, :, :n]
        c.scales[:, dst, :, :, :n] = was_scales[:, src, :, :, :n]
    codes, scales, refs = c.read()
    for i, d in enumerate(c.dev):
        assert np.array_equal(d.numpy(np.int32), c.tables[i]), i
    assert np.array_equal(refs, c.refs)
    assert not held or h.numpy(np.int32).tolist() == want
    assert np.array_equal(codes, c.codes) and np.array_equal(scales.view(np.uint32), c.scales.view(np.uint32))
    h.free()
    be.sync()
    return want


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_life_of_sequences(be, page):  # noqa: F811
    r = np.random.default_rng(page)
    lens = [0, 1, page, page + 1, 3 * page - 1, 70, 0, 0, 0, 0]
    c = P.Cache(be, lens, 2, 64, page, layers=3, spare=60, room=12, seed=page)
    lens = run(be, c, [(i, None, n, n + 5) for i, n in enumerate(lens[:6])])                                     # all grow
    lens = lens + [0, 0, 0, 0]
    lens[6:9] = run(be, c, [(6, 4, lens[4], lens[4]), (7, 4, lens[4], lens[4] + 1), (8, 4, page + 3, page + 3)])  # three begin with the fifth's pages
    got = run(be, c, [(4, None, lens[4], lens[4] + 1), (6, None, lens[6], lens[6] + 20), (8, None, lens[8], lens[8] + 1)])  # (a last page held by several that are written)
    lens[4], lens[6], lens[8] = got
    got = run(be, c, [(4, None, lens[4], 0), (9, 6, lens[6] - 3, lens[6] - 2), (3, None, lens[3], page), (5, None, lens[5], lens[5])])
    lens[4], lens[9], lens[3], lens[5] = got
    for step in range(12):      # whatever comes
        order = r.permutation(10)
        edits = []
        for t in order[:int(r.integers(1, 11))]:
            edits.append((int(t), None, lens[t], max(0, lens[t] + int(r.integers(-2 * page, 2 * page)))))
            edits[-1] = (*edits[-1][:3], min(edits[-1][3], len(c.tables[t]) * page))
        for (t, *_), n in zip(edits, run(be, c, edits)):
            lens[t] = n
        empty = [t for t in range(10) if lens[t] == 0]
        full = [t for t in range(10) if lens[t] > 0]
        if empty and full:
            t, f = empty[0], int(r.choice(full))
            n = min(int(r.integers(1, lens[f] + 1)), len(c.tables[t]) * page - 1)
            lens[t] = run(be, c, [(t, f, n, n + int(r.integers(0, 2)))])[0]
    run(be, c, [(t, None, lens[t], 0) for t in range(10)])
    assert (c.refs == 0).all()
    c.free()


def test_too_few_pages(be):  # noqa: F811
    """the first that finds too few stays, so do those behind it that need one; who needs none grows"""
    c = P.Cache(be, [16, 16, 10, 16, 20], 1, 32, 16, spare=3, room=5, seed=1)
    assert run(be, c, [(0, None, 16, 40), (1, None, 16, 60), (2, None, 10, 16), (3, None, 16, 17), (4, None, 20, 32)]) == [40, 16, 16, 16, 32]
    c.free()


def test_too_few_pages_for_copies(be):  # noqa: F811
    """four tables of one page that is not full: two get copies, the last one may not write what the third still holds"""
    c = P.Cache(be, [20, 0, 0, 0], 1, 32, 16, spare=1, room=3, seed=2)
    run(be, c, [(1, 0, 20, 20), (2, 0, 20, 20), (3, 0, 20, 20)])
    assert run(be, c, [(i, None, 20, 21) for i in range(4)]) == [21, 20, 20, 20]
    c.free()
    c = P.Cache(be, [20, 0, 0, 0], 1, 32, 16, spare=3, room=3, seed=2)
    run(be, c, [(1, 0, 20, 20), (2, 0, 20, 20), (3, 0, 20, 20)])
    assert run(be, c, [(i, None, 20, 21) for i in range(4)]) == [21, 21, 21, 21]
    assert c.tables[3][1] not in [c.tables[i][1] for i in range(3)]
    c.free()


def test_pages_freed_by_the_call_are_taken_by_it(be):  # noqa: F811
    c = P.Cache(be, [64, 5, 0], 1, 32, 16, spare=0, room=4, seed=3)
    assert run(be, c, [(1, None, 5, 60), (0, None, 64, 0)]) == [60, 0]
    assert run(be, c, [(2, 1, 60, 61), (1, None, 60, 0)], held=False) == [61, 0]     # (its page has one holder left, who keeps it)
    c.free()


def test_many_edits_and_many_pages(be):  # noqa: F811
    """a full call; the free pages lie behind thousands that are held"""
    n = capi.PAGE_EDITS
    c = P.Cache(be, [16 * 40] + [3] * (n - 1), 1, 32, 16, spare=2 * n + 7, room=3, seed=4)
    c.refs[:-n - 500] += 1        # (held by tables elsewhere)
    be._ck(be.L.ps_cuda_memcpy_h2d(be.h, c.cache.refs.ptr, c.refs.ctypes.data, c.refs.nbytes))
    run(be, c, [(i, None, x, x + 17) for i, x in enumerate(c.lens)])
    c.free()


@pytest.mark.parametrize("off", [0, 4, 8])
def test_counts_that_begin_anywhere(be, off):  # noqa: F811
    c = P.Cache(be, [20, 40], 1, 32, 16, spare=9000, room=300, seed=5)
    buf = be.upload(np.concatenate([np.zeros(off // 4, np.int32), c.refs]))
    cache = capi.PagedCache(be, 1, c.n_pages, 16, 1, 32, codes=c.cache.codes, scales=c.cache.scales, refs=buf.ptr + off)
    rec = np.array([(c.dev[0].ptr, 0, 20, 4000, len(c.tables[0]), 0), (c.dev[1].ptr, 0, 40, 3999, len(c.tables[1]), 0)], capi.PAGE_EDIT)
    be.paged_edit(cache, rec)
    P.edit(c.refs, 16, [(c.tables[0], None, 20, 4000), (c.tables[1], None, 40, 3999)])
    assert np.array_equal(buf.numpy(np.int32)[off // 4:], c.refs)
    assert all(np.array_equal(d.numpy(np.int32), t) for d, t in zip(c.dev, c.tables))
    buf.free()
    c.free()


def test_a_page_that_nobody_holds_is_given_back(be):  # noqa: F811
    """reported, and it stays free; so does a table's entry that is no page"""
    c = P.Cache(be, [40, 40], 1, 32, 16, spare=1, seed=6)
    c.refs[c.tables[0][1]] = 0
    be._ck(be.L.ps_cuda_memcpy_h2d(be.h, c.cache.refs.ptr, c.refs.ctypes.data, c.refs.nbytes))
    rec = np.array([(c.dev[0].ptr, 0, 40, 0, len(c.tables[0]), 0)], capi.PAGE_EDIT)
    be.paged_edit(c.cache, rec)
    with pytest.raises(capi.PsCudaError, match="names what is not there"):
        be.sync()
    refs = c.cache.refs.numpy(np.int32)
    assert (refs[c.tables[0][:3]] == 0).all() and (refs[c.tables[1][:3]] == 1).all()
    t = c.tables[1].copy()
    t[0], t[2] = c.n_pages, -1
    be._ck(be.L.ps_cuda_memcpy_h2d(be.h, c.dev[1].ptr, t.ctypes.data, t.nbytes))
    rec = np.array([(c.dev[1].ptr, 0, 40, 0, 3, 0), (c.dev[0].ptr, c.dev[1].ptr, 40, 40, 3, 0)], capi.PAGE_EDIT)
    be.paged_edit(c.cache, rec)
    with pytest.raises(capi.PsCudaError, match="names what is not there"):
        be.sync()
    assert c.cache.refs.numpy(np.int32)[c.tables[1][1]] == 1
    c.free()


# ---------------------------------------------------------------------------------------------------------------- slots that move together
def move(be, c, jobs, dev=True, spare=0):  # noqa: F811
    """jobs: (sequence, first, kept slots); spare: entries of the lists behind the count"""
    rec, bufs = np.zeros(len(jobs), capi.PAGE_MOVE), []
    for e, (i, first, keep) in enumerate(jobs):
        bufs += [be.upload(np.array(list(keep) + [-1] * spare, np.int32)), be.upload(np.array([len(keep)], np.int32))]
        rec[e] = (c.dev[i].ptr, bufs[-2].ptr, bufs[-1].ptr if dev else 0, first, c.lens[i], min(len(keep) + spare, c.lens[i] - first) if dev else len(keep), len(c.tables[i]))
    be.paged_compact(c.cache, rec)
    for i, first, keep in jobs:
        P.compact(c, i, first, list(keep))
    codes, scales, _ = c.read()
    assert np.array_equal(codes, c.codes) and np.array_equal(scales.view(np.uint32), c.scales.view(np.uint32))
    be.sync()
    for b in bufs:
        b.free()


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_compaction(be, D, page):  # noqa: F811
    r = np.random.default_rng(D)
    lens = [13, 40, 200, 333, 65, 700]
    c = P.Cache(be, lens, 2, D, page, layers=2, seed=D)
    some = lambda n, k: np.sort(r.choice(n, k, replace=False))    # noqa: E731
    move(be, c, [(0, 0, some(13, 5)), (1, 28, [0, 3, 4, 11]), (2, 189, [0, 1, 2]), (3, 1, some(332, 100)), (4, 64, [0]), (5, 130, some(570, 400))], spare=3)
    move(be, c, [(5, 0, some(700, 699)), (3, 16, range(317)), (2, 5, [194]), (1, 0, some(40, 17))], dev=False)
    c.free()


def test_what_need_not_move_is_not_rounded(be):  # noqa: F811
    c = P.Cache(be, [100, 100], 1, 64, 16, seed=7)
    was = c.codes.copy()
    move(be, c, [(0, 7, range(60)), (1, 96, [0, 1, 2, 3])])
    assert np.array_equal(c.codes, was)
    move(be, c, [(0, 16, range(16, 32))])       # a whole block moves by a block
    a, b = c.tables[0][1], c.tables[0][2]
    assert np.array_equal(c.codes[0, a], was[0, b])
    c.free()


def test_scales_of_zero(be):  # noqa: F811
    c = P.Cache(be, [64], 1, 32, 16, seed=8, junk=False)
    c.scales[:] = 0.0
    be._ck(be.L.ps_cuda_memcpy_h2d(be.h, c.cache.scales.ptr, c.scales.ctypes.data, c.scales.nbytes))
    move(be, c, [(0, 3, [1, 20, 30])])
    c.free()


@pytest.mark.parametrize("keep", [[0, 2, 2], [0, 5, 4], [1, 0], [0, 50], [3, -1], [0, 2 ** 31 - 1]])
def test_lists_that_do_not_rise_or_leave_the_slots(be, keep):  # noqa: F811
    """they are reported, and nothing outside the sequence's own slots changes"""
    c = P.Cache(be, [60, 60], 2, 64, 16, seed=9)
    rec = np.zeros(2, capi.PAGE_MOVE)
    k, good = be.upload(np.array(keep, np.int32)), be.upload(np.array([1, 4, 9], np.int32))
    rec[0] = (c.dev[0].ptr, k.ptr, 0, 20, 60, len(keep), len(c.tables[0]))
    rec[1] = (c.dev[1].ptr, good.ptr, 0, 20, 60, 3, len(c.tables[1]))
    be.paged_compact(c.cache, rec)
    with pytest.raises(capi.PsCudaError, match="names what is not there"):
        be.sync()
    P.compact(c, 1, 20, [1, 4, 9])
    codes, scales, _ = c.read()
    others = np.setdiff1d(np.arange(c.n_pages), c.tables[0][1:4])
    assert np.array_equal(codes[:, others], c.codes[:, others]) and np.array_equal(scales[:, others].view(np.uint32), c.scales[:, others].view(np.uint32))
    k.free()
    good.free()
    c.free()


def test_counts_of_the_device(be):  # noqa: F811
    """none, fewer than nothing, more than the list has"""
    c = P.Cache(be, [60, 60, 60], 1, 32, 16, seed=10)
    n, k = be.upload(np.array([0, -5, 99], np.int32)), be.upload(np.array([1, 4, 9], np.int32))
    rec = np.zeros(3, capi.PAGE_MOVE)
    for i in range(3):
        rec[i] = (c.dev[i].ptr, k.ptr, n.ptr + 4 * i, 20, 60, 3, len(c.tables[i]))
    be.paged_compact(c.cache, rec)
    P.compact(c, 2, 20, [1, 4, 9])
    codes, scales, _ = c.read()
    assert np.array_equal(codes, c.codes) and np.array_equal(scales.view(np.uint32), c.scales.view(np.uint32))
    n.free()
    k.free()
    c.free()


def test_many_moves(be):  # noqa: F811
    r = np.random.default_rng(11)
    lens = r.integers(20, 60, 300).tolist()
    c = P.Cache(be, lens, 1, 32, 16, seed=12)
    move(be, c, [(i, n - 12, np.sort(r.choice(12, int(r.integers(1, 13)), replace=False))) for i, n in enumerate(lens)])
    c.free()
