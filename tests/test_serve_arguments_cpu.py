"""What capi.CudaBackend's serving operators take from another library: a torch tensor that is not in the device's memory, of another type, in another order, or too
small for the call, never reaches the library, where it would be an address."""
import types

import numpy as np
import pytest

from powerserve_b200 import capi

torch = pytest.importorskip("torch")


class Library:
    """notes the calls instead of making them"""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.fixture
def be():
    b = object.__new__(capi.CudaBackend)
    b.L, b.h, b.device, b.desc = Library(), None, 0, None
    return b


def buffer(nbytes):
    b = object.__new__(capi.DeviceBuffer)
    b.nbytes, b.ptr = nbytes, 4096
    return b


class OnDevice(torch.Tensor):
    """a tensor that says it lies on a device"""
    is_cuda = True
    index = 0

    @property
    def device(self):
        return types.SimpleNamespace(index=self.index)


def on_device(t, index=0):
    t = t.as_subclass(OnDevice)
    t.index = index
    return t


def sample(be, **change):
    a = dict(ids=on_device(torch.zeros(3, dtype=torch.int32)), probs=on_device(torch.zeros(3)), logits=on_device(torch.zeros(3, 10)), vocab=10, rows=3, samplers=on_device(torch.zeros(3, 4)),
             u=on_device(torch.zeros(3))) | change
    be.sample(**a)


def caches(tok=2, n_kv=12):
    t = np.zeros(1, capi.CACHE)
    t["n_ctx"], t["n_kv"], t["n_tok"] = 16, n_kv, tok
    return t


def attend(be, table=None, **change):
    a = dict(out=on_device(torch.zeros(2, 4 * 32)), q=on_device(torch.zeros(2, 4 * 32)), caches=caches() if table is None else table, n_heads=4, n_kv_heads=2, head_size=32, scale=1.0,
             tree_mask=on_device(torch.zeros(2, 2, dtype=torch.uint8))) | change
    be.attn_tree(**a)


def test_what_is_right_goes_through(be):
    sample(be)
    sample(be, probs=None, ids=buffer(12), samplers=buffer(48), u=4096)
    wide = on_device(torch.zeros(3, 16))
    sample(be, logits=wide, row_stride=16)
    sample(be, logits=wide[:, :10], row_stride=16)
    sample(be, logits=wide[:, 6:], row_stride=16)
    attend(be)
    attend(be, tree_mask=None, out=buffer(1024))
    attend(be, tree_mask=on_device(torch.zeros(4, dtype=torch.bool)))
    assert [c[0] for c in be.L.calls] == ["ps_cuda_sample"] * 5 + ["ps_cuda_attn_tree"] * 3
    assert be.L.calls[1][1][2] is None and be.L.calls[1][1][8] == 4096


def test_rows_of_a_wider_tensor(be):
    """with no row_stride said, a matrix of as many rows as are drawn from brings its own"""
    strides = {"as wide": (on_device(torch.zeros(3, 10)), 10), "wider": (on_device(torch.zeros(3, 16)), 16), "a part": (on_device(torch.zeros(3, 16))[:, 2:12], 16), "flat": (on_device(torch.zeros(30)), 10),
               "other rows": (on_device(torch.zeros(6, 5)), 10), "a buffer": (buffer(120), 10), "an address": (np.uint64(4096), 10)}
    for name, (logits, want) in strides.items():
        sample(be, logits=logits)
        call = be.L.calls.pop()[1]
        assert call[4] == want and type(call[3]) is int, name
    one = on_device(torch.zeros(1, 16))     # (one row)
    sample(be, rows=1, logits=one)
    assert be.L.calls.pop()[1][4] >= 10


@pytest.mark.parametrize("name,what,match", [
    ("logits", torch.zeros(3, 10), "not in the memory"), ("u", torch.zeros(3), "not in the memory"), ("ids", np.zeros(3, np.int32), "ndarray"), ("probs", [0.0] * 3, "list"),
    ("ids", on_device(torch.zeros(3, dtype=torch.int64)), "int64"), ("logits", on_device(torch.zeros(3, 10, dtype=torch.bfloat16)), "bfloat16"), ("u", on_device(torch.zeros(3, dtype=torch.float64)), "float64"),
    ("u", on_device(torch.zeros(3), 1), "not in the memory"), ("u", on_device(torch.zeros(2)), "holds 8 bytes"), ("samplers", on_device(torch.zeros(2, 4)), "holds 32"), ("logits", on_device(torch.zeros(2, 10)), "holds 80"),
    ("ids", buffer(8), "holds 8"), ("u", on_device(torch.zeros(6))[::2], "follow one another"), ("logits", on_device(torch.zeros(10, 3)).T, "follow one another"),
    ("logits", on_device(torch.zeros(3, 20))[:, ::2], "follow one another")])
def test_samples_refused(be, name, what, match):
    with pytest.raises(capi.PsCudaError, match=match):
        sample(be, **{name: what})
    assert not be.L.calls


@pytest.mark.parametrize("name,what,match", [
    ("q", torch.zeros(2, 128), "not in the memory"), ("out", on_device(torch.zeros(2, 128, dtype=torch.float16)), "float16"), ("out", on_device(torch.zeros(1, 128)), "holds 512"), ("q", buffer(1020), "holds 1020"),
    ("tree_mask", on_device(torch.zeros(4)), "float32"), ("tree_mask", on_device(torch.zeros(3, dtype=torch.uint8)), "holds 3"), ("q", on_device(torch.zeros(2, 256))[:, ::2], "follow one another")])
def test_attention_refused(be, name, what, match):
    with pytest.raises(capi.PsCudaError, match=match):
        attend(be, **{name: what})
    assert not be.L.calls


def test_settings_of_the_last_pass_s_rows(be):
    """SAMPLER records or tuples, one for each row or one for all"""
    m = object.__new__(capi.CudaModel)
    m.be, seen = be, []

    def sample_last(h, rows, settings, u, ids, probs):
        seen.append(np.ctypeslib.as_array((capi.C.c_uint8 * (16 * rows)).from_address(settings)).copy().view(capi.SAMPLER) if rows else None)
        return 0

    be.L.ps_cuda_sample_last = sample_last
    rows = [(1.0, 0, 0.9, 0.0), (0.5, 40, 0.95, 0.02), (0.0, 0, 1.0, 0.0), (1.5, 7, 0.5, 0.25)]
    table = np.array(rows, capi.SAMPLER)
    for each in (rows, tuple(rows), table, list(table), [list(r) for r in rows], [tuple(np.float32(f) for f in r) for r in rows]):
        m.sample(each, [0.5] * 4)
        assert np.array_equal(seen.pop(), table)
    for one in (rows[1], list(rows[1]), [rows[1]], table[1], table[1:2], tuple(np.float64(f) for f in rows[1])):
        for n in (1, 4):
            m.sample(one, [0.5] * n)
            assert np.array_equal(seen.pop(), np.array([rows[1]] * n, capi.SAMPLER))
    m.sample(rows[:0], [])
    m.sample(rows[0], [])
    for wrong in (rows[:3], table[:3], np.zeros((4, 4), np.float32)):
        with pytest.raises((ValueError, TypeError)):
            m.sample(wrong, [0.5] * 4)


def test_calls_that_the_library_refuses_reach_it(be):
    """sizes follow from what is asked for; where that makes no sense, the library says so"""
    sample(be, rows=-1)
    sample(be, vocab=1 << 19, row_stride=1 << 19)
    sample(be, vocab=10, row_stride=3)
    attend(be, n_heads=5)
    attend(be, n_heads=66)
    attend(be, head_size=288)
    attend(be, caches(13))
    attend(be, caches(-1))
    assert len(be.L.calls) == 8
