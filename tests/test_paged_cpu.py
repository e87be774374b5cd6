"""The paged cache without a GPU: refusals ahead of the library, and the float64 restatement against hand-worked cases."""
import ctypes as C

import numpy as np
import pytest

import paged_cases as ref
from ruai_b200 import _lib, nn


class NoCalls:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


class Dev:
    ordinal, L, ctx = 0, NoCalls(), None


def fake(shape, np_dtype=np.float32, rdtype=None, ordinal=0):
    t = nn.Tensor.__new__(nn.Tensor)
    t.dev = Dev()
    t.dev.ordinal = ordinal
    t.shape, t.np_dtype, t.ptr = tuple(shape), np.dtype(np_dtype), None
    t.rdtype = {np.dtype(np.float32): nn.F32, np.dtype(np.float16): nn.F16}.get(t.np_dtype) if rdtype is None else rdtype
    return t


def ints(*shape, **kw):
    return fake(shape, np.int32, **kw)


def plan_args(R=3, pages=10, tokens=5):
    return dict(cached=ints(R), fresh=ints(R), table=ints(R, 4), ring=ints(pages), words=ints(3), page=16, out=nn.PagePlan(ints(R + 1), ints(tokens), ints(tokens), ints(3)))


@pytest.mark.parametrize("change", [dict(fresh=ints(2)), dict(table=ints(2, 4)), dict(table=ints(12)), dict(ring=ints(2, 5)), dict(words=ints(2)), dict(cached=fake((3,))),
                                    dict(out=nn.PagePlan(ints(3), ints(5), ints(5), ints(3))), dict(out=nn.PagePlan(ints(4), ints(5), ints(4), ints(3))), dict(out=None),
                                    dict(fresh=ints(3, ordinal=1))])
def test_plan_refuses(change):
    with pytest.raises(ValueError):
        nn.page_plan(**{**plan_args(), **change})


def append_args():
    return dict(qkv=fake((5, 8 * 16)), positions=ints(5), slots=ints(5), k_pages=fake((10, 2, 16, 16)), v_pages=fake((10, 2, 16, 16)), rope=fake((100, 8, 2)), out=fake((5, 4, 16)))


@pytest.mark.parametrize("change", [dict(qkv=fake((5, 100))), dict(qkv=fake((5, 4 * 16))), dict(qkv=ints(5, 128)), dict(positions=ints(4)), dict(slots=fake((5,))), dict(v_pages=fake((10, 2, 32, 16))),
                                    dict(v_pages=fake((10, 2, 16, 16), np.float16)), dict(rope=fake((100, 16))), dict(rope=fake((100, 8, 2), np.float16)), dict(out=fake((5, 4, 16), np.float16)),
                                    dict(out=fake((5, 8, 16))), dict(k_pages=fake((10, 2, 16))), dict(slots=ints(5, ordinal=1))])
def test_append_refuses(change):
    with pytest.raises(ValueError):
        nn.paged_append(**{**append_args(), **change})


def attention_args():
    return dict(q=fake((5, 4, 16)), k_pages=fake((10, 2, 16, 16)), v_pages=fake((10, 2, 16, 16)), table=ints(3, 4), cached=ints(3), starts=ints(4), most_fresh=2, most_len=40, out=fake((5, 4, 16)))


@pytest.mark.parametrize("change", [dict(q=fake((5, 64))), dict(q=fake((5, 4, 16), np.float16)), dict(q=fake((5, 4, 32))), dict(table=ints(2, 4)), dict(table=ints(12)), dict(cached=ints(2)),
                                    dict(starts=ints(3)), dict(out=fake((5, 2, 16))), dict(out=fake((5, 4, 16), np.uint16, nn.BF16)), dict(k_pages=ints(10, 2, 16, 16)), dict(cached=ints(3, ordinal=1))])
def test_attention_refuses(change):
    with pytest.raises(ValueError):
        nn.paged_attention(**{**attention_args(), **change})


def test_entry_points_refuse_a_null_context():
    L = _lib.load()
    p = C.c_void_p(64)
    assert L.ruai_page_plan(None, p, p, 1, 1, 16, p, 1, p, 1, p, p, p, p, p) == _lib.ERR_ARG
    assert L.ruai_paged_append(None, 0, p, 48, 16, 32, 1, 1, 0, None, 0, p, p, 0, p, p, 1, 1, 16, 16, p, 16) == _lib.ERR_ARG
    assert L.ruai_paged_attention(None, 0, p, 16, p, p, 1, 1, 16, 16, p, 1, p, p, 1, 1, 1, 1.0, 0, 1, 1, p, 16) == _lib.ERR_ARG


def test_restated_plan():
    table = np.array([[4, 7, -1], [2, -1, -1], [5, 1, -1]])
    ring = np.array([9, -1, -1, -1, -1, -1, -1, 0, 3, 6])
    t, r, starts, pos, slots, words = ref.plan([17, 16, 20], [2, 3, -1], table, ring, [7, 4, 0], 16, 7)
    assert t.tolist() == [[4, 7, -1], [2, 0, -1], [5, 1, -1]] and starts.tolist() == [0, 2, 5, 5]
    assert pos.tolist() == [17, 18, 16, 17, 18, -1, -1] and slots.tolist() == [113, 114, 0, 1, 2, -1, -1]
    assert words.tolist() == [8, 5, 0] and r.tolist() == [9, 5, 1, -1, -1, -1, -1, 0, 3, 6]
    assert ref.plan([17], [100], table[:1], ring, [7, 4, 0], 16, 100) is None


def test_restated_attention_sees_the_window_only():
    v = np.arange(32.0).reshape(2, 1, 16, 1).repeat(8, 3)
    out, _ = ref.attention(np.zeros((2, 1, 8)), np.zeros((2, 1, 16, 8)), v, np.array([[1, 0]]), [15], [0, 2], 1.0, 3, "f32")
    # positions 15 (last of page 1: values 16..31) and 16 (first of page 0)
    assert np.allclose(out[:, 0, 0], [(29 + 30 + 31) / 3, (30 + 31 + 0) / 3])


@pytest.mark.parametrize("change", [dict(window=-1), dict(most_fresh=-1), dict(most_len=-5)])
def test_attention_refuses_negative_bounds(change):
    """As unsigned numbers they would be no window, or bounds that every request keeps."""
    with pytest.raises(ValueError, match="negative"):
        nn.paged_attention(**{**attention_args(), **change})


def test_plan_refuses_a_negative_number_of_rows():
    with pytest.raises(ValueError, match="number of rows"):
        nn.page_plan(**{**plan_args(), "out": None, "tokens": -1})
