"""Which places of out relative to x the rotary entry takes, without a GPU:
rows that share no element, and x itself."""
import ctypes as C
import random

import pytest

import aigpu
from test_paged_refusals import PTR, _rotary


def _taken(**kw):
    if aigpu.available():
        pytest.skip("the pointers stand for nothing: no call is made beside a device")
    assert aigpu.lib().aigpu_rotary(C.byref(_rotary(**kw))) == 0
    why = aigpu.last_error()
    assert "no usable gfx950 device" in why or "overlap" in why, why
    return "overlap" not in why


def _elements(at, count, heads, dim, ts, hs):
    return {at + t * ts + h * hs + d for t in range(count) for h in range(heads) for d in range(dim)}


@pytest.mark.parametrize("count", [1, 4])
def test_the_halves_of_wider_heads(count):
    """[tokens][heads][2 dim]: from one half into the other, either way"""
    for shift in (64, -64):
        assert _taken(x=4 * PTR, out=4 * PTR + 4 * shift, count=count, heads=3, headStride=128, outHeadStride=128)
    assert not _taken(x=4 * PTR, out=4 * PTR + 4 * 32, count=count, heads=3, headStride=128, outHeadStride=128)


def test_places_of_equal_strides():
    """against the sets of elements: taken exactly where out is x or shares nothing with it"""
    r = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        count, heads, dim = r.randrange(1, 5), r.randrange(1, 5), r.choice([2, 4, 6])
        if r.random() < 0.5:
            hs = dim + r.randrange(0, 9)
            ts = (heads - 1) * hs + dim + r.randrange(0, 20)
        else:
            ts = dim + r.randrange(0, 9)
            hs = (count - 1) * ts + dim + r.randrange(0, 20)
        shift = r.randrange(-60, 61)
        apart = not (_elements(0, count, heads, dim, ts, hs) & _elements(shift, count, heads, dim, ts, hs))
        got = _taken(x=4 * PTR, out=4 * PTR + 4 * shift, count=count, heads=heads, dim=dim, rotaryDims=2,
                     tokenStride=ts, headStride=hs, outTokenStride=ts, outHeadStride=hs)
        assert got == (apart or shift == 0), (count, heads, dim, ts, hs, shift)
        seen[got] += 1
    assert min(seen.values()) > 500


def test_places_of_other_strides_share_nothing():
    r = random.Random(2)
    taken = 0
    for _ in range(4000):
        count, heads, dim = r.randrange(1, 5), r.randrange(1, 5), r.choice([2, 4])
        hs, ohs = dim + r.randrange(0, 9), dim + r.randrange(0, 9)
        ts = max(hs, ohs) * heads + r.randrange(0, 40)
        ots = r.choice([ts, heads * ohs + r.randrange(0, 9)])
        shift = r.randrange(-80, 81)
        if _taken(x=4 * PTR, out=4 * PTR + 4 * shift, count=count, heads=heads, dim=dim, rotaryDims=2, tokenStride=ts,
                  headStride=hs, outTokenStride=ots, outHeadStride=ohs):
            same = shift == 0 and (count == 1 or ts == ots) and (heads == 1 or hs == ohs)
            assert same or not (_elements(0, count, heads, dim, ts, hs) &
                                _elements(shift, count, heads, dim, ots, ohs)), (count, heads, dim, ts, hs, ots, ohs, shift)
            taken += 1
    assert taken > 300
