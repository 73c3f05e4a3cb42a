"""What needs no address where it has no place: a history without places, what no request holds."""
import ctypes

import pytest

from test_draft import lib, pick_desc, plan_desc  # noqa: F401


@pytest.mark.parametrize("history", [None, 256])
def test_history_without_places_is_taken(lib, history):  # noqa: F811
    d = pick_desc(history=history, history_wide=0, logits=258)
    assert lib.warp_pick_tokens(ctypes.byref(d), ctypes.c_void_p(256), None) == -1
    assert b"aligned" in lib.warp_last_error()


@pytest.mark.parametrize("kw", [dict(history=None), dict(history_len=None),
                                dict(history_len=None, history_wide=0)])
def test_history_goes_with_its_lengths(lib, kw):  # noqa: F811
    d = pick_desc(**kw)
    assert lib.warp_pick_tokens(ctypes.byref(d), ctypes.c_void_p(256), None) == -1
    assert b"together" in lib.warp_last_error()


def test_scratch_by_either_of_the_two(lib):  # noqa: F811
    many = dict(tokens=600, max_q=600, vocab=40000, row=40000, seen_words=10)
    need = [lib.warp_pick_scratch(ctypes.byref(pick_desc(**many, **kw)))
            for kw in ({}, dict(history=None), dict(history_len=None),
                       dict(history=None, history_len=None))]
    assert need[0] == need[1] == need[2] > need[3] > 0


@pytest.mark.parametrize("kw", [dict(held=None), dict(held=None, kv_len=None, pages=None), {}])
def test_a_plan_of_no_request(lib, kw):  # noqa: F811
    """Nothing to do, with a pool too: what [0] requests hold has no address."""
    assert lib.warp_step_plan(ctypes.byref(plan_desc(batch=0, tokens=0, **kw)), None) == 0


def test_tokens_of_no_request_are_refused(lib):  # noqa: F811
    assert lib.warp_step_plan(ctypes.byref(plan_desc(batch=0, held=None)), None) == -1
    assert b"no request" in lib.warp_last_error()
