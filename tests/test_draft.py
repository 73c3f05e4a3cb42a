"""What of a step of drafted tokens runs without a device: the refusals of its C
entry points and wrappers, and the layout of its descriptions."""
import ctypes

import pytest
import torch

from test_attention import attn_desc, kv_pages
from warp_b200 import ffi, ops


@pytest.fixture(scope="module")
def lib():
    from warp_b200 import build
    build.build()
    return ffi.load()


def filled(cls, good, kw):
    d = cls()
    for k, v in {**good, **kw}.items():
        setattr(d, k, v)
    return d


def plan_desc(**kw):
    return filled(ffi.PlanDesc, dict(
        batch=1, tokens=1, q_start=256, kv_len=256, pages=256, pages_row=4, pages_per_row=4,
        page_size=16, held=256, pool=256, pool_pages=8, parents=256, seen=256, max_q=1,
        positions=256, slots=256), kw)


def pick_desc(**kw):
    return filled(ffi.PickDesc, dict(
        tokens=2, batch=1, vocab=100, type=0, max_q=2, logits=256, row=100, picked=256,
        q_start=256, history=256, history_len=256, history_row=8, history_wide=8, repetition=256,
        drafted=256, seen=256, seen_words=1), kw)


def accept_desc(**kw):
    return filled(ffi.AcceptDesc, dict(
        batch=1, tokens=1, max_q=1, drafted=256, picked=256, seen=256, seen_words=1, q_start=256,
        kv_len=256, pages=256, pages_row=4, pages_per_row=4, count=768, path=256, chosen=256,
        kv_after=512), kw)


@pytest.mark.parametrize("fmt, cls", [("PLAN_DESC", "PlanDesc"), ("PICK_DESC", "PickDesc"),
                                      ("ACCEPT_DESC", "AcceptDesc")])
def test_packed_descriptions_match_the_structures(fmt, cls):
    fmt, cls = getattr(ffi, fmt), getattr(ffi, cls)
    values = list(range(1, len(cls._fields_) + 1))
    raw = fmt.pack(*values)
    assert fmt.size == ctypes.sizeof(cls)
    d = cls.from_buffer_copy(raw)
    assert [getattr(d, name) for name, _ in cls._fields_] == values


@pytest.mark.parametrize("kw, text", [
    (dict(batch=-1), b"negative"), (dict(tokens=-1), b"negative"), (dict(base=-1), b"negative"),
    (dict(max_q=-1), b"negative"), (dict(page_size=24), b"page_size"),
    (dict(page_size=8), b"page_size"), (dict(held=None), b"together"), (dict(pool=None), b"together"),
    (dict(pool_pages=-1), b"pool"), (dict(pool_pages=(1 << 31) - 1), b"pool"),
    (dict(batch=1 << 20, pages_per_row=1 << 12), b"2^31"), (dict(batch=0), b"no request"),
    (dict(kv_len=None), b"NULL"), (dict(pages=None), b"NULL"), (dict(q_start=None), b"NULL"),
    (dict(slots=None), b"NULL"), (dict(positions=None), b"NULL"), (dict(seen=None), b"masks"),
    (dict(seen=260), b"8-byte"), (dict(batch=2, pages_row=3), b"overlap")])
def test_plan_refusals(lib, kw, text):
    assert lib.warp_step_plan(ctypes.byref(plan_desc(**kw)), None) == -1
    assert text in lib.warp_last_error()


def test_nothing_to_do(lib):
    assert lib.warp_step_plan(None, None) == -1
    assert lib.warp_step_plan(ctypes.byref(plan_desc(batch=0, tokens=0)), None) == 0
    assert lib.warp_step_plan(ctypes.byref(plan_desc(tokens=0, held=None, pool=None)), None) == 0
    assert lib.warp_pick_tokens(None, None, None) == -1
    assert lib.warp_pick_scratch(None) == -1
    for kw in (dict(tokens=0), dict(batch=0), dict(max_q=0)):
        assert lib.warp_pick_scratch(ctypes.byref(pick_desc(**kw))) >= 0
        assert lib.warp_pick_tokens(ctypes.byref(pick_desc(**kw)), None, None) == 0
    assert lib.warp_tree_accept(None, None, 0, None, None, None) == -1
    assert lib.warp_tree_accept(ctypes.byref(accept_desc(batch=0)), None, 0, None, None, None) == 0
    for kw in (dict(tokens=0), dict(batch=0), dict(max_q=0)):
        assert lib.warp_tree_attention(ctypes.byref(attn_desc(**kw)), ctypes.byref(kv_pages()),
                                       None, 0, None, None) == 0


@pytest.mark.parametrize("kw, seen, words, text", [
    ({}, None, 1, b"masks"), ({}, 260, 1, b"8-byte"), ({}, 256, 0, b"words"),
    (dict(max_q=65, tokens=65), 256, 1, b"words"), ({}, 256, 1 << 24, b"words"),
    (dict(q=None), 256, 1, b"NULL"), (dict(head_dim=96), 256, 1, b"head_dim"),
    (dict(scale=0.0), 256, 1, b"scale")])
def test_tree_refusals(lib, kw, seen, words, text):
    c = kv_pages(head_dim=kw.get("head_dim", 64))
    p = None if seen is None else ctypes.c_void_p(seen)
    assert lib.warp_tree_attention(ctypes.byref(attn_desc(**kw)), ctypes.byref(c), p, words,
                                   ctypes.c_void_p(256), None) == -1
    error = lib.warp_last_error()
    assert text in error and b"warp_tree_attention" in error


@pytest.mark.parametrize("kw, text", [
    (dict(tokens=-1), b"negative"), (dict(max_q=-1), b"negative"), (dict(vocab=0), b"vocabulary"),
    (dict(vocab=1 << 30), b"vocabulary"), (dict(type=3), b"type"), (dict(row=-1), b"stride"),
    (dict(allowed_row=-1), b"stride"), (dict(q_start=None), b"rows of"),
    (dict(logits=None), b"NULL"), (dict(picked=None), b"NULL"), (dict(history=None), b"together"),
    (dict(history_len=None), b"together"), (dict(seen=None), b"together"),
    (dict(drafted=None), b"together"), (dict(seen=260), b"8-byte"), (dict(logits=258), b"aligned"),
    (dict(out=257, type=1), b"aligned"), (dict(out=256, out_row=104), b"layout"),
    (dict(q_start=None, batch=2), b"together")])
def test_pick_refusals(lib, kw, text):
    assert lib.warp_pick_tokens(ctypes.byref(pick_desc(**kw)), ctypes.c_void_p(256), None) == -1
    assert text in lib.warp_last_error()


def test_pick_refuses_bad_scratch(lib):
    many = pick_desc(tokens=600, max_q=600, vocab=40000, row=40000, seen_words=10)
    assert lib.warp_pick_scratch(ctypes.byref(many)) > 0
    for at in (None, 264):
        assert lib.warp_pick_tokens(ctypes.byref(many), at, None) == -1
        assert b"scratch" in lib.warp_last_error()


@pytest.mark.parametrize("kw, ckw, text", [
    (dict(batch=-1), {}, b"negative"), (dict(max_q=65), {}, b"words"),
    (dict(max_q=4097, seen_words=65), {}, b"nodes"), (dict(seen=None), {}, b"masks"),
    (dict(seen=260), {}, b"8-byte"), (dict(drafted=None), {}, b"NULL"), (dict(path=None), {}, b"NULL"),
    (dict(count=None), {}, b"NULL"), (dict(kv_after=256, count=768), {}, b"kv_after"),
    (dict(kv_len=512, count=512, kv_after=768), {}, b"count"),
    (dict(pages=None), {}, b"pages"), ({}, dict(page_size=24), b"page_size"),
    ({}, dict(type=0), b"fp16 or bf16"), ({}, dict(k_slot=0), b"strides"),
    ({}, dict(head_dim=63), b"odd")])
def test_accept_refusals(lib, kw, ckw, text):
    at = (ctypes.c_void_p * 2)(256, 512)
    assert lib.warp_tree_accept(ctypes.byref(accept_desc(**kw)), ctypes.byref(kv_pages(**ckw)), 2,
                                at, at, None) == -1
    assert text in lib.warp_last_error()


def test_accept_refuses_each_cache(lib):
    for bad in (None, 264):
        at = (ctypes.c_void_p * 2)(256, bad)
        good = (ctypes.c_void_p * 2)(256, 512)
        for k, v in ((at, good), (good, at)):
            assert lib.warp_tree_accept(ctypes.byref(accept_desc()), ctypes.byref(kv_pages()), 2, k,
                                        v, None) == -1
    assert lib.warp_tree_accept(ctypes.byref(accept_desc()), None, 1, good, good, None) == -1
    assert lib.warp_tree_accept(ctypes.byref(accept_desc()), ctypes.byref(kv_pages()), -1, good,
                                good, None) == -1


@pytest.mark.parametrize("k, v", [((256, 256), (512, 768)), ((512, 768), (256, 256)),
                                  ((256, 512), (768, 256)), ((256, 512), (256, 512))])
def test_accept_refuses_a_cache_twice(lib, k, v):
    k, v = ((ctypes.c_void_p * 2)(*x) for x in (k, v))
    assert lib.warp_tree_accept(ctypes.byref(accept_desc()), ctypes.byref(kv_pages()), 2, k, v,
                                None) == -1
    assert b"twice" in lib.warp_last_error()


def test_pool_on_the_host():
    pool = ops.page_pool(5, device="cpu")
    assert pool.dtype is torch.int32 and pool.tolist() == [5, 4, 3, 2, 1, 0]
    assert ops.page_pool(0, device="cpu").tolist() == [0]


def test_wrappers_refuse_host_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    seen = torch.zeros(2, 1, dtype=torch.int64)
    q = torch.zeros(2, 2, 64, dtype=torch.float16)
    kp = torch.zeros(2, 16, 1, 64, dtype=torch.float16)
    for call in (lambda: ops.step_plan(i, i[:1], i[None], 16, 2),
                 lambda: ops.tree_attention(q, kp, kp, i[None], i[:1], i, seen, 2, 16),
                 lambda: ops.pick_tokens(torch.zeros(2, 5)),
                 lambda: ops.tree_accept(i, i, seen, i, i[:1], 2)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
