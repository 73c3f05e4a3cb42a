"""What of the attention operators runs without a device: rotary frequencies
and the refusals of the C entry points."""
import ctypes
import math

import pytest
import torch

from warp_b200 import ffi, ops


@pytest.fixture(scope="module")
def lib():
    from warp_b200 import build
    build.build()
    return ffi.load()


def test_frequencies_plain():
    f, s = ops.rope_inv_freq(64, base=5e5)
    assert f.dtype == torch.float64 and f.numel() == 32 and s == 1.0
    for i in (0, 7, 31):
        assert math.isclose(f[i].item(), 5e5 ** (-2 * i / 64), rel_tol=1e-14)


def test_frequencies_scaled():
    f, _ = ops.rope_inv_freq(64)
    g, s = ops.rope_inv_freq(64, scaling="linear", factor=4.0)
    assert s == 1.0 and torch.allclose(g * 4, f, rtol=1e-14)
    # ntk: the slowest pair is divided by the factor, the fastest stays
    g, s = ops.rope_inv_freq(64, scaling="ntk", factor=4.0)
    assert s == 1.0 and g[0] == 1.0 and math.isclose(g[-1] * 4, f[-1], rel_tol=1e-12)
    # yarn: fast pairs as they are, slow ones divided by the factor
    g, s = ops.rope_inv_freq(64, scaling="yarn", factor=4.0, trained=4096)
    turns = 4096 * f / (2 * math.pi)
    assert math.isclose(s, 0.1 * math.log(4.0) + 1)
    assert torch.equal(g[turns > 64], f[turns > 64])
    assert torch.allclose(g[turns < 0.5] * 4, f[turns < 0.5], rtol=1e-14)
    assert (g <= f).all() and (g >= f / 4 * (1 - 1e-12)).all()


@pytest.mark.parametrize("kw", [dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=8, scaling="x"),
                                dict(rot_dim=8, scaling="linear", factor=0.5),
                                dict(rot_dim=2, scaling="ntk", factor=2.0),
                                dict(rot_dim=8, scaling="yarn", factor=2.0)])
def test_frequencies_refused(kw):
    with pytest.raises(ValueError):
        ops.rope_inv_freq(**kw)


def rope_desc(**kw):
    d = ffi.RopeDesc()
    good = dict(tokens=1, q_heads=2, kv_heads=1, head_dim=64, type=1, out_type=1, q=256, k=256,
                v=256, q_out=256, k_out=256, inv_freq=256, rot_dim=64, positions=256)
    for k, v in {**good, **kw}.items():
        setattr(d, k, v)
    return d


def kv_pages(**kw):
    c = ffi.KVPages()
    good = dict(k=256, v=256, type=1, page_size=16, kv_heads=1, head_dim=64, pages=4, k_page=1024,
                k_slot=64, k_head=64, v_page=1024, v_slot=64, v_head=64)
    for k, v in {**good, **kw}.items():
        setattr(c, k, v)
    return c


def attn_desc(**kw):
    d = ffi.AttnDesc()
    good = dict(batch=1, tokens=1, q_heads=2, kv_heads=1, head_dim=64, type=1, q=256, q_token=128,
                q_head=64, out=256, q_start=256, kv_len=256, pages=256, pages_row=4,
                pages_per_row=4, max_q=1, max_kv=64, causal=1, scale=0.125)
    for k, v in {**good, **kw}.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw, text", [
    (dict(tokens=-1), b"negative"), (dict(head_dim=63), b"head_dim"),
    (dict(head_dim=258), b"head_dim"), (dict(rot_dim=66), b"rot_dim"),
    (dict(rot_dim=3), b"rot_dim"), (dict(type=1, out_type=2), b"type"),
    (dict(type=3), b"type"), (dict(out_type=-1), b"type"), (dict(q=None), b"queries"),
    (dict(k=None), b"keys"), (dict(k_out=None), b"keys"), (dict(positions=None), b"positions"),
    (dict(inv_freq=None), b"inv_freq"), (dict(q_heads=70000), b"heads")])
def test_rope_refusals(lib, kw, text):
    assert lib.warp_qk_norm_rope(ctypes.byref(rope_desc(**kw)), None) == -1
    assert text in lib.warp_last_error()
    assert lib.warp_qk_norm_rope(None, None) == -1
    assert lib.warp_qk_norm_rope(ctypes.byref(rope_desc(tokens=0)), None) == 0


@pytest.mark.parametrize("kw, ckw, text", [
    (dict(v=None), {}, b"values"), (dict(out_type=2, type=2), {}, b"pages'"),
    ({}, dict(type=0), b"fp16 or bf16"), ({}, dict(page_size=24), b"page_size"),
    ({}, dict(page_size=8), b"page_size"), ({}, dict(kv_heads=2), b"heads"),
    ({}, dict(head_dim=128), b"heads"), ({}, dict(k=None), b"NULL pages"),
    ({}, dict(k=264), b"16-byte"), ({}, dict(k_slot=68), b"strides"),
    ({}, dict(v_page=-64), b"strides"), ({}, dict(pages=0), b"pages")])
def test_append_refusals(lib, kw, ckw, text):
    rc = lib.warp_kv_append(ctypes.byref(rope_desc(**kw)), ctypes.byref(kv_pages(**ckw)),
                            ctypes.c_void_p(256), None)
    assert rc == -1 and text in lib.warp_last_error()
    assert lib.warp_kv_append(ctypes.byref(rope_desc()), ctypes.byref(kv_pages()), None,
                              None) == -1
    assert lib.warp_kv_append(ctypes.byref(rope_desc()), None, None, None) == -1


@pytest.mark.parametrize("ckw", [dict(k_slot=0), dict(v_page=0), dict(kv_heads=2, k_head=0),
                                 dict(kv_heads=2, v_head=0)])
def test_broadcast_pages_are_refused(lib, ckw):
    """A stride of 0 has a meaning only where there is one entry."""
    heads = ckw.get("kv_heads", 1)
    c = kv_pages(**ckw)
    assert lib.warp_kv_append(ctypes.byref(rope_desc(kv_heads=heads)), ctypes.byref(c),
                              ctypes.c_void_p(256), None) == -1
    assert b"strides" in lib.warp_last_error()
    d = attn_desc(kv_heads=heads, max_q=100, tokens=100)
    assert lib.warp_attn_scratch(ctypes.byref(d), ctypes.byref(c)) == -1
    one = kv_pages(k_head=0, v_head=0, pages=1, k_page=0, v_page=0)
    assert lib.warp_attn_scratch(ctypes.byref(attn_desc()), ctypes.byref(one)) >= 0


@pytest.mark.parametrize("kw, ckw, text", [
    (dict(tokens=-1), {}, b"negative"), (dict(q_heads=3, kv_heads=2), dict(kv_heads=2), b"over"),
    (dict(q_heads=0), {}, b"over"), (dict(head_dim=96), dict(head_dim=96), b"head_dim"),
    (dict(type=2), {}, b"type"), (dict(type=0), dict(type=0), b"fp16 or bf16"),
    (dict(scale=0.0), {}, b"scale"), (dict(scale=float("nan")), {}, b"scale"),
    (dict(scale=float("inf")), {}, b"scale"), (dict(max_kv=1 << 30), {}, b"2^30"),
    (dict(batch=70000), {}, b"65535"), (dict(q=None), {}, b"NULL"), (dict(pages=None), {}, b"page"),
    (dict(prefix_len=5), {}, b"prefix"), (dict(q=264), {}, b"16-byte"),
    (dict(q_token=100), {}, b"strides"), (dict(kv_len=None), {}, b"NULL")])
def test_attention_refusals(lib, kw, ckw, text):
    rc = lib.warp_paged_attention(ctypes.byref(attn_desc(**kw)), ctypes.byref(kv_pages(**ckw)),
                                  ctypes.c_void_p(256), None)
    assert rc == -1 and text in lib.warp_last_error()


def test_attention_nothing_to_do(lib):
    for kw in (dict(tokens=0), dict(batch=0), dict(max_q=0)):
        d = attn_desc(**kw)
        assert lib.warp_attn_scratch(ctypes.byref(d), ctypes.byref(kv_pages())) >= 0
        assert lib.warp_paged_attention(ctypes.byref(d), ctypes.byref(kv_pages()), None, None) == 0


@pytest.mark.parametrize("fmt, cls", [("KV_PAGES", "KVPages"), ("ROPE_DESC", "RopeDesc"),
                                      ("ATTN_DESC", "AttnDesc")])
def test_packed_descriptions_match_the_structures(fmt, cls):
    fmt, cls = getattr(ffi, fmt), getattr(ffi, cls)
    values = list(range(1, len(cls._fields_) + 1))
    raw = fmt.pack(*values)
    assert fmt.size == ctypes.sizeof(cls)
    d = cls.from_buffer_copy(raw)
    assert [getattr(d, name) for name, _ in cls._fields_] == values


def test_slots_refusals(lib):
    p = ctypes.c_void_p(256)
    assert lib.warp_kv_slots(p, p, 1, 1, p, 4, 4, 12, 0, p, p, None) == -1
    assert lib.warp_kv_slots(p, p, -1, 1, p, 4, 4, 16, 0, p, p, None) == -1
    assert lib.warp_kv_slots(None, p, 1, 1, p, 4, 4, 16, 0, p, p, None) == -1
    assert lib.warp_kv_slots(None, None, 0, 0, None, 0, 0, 16, 0, None, None, None) == 0


def test_wrapper_refuses_host_tensors():
    x = torch.zeros(1, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.qk_norm_rope(x, x, None, None)
