"""A step's plan reports the keys it has no place for."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def plan(q_start, kv_len, pages, tokens):
    from warp_b200 import ops
    i32 = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (q_start, kv_len, pages)]
    ops.attn_status()
    return [x.tolist() for x in ops.kv_slots(*i32, 16, tokens)]


def test_negative_page_is_reported(cuda):
    from warp_b200 import ffi, ops
    pos, slots = plan([0, 2, 3], [18, 5], [[4, -1], [2, -1]], 3)
    assert pos == [16, 17, 4] and slots == [-1, -1, 36]
    with pytest.raises(ffi.WarpError, match="page number"):
        ops.attn_status()
    ops.attn_status()


def test_key_past_the_row_is_reported(cuda):
    from warp_b200 import ffi, ops
    pos, slots = plan([0, 2], [33], [[4, 0]], 2)
    assert pos == [31, 32] and slots == [15, -1]
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()
    ops.attn_status()


def test_tokens_without_a_key_are_not(cuda):
    """More queries than keys, a request without any and tokens of no request."""
    from warp_b200 import ops
    _, slots = plan([0, 3, 4, 4], [2, 0, 16], [[1], [-1], [-1]], 6)
    assert slots == [-1, 16, 17, -1, -1, -1]
    ops.attn_status()
