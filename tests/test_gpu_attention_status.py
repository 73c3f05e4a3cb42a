"""What the attention kernels leave out is reported, wherever they ran."""
import pytest
import torch

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu


def test_status_waits_for_other_streams(cuda):
    """A call on a stream of its own, behind earlier work there, is seen."""
    from warp_b200 import ffi, ops
    c = Case([1], [200], 8, 2, 64, 16, torch.bfloat16, seed=31)
    args = [x.cuda() for x in (c.q, c.k, c.v, c.pages, c.kv_len, c.q_start)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for max_kv in (200, 100):
            ops.attn_status()
            torch.cuda._sleep(100_000_000)      # some 50 ms
            ops.paged_attention(*args, 1, max_kv)
            if max_kv == 200:
                ops.attn_status()
    with pytest.raises(ffi.WarpError, match="length"):
        ops.attn_status()
    torch.cuda.synchronize()
    ops.attn_status()                           # cleared for good


def test_status_keeps_what_it_is_not_to_clear(cuda):
    from warp_b200 import ffi, ops
    c = Case([1], [200], 8, 2, 64, 16, torch.bfloat16, seed=32)
    args = [x.cuda() for x in (c.q, c.k, c.v, c.pages, c.kv_len, c.q_start)]
    ops.attn_status()
    ops.paged_attention(*args, 1, 100)
    for clear in (False, False, True):
        with pytest.raises(ffi.WarpError, match="length"):
            ops.attn_status(clear)
    ops.attn_status()
