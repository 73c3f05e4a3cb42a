"""More requests than fit 31 bits of the counting kernel's threads."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_pick_of_two_million_requests(cuda):
    """A small vocabulary, a short history each: 2^21 blocks of 1024 threads and more."""
    from warp_b200 import ops
    B, V, H = (1 << 21) + 1031, 8, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(B, V, generator=g, device="cuda")
    history = torch.randint(0, V, (B, H), generator=g, device="cuda", dtype=torch.int32)
    lens = torch.randint(0, H + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    presence = torch.rand(B, generator=g, device="cuda")
    out = torch.empty_like(x)
    picked = ops.pick_tokens(x, history=history, history_len=lens, presence=presence, out=out)
    ops.attn_status()
    hit = torch.zeros(B, V, device="cuda")
    held = (torch.arange(H, device="cuda") < lens[:, None]).float()
    hit.scatter_add_(1, history.long(), held)
    want = torch.where(hit > 0, x - presence[:, None], x)
    assert torch.equal(out, want)
    best = want.max(1).values
    assert torch.equal(want.gather(1, picked[:, None].long())[:, 0], best)
    assert torch.equal((want == best[:, None]).float().argmax(1).int(), picked)
