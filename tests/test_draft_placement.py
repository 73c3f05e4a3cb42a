"""Every tensor of a call on drafted tokens has to be on the current device: stand-ins
that say where they are, and a library that must not be reached."""
import pytest
import torch

from test_attention_placement import Reached, attend, batch, device_0, on  # noqa: F401
from warp_b200 import ops


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def seen(tokens):
    return torch.zeros(tokens, 1, dtype=torch.int64)


def plan():
    x = dict(batch(), held=i32(1), pool=i32(3), parents=i32(3))
    return lambda **x: ops.step_plan(page_size=16, tokens=3, max_q=3, **x), x


def tree():
    x = dict(attend()[1], seen=seen(3))
    return lambda **x: ops.tree_attention(max_q=3, max_kv=16, prefix_len=5, **x), x


def pick():
    x = dict(logits=torch.zeros(3, 40), q_start=i32(2), history=i32(1, 7), history_len=i32(1),
             repetition=torch.zeros(1), frequency=torch.zeros(1), presence=torch.zeros(1),
             bias=torch.zeros(1, 40), allowed=i32(3, 2), drafted=i32(3), seen=seen(3),
             out=torch.zeros(3, 40))
    return lambda **x: ops.pick_tokens(max_q=3, **x), x


def accept():
    pair = dict(k=torch.zeros(2, 4, 16, 2, 64, dtype=torch.float16),
                v=torch.zeros(2, 4, 16, 2, 64, dtype=torch.float16))
    x = dict(batch(), drafted=i32(3), picked=i32(3), seen=seen(3), **pair)
    return lambda k, v, **x: ops.tree_accept(max_q=3, caches=(k, v), **x), x


def accept_list():
    call, x = accept()
    x.update(k=x["k"][0], v=x["v"][0])
    return lambda k, v, **x: ops.tree_accept(max_q=3, caches=[(k, v)], **x), x


def accept_alone():
    x = accept()[1]
    for name in ("k", "v", "pages"):
        del x[name]
    return lambda **x: ops.tree_accept(max_q=3, **x), x


CALLS = dict(plan=plan, tree=tree, pick=pick, accept=accept, accept_list=accept_list,
             accept_alone=accept_alone)
EACH = [(n, k) for n in CALLS for k in CALLS[n]()[1]]


@pytest.mark.parametrize("name", CALLS)
def test_all_here_reaches_the_library(name):
    call, x = CALLS[name]()
    with pytest.raises(Reached):
        call(**{k: on(v) for k, v in x.items()})


@pytest.mark.parametrize("name, which", EACH)
def test_one_elsewhere_is_refused(name, which):
    call, x = CALLS[name]()
    with pytest.raises(ValueError, match="not the current device"):
        call(**{k: on(v, int(k == which)) for k, v in x.items()})


@pytest.mark.parametrize("name, which", EACH)
def test_one_on_the_host_is_refused(name, which):
    call, x = CALLS[name]()
    with pytest.raises(ValueError, match="CUDA tensors"):
        call(**{k: v if k == which else on(v) for k, v in x.items()})
