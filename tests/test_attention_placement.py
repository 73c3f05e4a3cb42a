"""Every tensor of an attention call has to be on the current device: stand-ins
that say where they are, and a library that must not be reached."""
import pytest
import torch

from warp_b200 import ffi, ops


class Placed(torch.Tensor):
    """A host tensor that says it is on CUDA device `at`."""
    at = 0

    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.at))

    def get_device(self):
        return self.at


def on(x, at=0):
    x = x.as_subclass(Placed)
    x.at = at
    return x


class Reached(Exception):
    pass


@pytest.fixture(autouse=True)
def device_0(monkeypatch):
    def load():
        raise Reached
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(ffi, "load", load)
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **kw: on(torch.zeros(1)))
    monkeypatch.setattr(torch, "empty_like", lambda x, **kw: on(torch.zeros(x.shape, dtype=kw.get(
        "dtype"))))


def rope():
    x = dict(q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64),
             positions=torch.zeros(3, dtype=torch.int32),
             inv_freq=torch.zeros(32, dtype=torch.float64), q_norm=torch.zeros(64),
             k_norm=torch.zeros(64))
    return ops.qk_norm_rope, x


def append():
    x = rope()[1]
    x.update(v=torch.zeros(3, 2, 64), k_pages=torch.zeros(2, 16, 2, 64, dtype=torch.float16),
             v_pages=torch.zeros(2, 16, 2, 64, dtype=torch.float16),
             slots=torch.zeros(3, dtype=torch.int64))
    return ops.kv_append, x


def batch():
    return dict(q_start=torch.zeros(2, dtype=torch.int32), kv_len=torch.zeros(1, dtype=torch.int32),
                pages=torch.zeros(1, 2, dtype=torch.int32))


def slots():
    return lambda **x: ops.kv_slots(page_size=16, tokens=3, **x), batch()


def attend():
    x = dict(q=torch.zeros(3, 4, 64, dtype=torch.float16),
             k_pages=torch.zeros(2, 16, 2, 64, dtype=torch.float16),
             v_pages=torch.zeros(2, 16, 2, 64, dtype=torch.float16),
             prefix_pages=torch.zeros(1, dtype=torch.int32),
             out=torch.zeros(3, 4, 64, dtype=torch.float16), **batch())
    return lambda **x: ops.paged_attention(max_q=3, max_kv=16, prefix_len=5, **x), x


CALLS = dict(rope=rope, append=append, slots=slots, attend=attend)


@pytest.mark.parametrize("name", CALLS)
def test_all_here_reaches_the_library(name):
    call, x = CALLS[name]()
    with pytest.raises(Reached):
        call(**{k: on(v) for k, v in x.items()})


@pytest.mark.parametrize("name, which", [(n, k) for n in CALLS for k in CALLS[n]()[1]])
def test_one_elsewhere_is_refused(name, which):
    call, x = CALLS[name]()
    with pytest.raises(ValueError, match="not the current device"):
        call(**{k: on(v, int(k == which)) for k, v in x.items()})


@pytest.mark.parametrize("name, which", [(n, k) for n in CALLS for k in CALLS[n]()[1]])
def test_one_on_the_host_is_refused(name, which):
    call, x = CALLS[name]()
    with pytest.raises(ValueError, match="CUDA tensors"):
        call(**{k: v if k == which else on(v) for k, v in x.items()})


def test_one_side_elsewhere():
    for q, k in ((None, 1), (1, None)):
        x = rope()[1]
        x = {n: on(v) for n, v in x.items()}
        x["q"] = None if q is None else on(x["q"], q)
        x["k"] = None if k is None else on(x["k"], k)
        with pytest.raises(ValueError, match="not the current device"):
            ops.qk_norm_rope(**x)
