"""The serving operators' binding on tensors of the wrong place (CPU: stand-ins
for device tensors; nothing is launched)."""
import contextlib

import pytest
import torch

import bq


class Fake:
    """What the binding looks at of a device tensor."""

    def __init__(self, dtype, *shape, index=0, cuda=True, contiguous=True):
        self.dtype, self.shape, self.is_cuda, self._c = dtype, tuple(shape), cuda, contiguous
        self.device = torch.device("cuda", index) if cuda else torch.device("cpu")

    def dim(self):
        return len(self.shape)

    def stride(self, i):
        n = 1
        for s in self.shape[i + 1:]:
            n *= s
        return n

    def is_contiguous(self):
        return self._c

    def data_ptr(self):
        return 1 << 20

    def numel(self):
        return self.stride(0) * self.shape[0]

    def element_size(self):
        return self.dtype.itemsize


I, F = torch.int32, torch.float32
D, P = 64, 16


def _cache(table=None):
    return bq.KvCache(Fake(torch.uint8, 4, bq.kv_page_bytes("bf16", 1, D, P)), table or Fake(I, 1, 2), "bf16", 1, D, P)


ARGS = {"append": dict(q=(F, 3, D), k=(F, 3, D), v=(F, 3, D), pos=(I, 3), q_out=(F, 3, D), seq=(I, 3), q_weight=(F, D), k_weight=(F, D),
                       rope=(F, 8, D)),
        "attention": dict(q=(F, 1, D), out=(F, 1, D), kv_len=(I, 1), row0=(I, 2), work=(F, 100)),
        "sampler": dict(logits=(F, 2, 100), out=(I, 2), u=(F, 2), temperature=(F, 2), top_k=(I, 2), top_p=(F, 2), min_p=(F, 2),
                        work=(torch.uint8, 1 << 20))}


def _make(op, name=None, **how):
    """The operator's object over tensors of device 0, `name` made otherwise."""
    a = {n: Fake(*t, **(how if n == name else {})) for n, t in ARGS[op].items()}
    if op == "sampler":
        return bq.Sampler(**a)
    return (bq.Append if op == "append" else bq.Attention)(_cache(), **a)


@pytest.mark.parametrize("op", list(ARGS))
def test_tensors_of_another_device(op):
    """Each tensor on a second GPU, and on the host: refused before anything is called."""
    _make(op)
    for name in ARGS[op]:
        for how in (dict(index=1), dict(cuda=False)):
            with pytest.raises(ValueError):
                _make(op, name, **how)
    with pytest.raises(ValueError):
        _cache(Fake(I, 1, 2, index=1))


def test_workspaces_that_are_not_there():
    """A strided or expanded workspace has fewer bytes in a row than its elements say."""
    for op in ("attention", "sampler"):
        with pytest.raises(ValueError):
            _make(op, "work", contiguous=False)


@pytest.mark.parametrize("current", [0, 1])
def test_calls_go_to_the_tensors_device(monkeypatch, current):
    """The launch, not only the stream, is the tensors' device's, whichever is current; the current one comes back."""
    now, seen = [current], []

    @contextlib.contextmanager
    def device(d):
        before, now[0] = now[0], d
        yield
        now[0] = before
    bq._bind_device()
    monkeypatch.setattr(bq, "_current", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(bq, "_raw_stream", lambda d: 1000 + d)
    call = lambda *a: seen.append((now[0], a[-1])) or 0
    for run, obj, name in (("run", _make("append"), "_run"), ("decode", _make("attention"), "_decode"), ("prefill", _make("attention"), "_prefill"),
                           ("run", _make("sampler"), "_run")):
        setattr(obj, name, call)
        getattr(obj, run)()
    cache = _cache()
    cache._read = call
    cache.read(Fake(I, 3), Fake(torch.bfloat16, 3, D))
    assert seen == [(0, 1000)] * 5 and now == [current]
