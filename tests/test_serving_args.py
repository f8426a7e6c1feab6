"""Argument checks of the session's serving calls that come before any call of
the library, on stand-ins (no GPU)."""
from types import SimpleNamespace

import numpy as np
import pytest

import myelith_b200 as myl
from myelith_b200.model import Session

torch = pytest.importorskip("torch")


class Logits:
    """A CUDA tensor as far as the checks look at it."""

    def __init__(self, device, shape=(1, 2, 5), dtype=torch.int32, contiguous=True):
        self.dtype, self.shape, self.device, self.is_cuda = dtype, torch.Size(shape), f"cuda:{device}", device >= 0
        self._device, self._contiguous = device, contiguous

    def get_device(self):
        return self._device

    def dim(self):
        return len(self.shape)

    def stride(self, d=None):
        s = (self.shape[1] * self.shape[2], self.shape[2], 1)
        return s if d is None else s[d]

    def numel(self):
        return self.shape.numel()

    def is_contiguous(self):
        return self._contiguous


@pytest.fixture
def session(monkeypatch):
    import myelith_b200.model as mod

    def reached():
        raise AssertionError("the library was reached")

    monkeypatch.setattr(mod, "_lib", reached)
    s = Session.__new__(Session)
    s._h, s.batch = None, 1
    s.model = SimpleNamespace(ctx=SimpleNamespace(device=0, handle=None), handle=None, vocab=5)
    return s


@pytest.mark.parametrize("bad", [dict(device=1), dict(device=-1), dict(device=0, dtype=torch.int64),
                                 dict(device=0, shape=(1, 3, 5)), dict(device=0, shape=(1, 2, 6)),
                                 dict(device=0, contiguous=False)])
def test_forward_logits_takes_a_tensor_of_its_own_device(session, bad):
    with pytest.raises(myl.MylError):
        session.forward_logits_dev(np.zeros((1, 2), np.int32), Logits(**bad))


def test_set_adapters_refuses_an_unknown_projection(session):
    with pytest.raises(myl.MylError):
        session.set_adapters(0, "mlp", None)
