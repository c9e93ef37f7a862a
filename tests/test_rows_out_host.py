"""Where the operators on rows of class scores write a gradient: what torch and the library know of that memory (no GPU)."""
import ctypes as C

import pytest
import torch

N, K = 4, 6
IDS = torch.zeros(N, 2, dtype=torch.int64)
TEACHER, STATS, ROW = torch.zeros(N, 2), torch.zeros(N, 2), torch.zeros(N)


@pytest.fixture
def host_engine(monkeypatch):
    """An Engine on CPU tensors whose library calls succeed and compute nothing."""
    from cutdet import engine

    class Library:
        rc = 0

        def __getattr__(self, name):
            return lambda *args: self.rc

    eng = engine.Engine.__new__(engine.Engine)
    eng.device, eng._h = torch.device("cpu"), C.c_void_p(0)
    eng._new_f32, eng._new_i64 = torch.zeros(0).new_empty, IDS.new_empty
    eng._stream = lambda: None
    eng.library = Library()
    monkeypatch.setattr(engine, "lib", eng.library)
    return eng


def ways(eng, x, out):
    return {"log_probs_backward": lambda: eng.log_probs_backward(x, IDS[:, 0], STATS, ROW, ROW, ROW, out=out),
            "distill": lambda: eng.distill(x, IDS, TEACHER, grad=True, out=out),
            "distill_backward": lambda: eng.distill_backward(x, IDS, TEACHER, STATS, ROW, out=out)}


@pytest.mark.parametrize("way", ["log_probs_backward", "distill", "distill_backward"])
def test_a_gradient_over_the_scores_counts_as_a_change_of_them(host_engine, way):
    x = torch.zeros(N, K, requires_grad=True)
    loss = (x * x).sum()                                      # saves x
    before = x._version
    ways(host_engine, x.detach(), None)[way]()
    assert x._version == before                               # a gradient of its own changes nothing
    ways(host_engine, x.detach(), x.detach())[way]()
    assert x._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():                              # (such a tensor has no count)
        y = torch.zeros(N, K)
        assert ways(host_engine, y, y)[way]() is not None


def test_a_refused_call_changes_nothing(host_engine):
    from cutdet import _lib
    x = torch.zeros(N, K)
    host_engine.library.rc = _lib.CD_EINVAL
    for call in ways(host_engine, x, x).values():
        with pytest.raises(_lib.CutdetError):
            call()
    assert x._version == 0
