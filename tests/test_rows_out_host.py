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
    monkeypatch.setattr(engine, "_rows_workspace", lambda *args: 0)
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


# ---- which memory the library takes for a gradient ---------------------------------------------------------------
BASE, WIDE = 1 << 40, 1 << 15                   # an address that nothing reads; rows of 128 KB in 32 bits


def distill_with_gradient_at(offset, grad_stride, n=4, stride=WIDE, k=WIDE):
    """What cd_distill answers for scores at BASE and a gradient `offset` elements behind; rows this long need a
    workspace, which is checked last and missing here, so that no call gets further."""
    from cutdet import _lib
    assert _lib.lib.cd_rows_workspace(n, k, _lib.CD_T_F32, 0) > 0
    some = C.cast(C.create_string_buffer(64), C.c_void_p)
    return _lib.lib.cd_distill(some, BASE, _lib.CD_T_F32, n, k, stride, 1.0, some, some, _lib.CD_T_F32, 3, None, some, some,
                               BASE + 4 * offset, grad_stride, None, 0, None)


@pytest.mark.parametrize("offset,grad_stride,n,stride,ok", [
    (WIDE, 2 * WIDE, 4, 2 * WIDE, True),                      # the other half of every row of one buffer
    (-WIDE, 2 * WIDE, 4, 2 * WIDE, True),
    (WIDE - 1, 2 * WIDE, 4, 2 * WIDE, False),
    (1 - WIDE, 2 * WIDE, 4, 2 * WIDE, False),
    (5 * WIDE, 2 * WIDE, 4, 2 * WIDE, True),                  # the same, two rows further on
    (5 * WIDE + 1, 2 * WIDE, 4, 2 * WIDE, False),
    (0, 2 * WIDE, 4, 2 * WIDE, True),                         # the scores themselves
    (2 * WIDE, 2 * WIDE, 4, 2 * WIDE, False),                 # ... a row further on
    (6 * WIDE, 2 * WIDE, 4, 2 * WIDE, False),
    (8 * WIDE, 2 * WIDE, 4, 2 * WIDE, True),
    (0, 2 * WIDE, 1, WIDE, True),
    (0, 2 * WIDE, 4, WIDE, False),                            # other strides
    (3 * WIDE, 5 * WIDE, 2, 8 * WIDE, False),
    (WIDE, 3 * WIDE, 2, 5 * WIDE, True),                      # scores 0, 5; gradients 1, 4
    (WIDE, 4 * WIDE, 2, 5 * WIDE, False),                     # scores 0, 5; gradients 1, 5
    (-3 * WIDE, 4 * WIDE, 4, 0, True),                        # one row of scores for all, in a gap
    (-4 * WIDE + 1, 4 * WIDE, 4, 0, False),
])
def test_a_gradient_may_lie_between_the_rows_of_scores(offset, grad_stride, n, stride, ok):
    from cutdet import _lib
    want = _lib.CD_ECAP if ok else _lib.CD_EINVAL
    assert distill_with_gradient_at(offset, grad_stride, n, stride) == want
    assert (b"workspace" if ok else b"overlaps") in _lib.lib.cd_last_error()


def test_memory_of_scores_and_gradients_against_every_element():
    """Random strides and distances, against a comparison of every row with every other."""
    import random

    from cutdet import _lib
    rng, seen = random.Random(7), set()
    for _ in range(4000):
        n = rng.randint(1, 6)
        unit = rng.choice([1, 64, WIDE // 4])
        stride = rng.choice([0, WIDE // 2, WIDE, WIDE + unit, 2 * WIDE, 3 * WIDE, 3 * WIDE + unit])
        grad_stride = rng.choice([WIDE, WIDE + unit, 2 * WIDE, 3 * WIDE, 3 * WIDE + unit, 7 * WIDE])
        offset = unit * rng.randint(-8 * WIDE // unit, 20 * WIDE // unit) if rng.random() < 0.9 else 0
        apart = all(abs(i * stride - (offset + j * grad_stride)) >= WIDE for i in range(n) for j in range(n))
        ok = apart or (offset == 0 and (n == 1 or stride == grad_stride))
        assert distill_with_gradient_at(offset, grad_stride, n, stride) == (_lib.CD_ECAP if ok else _lib.CD_EINVAL), \
            (n, stride, grad_stride, offset)
        seen.add((ok, stride == grad_stride))
    assert len(seen) == 4
