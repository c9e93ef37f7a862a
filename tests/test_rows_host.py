"""Operators on rows of class scores: the checks of their arguments (no GPU), and the 64-bit reference against differences."""
import ctypes as C
import math

import pytest
import torch

import rows_reference as ref


@pytest.fixture(scope="module")
def lib():
    from cutdet import _lib
    return _lib


BUF = C.create_string_buffer(1 << 16)          # stands for handle and device memory: a refused call reads neither
PTR = C.cast(BUF, C.c_void_p)


def _at(offset):
    return C.c_void_p(C.addressof(BUF) + offset)


def _log_probs(lib, **kw):
    a = dict(h=PTR, x=_at(0), ty=0, n=2, k=5, stride=5, t=1.0, ids=None, top=0, stats=PTR, logp=None, ent=None, tl=None,
             ti=None, ws=None, wsn=0)
    a.update(kw)
    return lib.lib.cd_log_probs(a["h"], a["x"], a["ty"], a["n"], a["k"], a["stride"], a["t"], a["ids"], a["top"],
                                a["stats"], a["logp"], a["ent"], a["tl"], a["ti"], a["ws"], a["wsn"], None)


def _distill(lib, **kw):
    a = dict(h=PTR, x=_at(0), ty=0, n=2, k=5, stride=5, t=1.0, ids=PTR, te=_at(0), tt=0, e=3, w=None, stats=PTR,
             loss=PTR, g=None, gs=0)
    a.update(kw)
    return lib.lib.cd_distill(a["h"], a["x"], a["ty"], a["n"], a["k"], a["stride"], a["t"], a["ids"], a["te"], a["tt"],
                              a["e"], a["w"], a["stats"], a["loss"], a["g"], a["gs"], None, 0, None)


COMMON = [dict(h=None), dict(x=None), dict(ty=3), dict(ty=-1), dict(n=0), dict(n=-1), dict(k=0), dict(k=(1 << 30) + 1),
          dict(stride=-1), dict(n=1 << 30, stride=1 << 40), dict(t=0.0), dict(t=-1.0), dict(t=float("nan")),
          dict(t=float("inf")), dict(t=1e-6), dict(t=1e6), dict(x=_at(2)), dict(ty=1, x=_at(1)), dict(stats=None)]


@pytest.mark.parametrize("bad", COMMON + [dict(ids=PTR), dict(logp=PTR), dict(top=-1), dict(top=6, tl=PTR, ti=PTR),
                                          dict(k=100, top=65, tl=PTR, ti=PTR), dict(top=2), dict(top=2, tl=PTR)],
                         ids=lambda d: ",".join(d))
def test_log_probs_refuses(lib, bad):
    assert _log_probs(lib, **bad) == lib.CD_EINVAL
    assert b"cd_log_probs" in lib.lib.cd_last_error()


@pytest.mark.parametrize("bad", COMMON + [dict(ids=None), dict(te=None), dict(tt=7), dict(te=_at(2)), dict(e=0),
                                          dict(e=257), dict(loss=None), dict(g=_at(4096), gs=4),
                                          dict(g=_at(4098), gs=5), dict(g=_at(20), gs=5), dict(g=_at(0), gs=6)],
                         ids=lambda d: ",".join(d))
def test_distill_refuses(lib, bad):
    assert _distill(lib, **bad) == lib.CD_EINVAL
    assert b"cd_distill" in lib.lib.cd_last_error()


@pytest.mark.parametrize("bad", [dict(g=None), dict(gs=4), dict(g=_at(8)), dict(stats=None), dict(gl=PTR),
                                 dict(ge=PTR), dict(n=0), dict(t=0.0)], ids=lambda d: ",".join(d))
def test_log_probs_backward_refuses(lib, bad):
    a = dict(n=2, t=1.0, ids=None, stats=PTR, ent=None, gl=None, ge=None, g=_at(4096), gs=5)
    a.update(bad)
    rc = lib.lib.cd_log_probs_backward(PTR, _at(0), 0, a["n"], 5, 5, a["t"], a["ids"], a["stats"], a["ent"], a["gl"],
                                       a["ge"], a["g"], a["gs"], None)
    assert rc == lib.CD_EINVAL


@pytest.mark.parametrize("bad", [dict(g=None), dict(gs=4), dict(g=_at(8)), dict(stats=None), dict(gl=None), dict(e=0),
                                 dict(n=0)], ids=lambda d: ",".join(d))
def test_distill_backward_refuses(lib, bad):
    a = dict(n=2, e=3, stats=PTR, gl=PTR, g=_at(4096), gs=5)
    a.update(bad)
    rc = lib.lib.cd_distill_backward(PTR, _at(0), 0, a["n"], 5, 5, 1.0, PTR, _at(0), 0, a["e"], None, a["stats"],
                                     a["gl"], a["g"], a["gs"], None)
    assert rc == lib.CD_EINVAL


def test_workspace_is_asked_for_and_checked(lib):
    size = lib.lib.cd_rows_workspace
    assert size(0, 5, 0, 0) == 0 and size(10, 0, 0, 0) == 0 and size(1, 1 << 20, 0, 65) == 0
    assert size(200000, 3, 0, 2) == 0
    need = size(1, 1 << 20, 0, 20)
    if need:
        for ws, n in ((None, 0), (PTR, need - 1), (_at(8), need)):
            rc = _log_probs(lib, n=1, k=1 << 20, stride=1 << 20, top=20, tl=PTR, ti=PTR, ws=ws, wsn=n)
            assert rc == lib.CD_ECAP and b"workspace" in lib.lib.cd_last_error()


@pytest.fixture(scope="module")
def host_engine():
    """An Engine whose tensors would be on the CPU: every call below has to be refused before it reaches the library."""
    from cutdet.engine import Engine
    eng = Engine.__new__(Engine)
    eng.device, eng._h = torch.device("cpu"), C.c_void_p(0)
    return eng


X = torch.zeros(4, 6)
IDS = torch.zeros(4, 2, dtype=torch.int64)


@pytest.mark.parametrize("call,error", [
    (lambda e: e.log_probs([[1.0]]), RuntimeError),
    (lambda e: e.log_probs(X.to("meta")), RuntimeError),
    (lambda e: e.log_probs(X.double()), TypeError),
    (lambda e: e.log_probs(X[0]), ValueError),
    (lambda e: e.log_probs(X[:, :0]), ValueError),
    (lambda e: e.log_probs(torch.zeros(1).expand(1, (1 << 32) + 5)), ValueError),      # 5 in 32 bits
    (lambda e: e.log_probs(X, top=7), ValueError),
    (lambda e: e.log_probs(X, top=-1), ValueError),
    (lambda e: e.log_probs(torch.zeros(1, 100), top=65), ValueError),
    (lambda e: e.log_probs(X, torch.zeros(4, dtype=torch.int32)), TypeError),
    (lambda e: e.log_probs(X, torch.zeros(3, dtype=torch.int64)), ValueError),
    (lambda e: e.log_probs_backward(X, None, None, None), ValueError),
    (lambda e: e.log_probs_backward(X, None, torch.zeros(4, 2), None, torch.zeros(4)), ValueError),
    (lambda e: e.log_probs_backward(X, None, torch.zeros(4, 2), None, None, torch.zeros(4)), ValueError),
    (lambda e: e.log_probs_backward(X, None, torch.zeros(4, 3), None), ValueError),
    (lambda e: e.log_probs_backward(X, None, torch.zeros(4, 2), None, out=torch.zeros(4, 7)), ValueError),
    (lambda e: e.log_probs_backward(X, None, torch.zeros(4, 2), None, out=X.half()), TypeError),
    (lambda e: e.log_probs_backward(X, None, torch.zeros(4, 2), None, out=torch.zeros(6, 4).t()), ValueError),
    (lambda e: e.log_probs_backward(X, None, torch.zeros(4, 2), None, out=torch.zeros(6).expand(4, 6)), ValueError),
    (lambda e: e.distill(X, IDS.int(), torch.zeros(4, 2)), TypeError),
    (lambda e: e.distill(X, IDS[:3], torch.zeros(3, 2)), ValueError),
    (lambda e: e.distill(X, IDS, torch.zeros(4, 3)), ValueError),
    (lambda e: e.distill(X, IDS, torch.zeros(4, 2).double()), TypeError),
    (lambda e: e.distill(X, torch.zeros(4, 257, dtype=torch.int64), torch.zeros(4, 257)), ValueError),
    (lambda e: e.distill(X, IDS[:, :0], torch.zeros(4, 0)), ValueError),
    (lambda e: e.distill(X, IDS, torch.zeros(4, 2), torch.zeros(3)), ValueError),
    (lambda e: e.distill(X, IDS, torch.zeros(4, 2), torch.zeros(4).half()), TypeError),
    (lambda e: e.distill(X, IDS, torch.zeros(4, 2), out=torch.zeros(4, 6)), ValueError),
    (lambda e: e.distill_backward(X, IDS, torch.zeros(4, 2), None, torch.zeros(4)), ValueError),
    (lambda e: e.distill_backward(X, IDS, torch.zeros(4, 2), torch.zeros(4, 2), None), ValueError),
])
def test_engine_refuses(host_engine, call, error):
    with pytest.raises(error):
        call(host_engine)


def test_losses_refuse_cpu_tensors_and_constants_with_gradients():
    from cutdet import losses
    with pytest.raises(RuntimeError):
        losses.log_probs(X, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(TypeError):
        losses.log_probs(X, None)
    with pytest.raises(RuntimeError):
        losses.distill_loss(X, IDS, torch.zeros(4, 2))
    with pytest.raises(ValueError):
        losses.distill_loss(X, IDS, torch.zeros(4, 2, requires_grad=True))
    with pytest.raises(ValueError):
        losses.distill_loss(X, IDS, torch.zeros(4, 2), torch.zeros(4, requires_grad=True))


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_reference_gradients_against_differences(temperature):
    """The 64-bit formulas that the kernels are tested against, against central differences of their own forward."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 7, generator=g, dtype=torch.float64) * 2
    ids = torch.tensor([4, -1, 0])
    gl, gh = torch.randn(3, generator=g).double(), torch.randn(3, generator=g).double()
    at = torch.tensor([[1, 5, 1], [2, -1, 9], [-1, -1, -1]])
    te, w = torch.randn(3, 3, generator=g).double(), torch.tensor([0.5, 2.0, 1.0]).double()

    def policy(v):
        r = ref.log_probs64(v, ids, temperature)
        return float((gl * r["logp"] + gh * r["entropy"]).sum())

    def distill(v):
        return float(ref.distill64(v, at, te, w, temperature)[0].sum())

    for f, want in ((policy, ref.log_probs_grad64(x, ids, gl, gh, temperature)[0]),
                    (distill, ref.distill64(x, at, te, w, temperature)[2])):
        for i in range(3):
            for j in range(7):
                d = torch.zeros_like(x)
                d[i, j] = 1e-5
                # the third derivative is of order 1 / T^3: h^2 of it, and 2^-52 / h of rounding
                assert abs((f(x + d) - f(x - d)) / 2e-5 - float(want[i, j])) < 1e-9 / temperature ** 3 + 1e-9, (i, j)


def test_reference_orders_as_the_engine_documents():
    x = torch.tensor([[0.0, -0.0, math.nan, 1.0, 1.0, -math.inf, math.inf]])
    assert ref.top64(x, 7).tolist() == [[2, 6, 3, 4, 0, 1, 5]]
