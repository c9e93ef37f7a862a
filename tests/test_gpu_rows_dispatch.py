"""Every way that rows of class scores are taken apart, by number of rows, length, type and what is asked for: sizes just past
each limit, and each way with the gradient over the scores."""
import pytest
import torch

import rows_reference as ref
from test_gpu_rows import (TYPES, check_backward, check_distill, check_log_probs, eng, labels, rows,      # noqa: F401
                           teacher, vector)

pytestmark = pytest.mark.gpu

# rows and classes of 32 bits, threads of the workgroup that a row has; 16 bits: twice the classes
BLOCKS = [(600, 2500, 128), (600, 4001, 128), (100, 4001, 256), (600, 5003, 256), (300, 5003, 512), (520, 20000, 512),
          (800, 16500, 256), (1537, 16500, 512), (70, 20000, 1024)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,k,threads", BLOCKS)
def test_log_probs_by_workgroups(eng, n, k, threads, dtype):
    k = k if dtype == "f32" else 2 * k
    x, ids = rows(n, k, dtype, pad=3), labels(n, k)
    for top, t in ((1, 1.0), (25, 0.7), (64, 1.0)):
        check_log_probs(eng, x, ids, top, t, entropy=top != 25)
    check_backward(eng, x, ids)


def with_weights(n):
    w = vector(n, 5).abs() + 0.1
    w[::3] = 0.0
    return w


# loss and gradient from registers (256 x 8 vectors, 512 x 8, 512 x 16, 1024 x 16), and in two passes
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,k", [(600, 2500), (600, 4500), (300, 8192), (65, 8197), (300, 12000), (70, 20000), (130, 32768),
                                 (65, 32773), (130, 40000), (65, 65540), (70, 70001), (300, 70001), (800, 70001)])
def test_distill_by_workgroups(eng, n, k, dtype):
    k = k if dtype == "f32" else 2 * k
    x = rows(n, k, dtype, pad=1)
    for entries, t in ((20, 1.0), (65, 2.0), (256, 0.7)):
        if n * k > 3e7 and entries == 65:
            continue
        ids, te = teacher(n, k, entries, 1)
        check_distill(eng, x, ids, te, with_weights(n) if entries == 20 else None, t)


# a thread, 16 lanes, a wave (one score at a time; vectors), registers of workgroups, two passes, several workgroups per row
WAYS = [(20, 3, "f32"), (20, 16, "bf16"), (20, 60, "f32"), (20, 200, "f16"), (20, 500, "f32"), (20, 1000, "bf16"),
        (20, 2000, "f32"), (20, 4000, "bf16"), (20, 3001, "f32"), (20, 12001, "f32"), (70, 40001, "f16"),
        (70, 80001, "bf16"), (70, 70001, "f32"), (5, 70001, "f32"), (2, 200003, "bf16")]


@pytest.mark.parametrize("entries", [3, 40, 130])
@pytest.mark.parametrize("n,k,dtype", WAYS)
def test_gradients_over_the_scores(eng, n, k, dtype, entries):
    """The same bits as in memory of its own, which begins at the same place of a 128-byte line."""
    x, ids = rows(n, k, dtype).clone(), labels(n, k)
    at, te = teacher(n, k, entries, 2)
    w, g, gh = with_weights(n), vector(n, 7), vector(n, 8)
    assert x.data_ptr() % 128 == 0
    apart = eng.distill(x, at, te, w, 1.5, grad=True)
    assert apart["grad"].data_ptr() % 128 == 0
    loss, size, grad, gsize = ref.distill64(x, at, te, w, 1.5)
    ref.check_grad(apart["grad"], grad, gsize, k)
    same = x.clone()
    over = eng.distill(same, at, te, w, 1.5, grad=True, out=same)
    assert over["grad"].data_ptr() == same.data_ptr()
    for key in ("loss", "stats", "grad"):
        assert torch.equal(over[key], apart[key]), key
    late = eng.distill_backward(x, at, te, apart["stats"], g, w, 1.5)
    ref.check_grad(late, grad * g.double()[:, None], gsize * g.double().abs()[:, None], k)
    same = x.clone()
    assert torch.equal(eng.distill_backward(same, at, te, apart["stats"], g, w, 1.5, out=same), late)
    r = eng.log_probs(x, ids)
    want = eng.log_probs_backward(x, ids, r["stats"], r["entropy"], g, gh)
    same = x.clone()
    assert torch.equal(eng.log_probs_backward(same, ids, r["stats"], r["entropy"], g, gh, out=same), want)
