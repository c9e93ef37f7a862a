"""Gradients of rows of class scores written to memory of the caller's: over the scores, and beside them."""
import pytest
import torch

import rows_reference as ref
from test_gpu_rows import TYPES, eng, labels, rows, teacher, vector       # noqa: F401  (eng: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [3, 5000])
def test_scores_that_a_backward_pass_needs_are_missed_when_overwritten(eng, k):
    """log_probs keeps the scores for its backward pass; a gradient written over them must not be taken for them."""
    from cutdet import losses
    n = 6
    ids, (at, te) = labels(n, k), teacher(n, k, 4)
    for way in (lambda x: eng.distill(x, at, te, grad=True, out=x),
                lambda x: eng.distill_backward(x, at, te, eng.distill(x, at, te)["stats"], vector(n, 2), out=x),
                lambda x: eng.log_probs_backward(x, ids, eng.log_probs(x)["stats"], None, vector(n, 2), out=x)):
        x = rows(n, k, "f32").clone().requires_grad_()
        logp, _ = losses.log_probs(x, ids)
        way(x.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            logp.sum().backward()
        assert x.grad is None


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("k", [3, 40, 300, 1001, 5003, 33001, 70001])
def test_gradients_between_the_rows_of_scores(eng, k, dtype):
    """Scores and gradient as the two parts of every row of one buffer, in either order."""
    n, pad = 9, 3
    ids, (at, te) = labels(n, k), teacher(n, k, 5)
    gl, gh = vector(n, 3), vector(n, 4)
    for first in (True, False):
        buf = torch.full((n, 2 * k + pad), 7.0, dtype=TYPES[dtype], device="cuda")
        x, out = (buf[:, :k], buf[:, k + pad:]) if first else (buf[:, k + pad:], buf[:, :k])
        x.copy_(rows(n, k, dtype))
        kept = x.clone()
        r = eng.log_probs(x, ids)
        eng.log_probs_backward(x, ids, r["stats"], r["entropy"], gl, gh, out=out)
        ref.check_grad(out, *ref.log_probs_grad64(kept, ids, gl, gh), k)
        loss, size, grad, gsize = ref.distill64(kept, at, te)
        d = eng.distill(x, at, te, grad=True, out=out)
        ref.check_loss(d["loss"], loss, size, k)
        ref.check_grad(out, grad, gsize, k)
        out.zero_()
        eng.distill_backward(x, at, te, d["stats"], gl, out=out)
        g = gl.double()[:, None]
        ref.check_grad(out, grad * g, gsize * g.abs(), k)
        assert torch.equal(x, kept) and (buf[:, k:k + pad] == 7).all()
