"""Gradients of rows of class scores written to memory of the caller's: over the scores, and beside them."""
import pytest
import torch

from test_gpu_rows import eng, labels, rows, teacher, vector       # noqa: F401  (eng: the fixture)

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
