"""Log probabilities and the distillation loss of rows of class scores, for torch's autograd.

Two functions over Engine.log_probs and Engine.distill whose results can be differentiated with respect to the scores:
the forward call keeps two numbers per row, the backward call is one kernel that reads the scores again and recomputes
the probabilities.  The scores may be float32, bfloat16 or float16 [n, k] on an MI355X; results are float32 [n].

For a step that is captured into a HIP graph, or that needs nothing but the loss and its gradient, call
Engine.distill(..., grad=True) (one pass for both) or Engine.log_probs and log_probs_backward: they use no autograd graph.
These functions refuse scores that require gradients, and their backward passes, while a stream is being captured.
"""
import torch

from . import api


def _engine(scores):
    if not torch.is_tensor(scores) or scores.device.type != "cuda":
        raise RuntimeError("cutdet.losses runs on an MI355X only; scores must be a tensor on the GPU (no CPU path)")
    return api.default_engine(scores.device)


def _not_captured():
    if torch.cuda.is_current_stream_capturing():
        # autograd keeps one accumulation node per leaf, tied to the stream of its first use; where an eager graph of
        # the same leaves is alive, a captured backward would pull that stream into the capture, which can end the process
        raise RuntimeError("gradients of a leaf cannot be captured safely into a HIP graph: use Engine.distill(..., "
                           "grad=True) or Engine.log_probs_backward there")


def _check_scores(scores):
    if torch.is_tensor(scores) and scores.is_cuda and scores.requires_grad and torch.is_grad_enabled():
        _not_captured()


def _constant(t, name):
    if t is not None and t.requires_grad:
        raise ValueError(f"{name} is a constant of the loss: detach it")
    return t


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, ids, temperature):
        eng = _engine(scores)
        r = eng.log_probs(scores, ids, temperature=temperature)
        ctx.engine, ctx.temperature = eng, temperature
        ctx.save_for_backward(scores, ids, r["stats"], r["entropy"])
        ctx.set_materialize_grads(False)
        return r["logp"], r["entropy"].clone()       # (the saved one stays as it is if the caller changes his)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logp, grad_entropy):
        _not_captured()                              # (the forward call may have been an eager one)
        scores, ids, stats, entropy = ctx.saved_tensors
        if grad_logp is None and grad_entropy is None:
            return None, None, None
        grad = ctx.engine.log_probs_backward(scores, ids, stats, entropy, grad_logp, grad_entropy, ctx.temperature)
        return grad, None, None


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, teacher_ids, teacher_scores, weights, temperature):
        eng = _engine(scores)
        r = eng.distill(scores, teacher_ids, teacher_scores, weights, temperature)
        ctx.engine, ctx.temperature = eng, temperature
        ctx.save_for_backward(scores, teacher_ids, teacher_scores, weights, r["stats"])
        return r["loss"]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        _not_captured()
        scores, teacher_ids, teacher_scores, weights, stats = ctx.saved_tensors
        grad = ctx.engine.distill_backward(scores, teacher_ids, teacher_scores, stats, grad_loss, weights,
                                           ctx.temperature)
        return grad, None, None, None, None


def log_probs(scores, ids, temperature=1.0):
    """(logp, entropy), float32 [n] each: of every row of softmax(scores / temperature) the log probability of class
    ids[row] (int64 [n]; 0, and without gradient, where the id is outside 0..k-1) and the entropy.  -logp is the
    cross-entropy of the labels."""
    if not torch.is_tensor(ids):
        raise TypeError("ids must be an int64 tensor [n]")
    _check_scores(scores)
    return _LogProbs.apply(scores, ids, float(temperature))


def distill_loss(scores, teacher_ids, teacher_scores, weights=None, temperature=1.0):
    """float32 [n]: weights * temperature^2 * KL(q || softmax(scores / temperature)) of every row, q being the
    distribution over the teacher's classes (Engine.distill; teacher_ids and teacher_scores as Engine.log_probs(...,
    top=...) of the teacher's scores gives them).  Differentiable with respect to the scores only."""
    _constant(teacher_scores, "teacher_scores")
    _constant(weights, "weights")
    _check_scores(scores)
    return _Distill.apply(scores, teacher_ids, teacher_scores, weights, float(temperature))
