"""cutdet.losses around a graph capture, as far as no GPU is needed."""
import pytest
import torch

from test_rows_out_host import IDS, K, N, TEACHER, host_engine       # noqa: F401  (the fixture)


@pytest.mark.parametrize("which", ["log_probs", "distill_loss"])
def test_a_backward_pass_is_refused_under_capture_also_where_its_forward_was_not(host_engine, monkeypatch, which):
    from cutdet import losses
    monkeypatch.setattr(losses, "_engine", lambda scores: host_engine)
    x = torch.zeros(N, K, requires_grad=True)
    call = {"log_probs": lambda: losses.log_probs(x, IDS[:, 0])[0],
            "distill_loss": lambda: losses.distill_loss(x, IDS, TEACHER)}[which]
    early = call()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        early.sum().backward()
    assert x.grad is None


def test_a_backward_pass_outside_a_capture_runs(host_engine, monkeypatch):
    from cutdet import losses
    monkeypatch.setattr(losses, "_engine", lambda scores: host_engine)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    x = torch.zeros(N, K, requires_grad=True)
    (losses.log_probs(x, IDS[:, 0])[0].sum() + losses.distill_loss(x, IDS, TEACHER).sum()).backward()
    assert x.grad.shape == (N, K)
