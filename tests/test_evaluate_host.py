"""ProdNet.evaluate without a batch (no GPU)."""
import math
import types

import torch

from frameID.net import ProdNet, Validation


def test_no_batches_give_empty_rows():
    """The keys that were asked for are there whatever the number of batches."""
    net = types.SimpleNamespace(engine=types.SimpleNamespace(device=torch.device("cpu")))
    plain = ProdNet.evaluate(net, [])
    assert set(plain) == {"correct", "total", "accuracy", "loss", "frames"} and plain["frames"] == 0
    got = ProdNet.evaluate(net, [], per_frame=True, teacher=net)
    assert set(got) == set(plain) | {"per_frame", "divergence"} and math.isnan(got["divergence"])
    per = got["per_frame"]
    assert {k: (v.dtype, tuple(v.shape)) for k, v in per.items()} == {
        "logp": (torch.float32, (0,)), "entropy": (torch.float32, (0,)), "top_logp": (torch.float32, (0, 2)),
        "top_ids": (torch.int64, (0, 2)), "divergence": (torch.float32, (0,))}
    assert set(Validation(net, per_frame=True).result()["per_frame"]) == set(per) - {"divergence"}
    assert set(Validation(net, teacher=net).result()["per_frame"]) == {"divergence"}
