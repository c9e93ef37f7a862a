"""The sums over a row, where almost all of its terms are equal: roundings then go one way and add up, so that what a
thread adds one after the other shows.

A thread takes its scores in pieces of PIECE (16 in 32 bits, 32 in 16 bits), adds a piece's terms among themselves and
the piece to its sum: at most ceil(k / (threads PIECE)) + PIECE + 3 roundings of u = 2^-24 each, the single scores at a row's
ends included.  The merges, the powers of two and the logarithm add what rows_reference.row_error counts for them."""
import math

import pytest
import torch

import rows_reference as ref
from test_gpu_rows import TYPES, eng       # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def sum_error(k, threads, dtype):
    piece = 16 if dtype == "f32" else 32
    terms = -(-k // (threads * piece)) + piece + 3
    return ref.U * (terms + 128 + 4 * math.log(k + 1) + 2 + 2 * (math.log2(k) + 1))


# rows, classes, type, threads that share a row: a group of lanes, a wave, workgroups of every size
SIZES = [(20, 250, "f32", 16), (20, 1000, "bf16", 64), (700, 2500, "f32", 128), (700, 8000, "bf16", 128),
         (100, 8000, "f16", 256), (700, 30000, "bf16", 256), (300, 30000, "f16", 512), (800, 262144, "f32", 256),
         (800, 262144, "bf16", 256), (300, 200003, "f32", 512), (65, 1 << 24, "bf16", 1024), (66, 1 << 22, "f32", 1024)]


@pytest.mark.parametrize("n,k,dtype,threads", SIZES)
@pytest.mark.parametrize("below", [0.1, 0.808, 1.3, 5.0])
def test_a_few_high_classes_before_many_equal_ones(eng, n, k, dtype, threads, below):
    """Every thread has one of the high classes first, so that the equal ones add terms that are no power of two."""
    x = torch.full((n, k), -below, dtype=TYPES[dtype], device="cuda")
    low = float(x[0, 0])
    high = min(k // 4, threads * 8 + 64)
    x[:, :high] = 0.0
    e = math.exp(low)
    s = high + (k - high) * e
    error = sum_error(k, threads, dtype)
    ids = torch.full((n,), k - 1, device="cuda")
    ids[::2] = 0
    want = torch.full((n,), low - math.log(s), dtype=torch.float64, device="cuda")
    want[::2] = -math.log(s)

    def close(got, want, bound):
        d = (got.double() - want).abs().max()
        assert d <= bound, f"off by {float(d):.3g}, {float(d) / bound:.3g} of the bound"

    tol = error + 5 * ref.U * (abs(low) + math.log(s))
    entropy = math.log(s) - (k - high) * e * low / s
    for asked in (True, False):
        got = eng.log_probs(x, ids, entropy=asked)
        close(got["logp"], want, tol)
        if asked:
            close(got["entropy"], entropy, 2 * error * (1 + math.log(k + 1)) + 2 * ref.U * entropy)
    one = torch.ones((n, 1), device="cuda")
    close(eng.distill(x, ids[:, None], one)["loss"], -want, tol)
    close(eng.distill(x, ids[:, None], one, grad=True, out=x)["loss"], -want, tol)


@pytest.mark.parametrize("k", [5, 600, 9000, 100000])
@pytest.mark.parametrize("level", [-7e5, -3e4, 0.0, 12.0, 1e5, 7e5, 2e6])
def test_maximum_and_sum_give_the_logarithm_of_the_sum(eng, k, level):
    """stats: max z + ln S is ln sum exp z to the rounding of max z log2(e) to 32 bits, which S is relative to."""
    n, t = 6, 0.8
    g = torch.Generator().manual_seed(3)
    x = (level + torch.randn((n, k), generator=g) * 2).float().cuda()
    want = torch.logsumexp(x.double() / t, 1)
    for stats in (eng.log_probs(x, temperature=t)["stats"],
                  eng.distill(x, torch.zeros((n, 1), dtype=torch.int64, device="cuda"), torch.zeros((n, 1), device="cuda"),
                              temperature=t)["stats"]):
        assert torch.equal(stats[:, 0], x.amax(1))
        z = stats[:, 0].double() / t
        d = (z + stats[:, 1].double().log() - want).abs()
        # besides: c = log2(e) / T of the scores' distances from the maximum, at most 16, is off by 2 u
        assert (d <= ref.U * (1 + 1e-5) * z.abs() + ref.row_error(k) + 32 * ref.U).all(), d.max()
