"""Operators on rows of class scores on the GPU against the 64-bit reference (tests/rows_reference.py, where the
tolerances are derived)."""
import math

import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LOWEST = {name: torch.finfo(t).min for name, t in TYPES.items()}


@pytest.fixture(scope="module")
def eng():
    from cutdet import api
    return api.default_engine("cuda:0")


def rows(n, k, dtype, seed=0, pad=0, offset=0):
    """Scores [n, k], `pad` elements between rows, starting `offset` elements into an allocation."""
    g = torch.Generator().manual_seed(seed * 7919 + n * 31 + k)
    buf = (torch.randn(offset + n * (k + pad), generator=g) * 2.5).to(TYPES[dtype]).cuda()
    return buf[offset:].view(n, k + pad)[:, :k]


def labels(n, k, seed=0):
    g = torch.Generator().manual_seed(seed + 17)
    ids = torch.randint(0, k, (n,), generator=g)
    ids[::5] = torch.tensor([-100, k, -1, k - 1, 0] * (n // 5 // 5 + 1))[:len(ids[::5])]
    return ids.cuda()


def vector(n, seed, scale=1.0):
    return (torch.randn(n, generator=torch.Generator().manual_seed(seed)) * scale).cuda()


def check_log_probs(eng, x, ids, top, temperature=1.0, entropy=True):
    k = x.shape[1]
    got = eng.log_probs(x, ids, top=top, temperature=temperature, entropy=entropy)
    want = ref.log_probs64(x, ids, temperature, top)
    if ids is not None:
        ref.check_logp(got["logp"], want["logp"], k)
    if entropy:
        ref.check_entropy(got["entropy"], want["entropy"], k)
    assert ("entropy" in got) == entropy and ("logp" in got) == (ids is not None) and ("top_ids" in got) == (top > 0)
    if top:
        assert torch.equal(got["top_ids"], want["top_ids"])
        ref.check_logp(got["top_logp"], want["top_logp"], k, "top")
    return got


def check_backward(eng, x, ids, temperature=1.0, which="both", out=None):
    n, k = x.shape
    r = eng.log_probs(x, ids, temperature=temperature)
    gl = vector(n, 3) if which != "entropy" else None
    gh = vector(n, 4) if which != "logp" else None
    want, size = ref.log_probs_grad64(x, ids, gl, gh, temperature)
    got = eng.log_probs_backward(x, ids if gl is not None else None, r["stats"], r["entropy"] if gh is not None else None,
                                 gl, gh, temperature, out=out)
    ref.check_grad(got, want, size, k)
    return got


# sizes around every boundary: threads, vectors, pieces, variants by length
KS = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 255, 257, 511, 513, 1000, 1023, 1024, 1025, 2047, 2048,
      2049, 4097, 8191, 8192, 8193, 12345]
LONG = [32000, 32768, 32769, 50021, 65536, 65543, 131072, 131075, 200003, 262144]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("k", KS)
def test_log_probs_short_rows(eng, k, dtype):
    for i, (n, top, t) in enumerate(((1, 1, 1.0), (13, min(5, k), 0.7), (70, min(64, k), 1.9), (5, 0, 1.0))):
        check_log_probs(eng, rows(n, k, dtype, i, pad=i, offset=3 * i), labels(n, k, i), top, t)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("k", LONG)
def test_log_probs_long_rows(eng, k, dtype):
    for i, (n, top, t) in enumerate(((1, 20, 1.0), (3, 64, 0.7), (19, 7, 1.9))):
        check_log_probs(eng, rows(n, k, dtype, i, pad=i, offset=i), labels(n, k, i), top, t)


@pytest.mark.parametrize("k", [3, 40, 5000, 70001])
def test_outputs_that_are_not_asked_for(eng, k):
    x, ids = rows(11, k, "bf16"), labels(11, k)
    for ids_, top, entropy in ((None, 0, True), (None, 3, False), (ids, 0, False), (None, 0, False), (ids, 3, True)):
        got = check_log_probs(eng, x, ids_, top, entropy=entropy)
        want_m = x.float().amax(1)
        assert torch.equal(got["stats"][:, 0], want_m)
        s = (x.double() - want_m.double()[:, None]).exp().sum(1)
        assert ((got["stats"][:, 1].double() - s).abs() <= ref.row_error(k) * s).all()


@pytest.mark.parametrize("n", [1, 255, 256, 257, 10000, 70000])
def test_many_rows_of_three_classes(eng, n):
    x = rows(n, 3, "f32")
    check_log_probs(eng, x, labels(n, 3), 3)
    check_backward(eng, x, labels(n, 3))
    assert torch.equal(eng.log_probs(x, top=1)["top_ids"][:, 0], eng.max_argmax(x)[1])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("k", [2, 5, 16, 50, 700, 1024, 3000, 40000, 150001])
def test_masked_scores(eng, k, dtype):
    """-inf in places; the type's lowest value in places; rows of nothing else; NaN and +inf."""
    n = 24
    x = rows(n, k, dtype, 3)
    g = torch.Generator().manual_seed(1)
    x[0:4].masked_fill_((torch.rand(4, k, generator=g) < 0.5).cuda(), -math.inf)
    x[4:8].masked_fill_((torch.rand(4, k, generator=g) < 0.5).cuda(), LOWEST[dtype])
    x[8, :] = -math.inf                      # no distribution
    x[9, :] = LOWEST[dtype]                  # all equal
    x[10, :] = -math.inf
    x[10, k // 2] = 1.5                      # one class left
    x[11, :] = LOWEST[dtype]
    x[11, k - 1] = -3.0
    x[12, :] = torch.finfo(TYPES[dtype]).max
    x[13, 0] = torch.finfo(TYPES[dtype]).max
    x[14, k - 1] = math.inf
    x[15, k // 3] = math.nan
    x[16, :] = math.nan
    x[17, 0], x[17, k - 1] = -math.inf, math.nan
    x[18, :] = 0.25                          # all equal
    x[19, ::2], x[19, 1::2] = 0.0, -0.0      # the two zeros are equal
    x[20, :] = -math.inf
    x[20, ::max(1, k // 3)] = 2.0            # few classes left, equal
    x[21, :] = -math.inf
    x[21, 0], x[21, k - 1] = LOWEST[dtype], LOWEST[dtype]
    ids = labels(n, k)
    for t, top in ((1.0, min(k, 20)), (0.5, min(k, 64)), (3.0, 1)):
        check_log_probs(eng, x, ids, top, t)
        for which in ("both", "logp", "entropy"):
            check_backward(eng, x, ids, t, which)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("k", [60, 1000, 4000, 33000, 140000])
def test_top_of_rows_in_unusual_orders(eng, k, dtype):
    """Rising, falling, few different values, values that repeat with the period of the threads' shares: more scores than
    the usual few are as large as the largest of a share."""
    i = torch.arange(k)
    made = [i / k, -i / k, (i % 7) / 7.0, (i % 1024 < 5) * 1.0, (i % 512 == 3) * 2.0 + (i % 64 == 1), (i // 64) / k,
            -(i // 1000) * 1.0, (i == k - 1) * 1.0, (i % 300 == 7) * (1.0 + (i % 11) / 11), torch.zeros(k)]
    g = torch.Generator().manual_seed(2)
    made += [torch.randint(0, m, (k,), generator=g) / m for m in (2, 20, 500)]
    made += [torch.where(torch.rand(k, generator=g) < p, 1.0, torch.rand(k, generator=g) * 0.5) for p in (.001, .005, .02)]
    x = torch.stack([v.float() for v in made]).to(TYPES[dtype]).cuda()
    for top in (1, 5, 20, 64):
        if top <= k:
            check_log_probs(eng, x, None, top)
    check_log_probs(eng, x.repeat(9, 1), None, min(k, 64))


@pytest.mark.parametrize("k", [5, 600, 9000, 100000])
@pytest.mark.parametrize("level", [1e4, 7e5, 726817.5, 726830.0, 2e6, 1e30])
def test_scores_far_from_zero(eng, k, level):
    """Levels where a product with log2(e) / T loses what sets the scores apart (the border of two ways to compute it at
    2^20 ln 2 = 726817.5 among them)."""
    n = 12
    step = float(torch.tensor(level).nextafter(torch.tensor(math.inf)) - torch.tensor(level))
    g = torch.Generator().manual_seed(3)
    steps = torch.randint(0, 40, (n, k), generator=g)
    x = (level + step * max(1, round(0.5 / step)) * steps).float()
    x[::2] = -x[::2]
    x = x.cuda()
    t = max(1.0, min(2.0 ** 16, step))
    ids, (at, te) = labels(n, k), teacher(n, k, 7)
    for temperature in (t, 0.99 * t):
        check_log_probs(eng, x, ids, min(k, 9), temperature)
        check_backward(eng, x, ids, temperature)
        check_distill(eng, x, at, te, None, temperature)


def test_offsets_beyond_32_bits(eng):
    """5.2 GB of scores: the last rows lie beyond 2^31 elements and 2^32 bytes."""
    n, k = 40000, 65536
    x = torch.zeros((n, k), dtype=torch.bfloat16, device="cuda")
    last = rows(8, k, "bf16", 1)
    x[-8:] = last
    ids = torch.zeros(n, dtype=torch.int64, device="cuda")
    ids[-8:] = labels(8, k)
    got = eng.log_probs(x, ids, top=5)
    part = {key: v[-8:] for key, v in got.items()}
    want = ref.log_probs64(last, ids[-8:], 1.0, 5)
    ref.check_logp(part["logp"], want["logp"], k)
    assert torch.equal(part["top_ids"], want["top_ids"])
    assert torch.equal(got["top_ids"][0].cpu(), torch.arange(5))
    gl = vector(n, 1)
    at = torch.stack([torch.arange(4, device="cuda")] * n) * 1000
    te = torch.ones((n, 4), device="cuda")
    want_l, size, want_g, gsize = ref.distill64(last, at[-8:], te[-8:])
    want_p = ref.log_probs_grad64(last, ids[-8:], gl[-8:], None)
    grad = eng.log_probs_backward(x, ids, got["stats"], None, gl)
    ref.check_grad(grad[-8:], *want_p, k)
    del grad
    d = eng.distill(x, at, te, grad=True, out=x)             # in place
    assert d["grad"].data_ptr() == x.data_ptr()
    ref.check_loss(d["loss"][-8:], want_l, size, k)
    ref.check_grad(x[-8:], want_g, gsize, k)


@pytest.mark.parametrize("n,k", [((4 << 20) + 5, 3), ((4 << 20) + 5, 520), ((16 << 20) + 21, 17), ((1 << 20) + 3, 2050)])
def test_more_rows_than_a_grid_holds(eng, n, k):
    """The rows beyond one launch's workgroups are taken by a loop."""
    x = torch.zeros((n, k), dtype=torch.bfloat16, device="cuda")
    at = torch.randint(0, n, (40,), generator=torch.Generator().manual_seed(1)).cuda()
    at[-8:] = torch.arange(n - 8, n, device="cuda")
    x[at] = rows(40, k, "bf16")
    some = x[at]
    ids = torch.zeros(n, dtype=torch.int64, device="cuda")
    ids[at] = labels(40, k)[:40]
    got = eng.log_probs(x, ids, top=2)
    want = ref.log_probs64(some, ids[at], 1.0, 2)
    ref.check_logp(got["logp"][at], want["logp"], k)
    ref.check_entropy(got["entropy"][at], want["entropy"], k)
    assert torch.equal(got["top_ids"][at], want["top_ids"])
    g = torch.ones(n, device="cuda")
    grad = eng.log_probs_backward(x, ids, got["stats"], got["entropy"], g, g)
    ref.check_grad(grad[at], *ref.log_probs_grad64(some, ids[at], g[at], g[at]), k)
    te = eng.distill(x, got["top_ids"], got["top_logp"], grad=True, out=grad)
    loss, size, dg, ds = ref.distill64(some, got["top_ids"][at], got["top_logp"][at])
    ref.check_loss(te["loss"][at], loss, size, k)
    ref.check_grad(grad[at], dg, ds, k)


def test_one_very_long_row(eng):
    k = (1 << 28) + 5
    x = torch.empty((1, k), dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(3))
    x[0, k - 1], x[0, 0] = 9.0, 9.0
    ids = torch.tensor([k - 2], device="cuda")
    got = eng.log_probs(x, ids, top=64)
    lp, p = ref.log_softmax64(x)
    ref.check_logp(got["logp"], lp[:, k - 2], k)
    h = torch.tensor([float(-(p * lp).sum())], dtype=torch.float64, device="cuda")
    ref.check_entropy(got["entropy"], h, k)
    order = torch.sort(x[0], descending=True, stable=True)[1][:64]
    assert torch.equal(got["top_ids"][0], order)
    at = order[None, :5].contiguous()
    d = eng.distill(x, at, torch.ones((1, 5), device="cuda"), grad=True)
    loss = 0.2 * (math.log(0.2) - lp[0, at[0]]).sum()
    ref.check_loss(d["loss"], loss[None], loss.abs()[None] + 30, k)
    p[0, at[0]] -= 0.2
    ref.check_grad(d["grad"], p, p.abs() + 1e-12, k)


def test_the_longest_rows_that_are_allowed(eng):
    """2^30 classes, where twice the number overflows 32 bits: the last scores count."""
    k = 1 << 30
    x = torch.zeros((1, k), dtype=torch.float16, device="cuda")
    x[0, k - 3:] = 30.0
    ids = torch.tensor([k - 1], device="cuda")
    got = eng.log_probs(x, ids, top=4)
    assert got["top_ids"].tolist() == [[k - 3, k - 2, k - 1, 0]]
    s = 3 + k * math.exp(-30.0)
    assert abs(float(got["logp"]) + math.log(s)) <= ref.row_error(k)
    grad = eng.log_probs_backward(x, ids, got["stats"], None, torch.ones(1, device="cuda"))
    p = 1 / s
    assert abs(float(grad[0, k - 1]) - (1 - p)) < 1e-3 and abs(float(grad[0, k - 2]) + p) < 1e-3
    assert float(grad[0, :k - 3].abs().max()) < 1e-6
    d = eng.distill(x, ids[:, None], torch.ones((1, 1), device="cuda"), grad=True, out=grad)
    assert abs(float(d["loss"]) - math.log(s)) <= ref.row_error(k) + 1e-6
    assert abs(float(grad[0, k - 1]) - (p - 1)) < 1e-3 and abs(float(grad[0, k - 2]) - p) < 1e-3


# ---------------------------------------------------------------------------------------------- gradients
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("k", [1, 3, 8, 16, 17, 65, 300, 1023, 1025, 5001, 32003, 131075])
def test_log_probs_backward(eng, k, dtype):
    for i, (n, t) in enumerate(((1, 1.0), (9, 0.7), (33, 2.5))):
        x = rows(n, k, dtype, i, pad=i, offset=i)
        for which in ("both", "logp", "entropy"):
            check_backward(eng, x, labels(n, k, i), t, which)
        none = eng.log_probs_backward(x, None, eng.log_probs(x)["stats"], None, None, None)
        assert not none.any()
        # rows apart in the output; what lies between them stays
        wide = torch.full((n, k + 5), 7.0, dtype=x.dtype, device="cuda")
        check_backward(eng, x, labels(n, k, i), t, out=wide[:, 2:k + 2])
        assert (wide[:, :2] == 7).all() and (wide[:, k + 2:] == 7).all()
        same = x.clone() if i == 0 else x
        want = check_backward(eng, x, labels(n, k, i), t).clone()
        r = eng.log_probs(same, labels(n, k, i), temperature=t)
        got = eng.log_probs_backward(same, labels(n, k, i), r["stats"], r["entropy"], vector(n, 3), vector(n, 4), t, out=same)
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("k", [3, 40, 200, 700, 1500, 4000, 33000, 150001])
def test_no_gradient_for_the_end_of_a_padded_batch(eng, k, dtype):
    """Rows without a label, or with upstream gradients of 0, may hold anything."""
    n = 12
    x = rows(n, k, dtype)
    ids = labels(n, k, 2) % k
    gl, gh = vector(n, 3), vector(n, 4)
    ids[2:5], gh[2:6], gl[5] = -100, 0.0, 0.0
    x[2:6] = math.nan
    x[3, 0], x[4, :] = math.inf, -math.inf
    r = eng.log_probs(x, ids)
    got = eng.log_probs_backward(x, ids, r["stats"], r["entropy"], gl, gh)
    assert not got[2:6].any()
    ref.check_grad(got, *ref.log_probs_grad64(x, ids, gl, gh), k)
    got = eng.log_probs_backward(x, ids, r["stats"], None, gl)
    ref.check_grad(got, *ref.log_probs_grad64(x, ids, gl, None), k)
    assert not got[2:6].any() and got[0].any()


def teacher(n, k, entries, seed=0, dtype="f32"):
    g = torch.Generator().manual_seed(seed + 99)
    ids = torch.randint(0, k, (n, entries), generator=g)              # a class may come twice
    te = (torch.randn(n, entries, generator=g) * 2 + 3).to(TYPES[dtype])
    unused = torch.rand(n, entries, generator=g) < 0.2
    ids[unused] = torch.tensor([-100, k, -1, 1 << 40])[torch.randint(0, 4, (int(unused.sum()),), generator=g)]
    te[unused] = math.nan                                             # must not be looked at
    return ids.cuda(), te.cuda()


def check_distill(eng, x, ids, te, w=None, t=1.0):
    k = x.shape[1]
    loss, size, grad, gsize = ref.distill64(x, ids, te, w, t)
    alone = eng.distill(x, ids, te, w, t)
    assert "grad" not in alone
    both = eng.distill(x, ids, te, w, t, grad=True)
    # (not bit for bit: the two calls may add the same terms in another order; each has to be within the bound)
    ref.check_loss(alone["loss"], loss, size, k)
    ref.check_loss(both["loss"], loss, size, k)
    ref.check_grad(both["grad"], grad, gsize, k)
    g = vector(x.shape[0], 8)
    late = eng.distill_backward(x, ids, te, alone["stats"], g, w, t)
    gd = g.double()[:, None]
    ref.check_grad(late, torch.where(grad == 0, grad, grad * gd), gsize * gd.abs(), k)
    return both


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("k", [1, 2, 3, 8, 16, 17, 64, 65, 300, 1024, 1025, 2500, 8193, 32003, 65536, 131075])
def test_distill(eng, k, dtype):
    for i, (n, entries, t) in enumerate(((1, 1, 1.0), (7, 3, 2.0), (30, 64, 0.7), (18, 65, 1.0), (4, 256, 3.0))):
        x = rows(n, k, dtype, i, pad=i, offset=i)
        ids, te = teacher(n, k, entries, i, dtype if i % 2 else "f32")
        w = None
        if i % 2:
            w = vector(n, 5).abs() + 0.1
            w[::3] = 0.0
        check_distill(eng, x, ids, te, w, t)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("k", [3, 16, 40, 1000, 3000, 40000, 150001])
def test_distill_of_masked_rows(eng, k, dtype):
    n = 16
    x = rows(n, k, dtype, 5)
    ids, te = teacher(n, k, 6, 5)
    w = torch.ones(n, device="cuda")
    ids[0], te[0] = torch.arange(6).cuda() % k, 1.0
    x[0, 1:] = -math.inf                     # the teacher names classes that the student rules out: an infinite loss
    x[1, :] = -math.inf                      # no distribution
    x[2, :] = LOWEST[dtype]
    x[3, 0] = math.nan
    x[4, :], w[4] = math.nan, 0.0            # the end of a padded batch
    te[5], w[5] = math.nan, 0.0
    ids[6] = -1                              # no teacher
    x[6, 0] = math.nan
    ids[7], te[7] = k - 1, 2.0               # one class six times
    te[8, 0], ids[8, 0] = -math.inf, 0       # an entry without a share
    te[9], ids[9] = -math.inf, 0             # no entry with a share
    te[10, 2], ids[10, 2] = math.nan, 0
    te[11, 2], ids[11, 2] = math.inf, 0
    w[12], w[13] = -1.5, math.nan
    te[14] = 1e30                            # equal shares whatever the size
    x[15, 0] = math.inf
    check_distill(eng, x, ids, te, w)
    check_distill(eng, x, ids, te, w, 2.0)
    got = eng.distill(x, ids, te, w, grad=True)
    assert got["loss"][4] == 0 and got["loss"][5] == 0 and got["loss"][6] == 0
    assert not got["grad"][[4, 5, 6]].any()
    assert math.isnan(got["loss"][3]) and math.isnan(got["loss"][13])


@pytest.mark.parametrize("k", [3, 100, 5000, 80000])
def test_gradients_against_differences(eng, k):
    """Central differences along a direction, of the kernels' own forward in 32 bits."""
    n, h = 6, 2.0 ** -6
    x = rows(n, k, "f32", 2)
    v = rows(n, k, "f32", 9) / 2.5
    ids, (at, te) = labels(n, k, 1), teacher(n, k, 20, 1)
    gl, gh = vector(n, 3), vector(n, 4)

    def policy(z):
        r = eng.log_probs(z, ids)
        return gl.double() * r["logp"].double() + gh.double() * r["entropy"].double()

    r = eng.log_probs(x, ids)
    for f, grad in ((policy, eng.log_probs_backward(x, ids, r["stats"], r["entropy"], gl, gh)),
                    (lambda z: eng.distill(z, at, te)["loss"].double(), eng.distill(x, at, te, grad=True)["grad"])):
        d = (f(x + h * v) - f(x - h * v)) / (2 * h)
        want = (grad.double() * v.double()).sum(1)
        # the third derivative along v is a cumulant of third order of |v| <= 5 standard normals times a few logarithms:
        # below 100; both forward values are off by row_error of at most ln k + 30
        tol = h * h / 6 * 100 + 3 * ref.row_error(k) * (math.log(k) + 30) / h
        assert ((d - want).abs() <= tol).all(), ((d - want).abs().max(), tol)


# ---------------------------------------------------------------------------------------------- autograd
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("k", [3, 2000, 40000])
def test_losses_differentiate(eng, k, dtype):
    from cutdet import losses
    n = 10
    x = rows(n, k, dtype, 4).clone().requires_grad_()
    ids, (at, te) = labels(n, k), teacher(n, k, 9, 3)
    w = vector(n, 5).abs()
    a, b, c = vector(n, 6), vector(n, 7), vector(n, 8)
    logp, ent = losses.log_probs(x, ids, 1.5)
    loss = losses.distill_loss(x, at, te, w, 2.0)
    (logp * a + ent * b).sum().backward()
    first = x.grad.clone()
    want, size = ref.log_probs_grad64(x.detach(), ids, a, b, 1.5)
    ref.check_grad(first, want, size, k)
    x.grad = None
    (loss * c).sum().backward()
    _, _, dg, ds = ref.distill64(x.detach(), at, te, w, 2.0)
    ref.check_grad(x.grad, dg * c.double()[:, None], ds * c.double().abs()[:, None], k)
    # one output alone; the entropies changed in place after the call
    x.grad = None
    logp, ent = losses.log_probs(x, ids)
    ent.data.zero_()
    ent.sum().backward()
    want, size = ref.log_probs_grad64(x.detach(), None, None, torch.ones(n, device="cuda"))
    ref.check_grad(x.grad, want, size, k)
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(losses.log_probs(x, ids)[0].sum(), x, create_graph=True)
        g.sum().backward()


def test_a_row_used_for_every_label_sums_its_gradients(eng):
    from cutdet import losses
    k, n = 700, 12
    base = rows(1, k, "f32").clone().requires_grad_()
    ids = labels(n, k)
    losses.log_probs(base.expand(n, k), ids)[0].sum().backward()
    want, size = ref.log_probs_grad64(base.detach().expand(n, k), ids, torch.ones(n, device="cuda"), None)
    # n gradients added in 32 bits
    d = (base.grad.double()[0] - want.sum(0)).abs()
    assert (d <= (ref.row_error(k) + 200 * ref.U + n * ref.U) * size.sum(0) + 1e-37).all()


def test_scores_in_other_orders(eng):
    """Columns apart, transposed, reversed by index, one row for all: as if they were contiguous."""
    x = rows(40, 600, "bf16")
    ids = labels(40, 600)
    views = {"every other class": x[:, ::2], "transposed": x.t().contiguous().t(), "rows apart": x[::3],
             "one row": x[:1].expand(40, 600), "one class": x[:, :1], "from the middle": x[:, 3:500]}
    for name, v in views.items():
        n, k = v.shape
        a = eng.log_probs(v, ids[:n], top=min(4, k))
        b = eng.log_probs(v.contiguous(), ids[:n], top=min(4, k))
        for key in a:
            assert torch.equal(a[key], b[key]), (name, key)
        at, te = teacher(n, k, 5)
        a, b = eng.distill(v, at, te, grad=True), eng.distill(v.contiguous(), at, te, grad=True)
        for key in a:
            assert torch.equal(a[key], b[key]), (name, key)


def test_refusals_on_the_gpu(eng):
    from cutdet import _lib
    x = rows(4, 50, "f32")
    at, te = teacher(4, 50, 3)
    for t in (0.0, -1.0, math.nan, math.inf, 1e9):
        with pytest.raises(_lib.CutdetError):
            eng.log_probs(x, temperature=t)
    with pytest.raises(RuntimeError):
        eng.log_probs(x.cpu())
    with pytest.raises(RuntimeError):
        eng.log_probs(x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        eng.distill(x, at, te.cpu())
    buf = rows(8, 50, "f32")
    with pytest.raises(_lib.CutdetError):                       # the gradient would overwrite rows not yet read
        eng.distill(buf[:4], at, te, grad=True, out=buf[1:5])
    with pytest.raises(_lib.CutdetError):
        eng.distill(buf[:4], at, te, grad=True, out=buf.view(-1)[3:203].view(4, 50))
    with pytest.raises(_lib.CutdetError):                       # four rows of scores are one row of the gradient
        eng.distill(buf[0].expand(4, 50), at, te, grad=True, out=buf[:4])


def test_empty_batch(eng):
    x = torch.empty((0, 9), device="cuda")
    ids = torch.empty((0,), dtype=torch.int64, device="cuda")
    r = eng.log_probs(x, ids, top=2)
    assert r["logp"].shape == (0,) and r["top_ids"].shape == (0, 2) and r["stats"].shape == (0, 2)
    assert eng.log_probs_backward(x, ids, r["stats"], r["entropy"], r["logp"]).shape == (0, 9)
    d = eng.distill(x, ids.view(0, 1)[:, :1].expand(0, 3), torch.empty((0, 3), device="cuda"), grad=True)
    assert d["loss"].shape == (0,) and d["grad"].shape == (0, 9)


# ---------------------------------------------------------------------------------------------- streams and graphs
def test_streams_at_once(eng):
    """Two streams, one handle, calls that need a workspace among them: what each would give alone."""
    jobs = [(rows(2, 150001, "bf16", 1), 20), (rows(3, 200003, "f32", 2), 64), (rows(50, 1000, "f16", 3), 8)]
    want = [eng.log_probs(x, top=top) for x, top in jobs]
    at, te = teacher(2, 150001, 30)
    want_d = eng.distill(jobs[0][0], at, te, grad=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(10):
        for s, (x, top) in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append((eng.log_probs(x, top=top), eng.distill(jobs[0][0], at, te, grad=True)))
    torch.cuda.synchronize()
    for i, (g, d) in enumerate(got):
        for key, v in want[i % 3].items():
            assert torch.equal(g[key], v), (i, key)
        for key, v in want_d.items():
            assert torch.equal(d[key], v), (i, key)


@pytest.mark.parametrize("n,k", [(300, 3), (64, 900), (20, 30000), (2, 200003)])
def test_graphs(eng, n, k):
    """Two captured graphs replayed in turns, with eager work between: every replay equals the eager result."""
    x, ids = rows(n, k, "bf16").clone(), labels(n, k)
    at, te = teacher(n, k, 12)
    gl, gh = vector(n, 3), vector(n, 4)

    def step():
        r = eng.log_probs(x, ids, top=min(3, k))
        g = eng.log_probs_backward(x, ids, r["stats"], r["entropy"], gl, gh)
        d = eng.distill(x, at, te, grad=True)
        return dict(r, g=g, loss=d["loss"], d=d["grad"], late=eng.distill_backward(x, at, te, d["stats"], gl))

    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for i in range(6):
        x.copy_(rows(n, k, "bf16", 20 + i))
        want = {key: v.clone() for key, v in step().items()}
        graphs[i % 2].replay()
        junk = torch.full((1 << 20,), float("nan"), device="cuda")          # may take the eager call's workspace
        graphs[(i + 1) % 2].replay()
        torch.cuda.synchronize()
        del junk
        for o in outs:
            for key, v in want.items():
                assert torch.equal(o[key], v), (i, key)


def test_captured_gradients_of_a_leaf_are_refused(eng):
    from cutdet import losses
    x, ids = rows(4, 20, "f32").clone().requires_grad_(), labels(4, 20)
    with pytest.raises(RuntimeError, match="leaf"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            losses.log_probs(x, ids)
    at, te = teacher(4, 20, 3)
    with pytest.raises(RuntimeError, match="captured"):                # not a leaf itself, but made of one
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            losses.distill_loss(x * 2, at, te)
    with torch.no_grad():                                              # nothing to differentiate: may be captured
        want = losses.distill_loss(x, at, te)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = losses.distill_loss(x, at, te)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert torch.isfinite(losses.log_probs(x, ids)[1]).all()


# ---------------------------------------------------------------------------------------------- used together
@pytest.mark.parametrize("k", [3, 5000])
def test_a_teachers_alternatives_train_a_student(eng, k):
    """The teacher's alternatives as log_probs gives them are distill's targets: following the gradient brings the
    student's own alternatives to the teacher's."""
    from cutdet import losses
    n, top = 16, min(k, 20)
    t = eng.log_probs(rows(n, k, "f32", 1) * 2, top=top, entropy=False)
    x = rows(n, k, "f32", 2).clone().requires_grad_()
    before = losses.distill_loss(x, t["top_ids"], t["top_logp"]).detach()
    both = eng.distill(x.detach(), t["top_ids"], t["top_logp"], grad=True)
    losses.distill_loss(x, t["top_ids"], t["top_logp"]).sum().backward()
    want = ref.distill64(x.detach(), t["top_ids"], t["top_logp"])
    for loss, grad in ((before, x.grad), (both["loss"], both["grad"])):
        ref.check_loss(loss, want[0], want[1], k)
        ref.check_grad(grad, want[2], want[3], k)
    after = eng.distill(x.detach() - 0.1 * x.grad, t["top_ids"], t["top_logp"])["loss"]
    assert (after < before).all()            # a descent step of a convex function with curvature below 1


# ---------------------------------------------------------------------------------------------- the classifier's own paths
def _clip(eng, n=37):
    cl = ([0] * 9 + [2] * 4 + [1] * 11 + [0] * 13)[:n]
    frames = eng.synth_frames(torch.tensor(cl, dtype=torch.uint8, device=eng.device), 180, 320, 5)
    return frames, torch.tensor(cl, device=eng.device)


def test_evaluate_per_frame_and_against_a_teacher(eng):
    from frameID.net import load_default_net
    frames, labels_ = _clip(eng)
    labels_[3] = -1
    nets = {d: load_default_net(d)[0].to("cuda:0") for d in ("f32", "bf16")}
    batches = [(frames[:16], labels_[:16]), (frames[16:], labels_[16:])]
    plain = nets["bf16"].evaluate(batches)
    assert set(plain) == {"correct", "total", "accuracy", "loss", "frames"}
    got = nets["bf16"].evaluate(batches, per_frame=True, teacher=nets["f32"])
    assert all(got[k] == plain[k] for k in plain if k != "loss") and abs(got["loss"] - plain["loss"]) < 1e-9
    logits = {d: net.classify_frames(frames)[0] for d, net in nets.items()}
    per = got["per_frame"]
    want = ref.log_probs64(logits["bf16"], labels_, 1.0, 2)
    ref.check_logp(per["logp"], want["logp"].cpu(), 3)
    ref.check_entropy(per["entropy"], want["entropy"].cpu(), 3)
    assert torch.equal(per["top_ids"], want["top_ids"].cpu())
    # the mean cross-entropy that eval_accumulate sums is the mean of -logp over the labelled frames
    assert abs(float(-per["logp"].double().sum()) / got["frames"] - got["loss"]) < 3 * ref.row_error(3) + 1e-6 * got["loss"]
    lp = ref.log_softmax64(logits["f32"])[0]
    loss, size, _, _ = ref.distill64(logits["bf16"], torch.arange(3, device="cuda").expand(37, 3), lp)
    # the teacher's log probabilities are the kernel's: each off by row_error, q by as much
    d = (per["divergence"].double() - loss.cpu()).abs()
    assert (d <= 3 * (ref.row_error(3) + 256 * ref.U) * size.cpu()).all()
    assert abs(got["divergence"] - float(per["divergence"].double().mean())) < 1e-12
    same = nets["f32"].evaluate(batches, teacher=nets["f32"])
    assert abs(same["divergence"]) <= 3 * (ref.row_error(3) + 256 * ref.U) * float(size.max())


def test_soft_targets_train_a_student_of_the_classifier(eng):
    """prod_net's answers as targets of a linear student on small frames: gradients through autograd as from the formula."""
    from cutdet import losses
    from frameID.net import load_default_net
    net = load_default_net()[0].to("cuda:0")
    frames, _ = _clip(eng)
    ids, logp = net.soft_targets(frames)
    assert ids.shape == logp.shape == (37, 3) and torch.equal(ids[:, 0], net.classify_frames(frames)[2])
    feats = frames[:, ::20, ::20].float().reshape(37, -1) / 255
    g = torch.Generator().manual_seed(1)
    weight = (torch.randn(3, feats.shape[1], generator=g) * 0.05).cuda().requires_grad_()
    scores = feats @ weight.t()
    losses.distill_loss(scores, ids, logp, temperature=2.0).mean().backward()
    _, _, grad, size = ref.distill64(scores.detach(), ids, logp, None, 2.0)
    want = (grad.t() / 37) @ feats.double()
    # 37 products added in 32 bits, each with the scores' gradient off by check_grad's bound
    bound = ((ref.row_error(3) + 144 * ref.U + 80 * ref.U) * size.t() / 37) @ feats.double()
    assert ((weight.grad.double() - want).abs() <= bound + 1e-30).all()
