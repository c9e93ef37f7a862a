"""The operators on rows of class scores in 64 bits, and how far 32-bit results may be from them.

u = 2^-24 bounds the relative error of one 32-bit rounding.  With t_i = (x_i - max) log2(e) / T:

* t_i: one rounding of log2(e) / T (in 32 bits: 2 u), one of the fma: 3 u |t_i|; the power of two is off by 1 ulp (2 u):
  p_i before normalising is off by the factor 1 + (3 |t_i| ln 2 + 2) u =: 1 + b_i u.
* S = sum of them, added in chains of at most CHAIN terms (a thread's share) and then in a tree of at most 2 * 16
  additions and rescalings (2 roundings and a power each, 6 u): relative error (CHAIN + 128) u plus the mean of b_i.
  sum_i p_i b_i <= 3 (entropy-like sum_i p_i |t_i| ln 2) + 2 <= 3 ln k + 2 (the mean of -(z_i - max) is at most ln S).
* ln S: the hardware's log2 is off by 1 ulp (2 u) of at most log2 k + 1.

`row_error` is the sum of these for one row: what log p is off by besides 5 u |log p| for its own t and rounding."""
import math

import torch

U = 2.0 ** -24


def chain(k):
    """Terms that one thread adds one after the other, at most: the shortest rows are spread over 64 threads at least 16
    wide, long ones over 256 threads or more in pieces of 32."""
    return max(64, -(-k // 256) + 64)


def row_error(k):
    return U * (chain(k) + 128 + 4 * math.log(k + 1) + 2 + 2 * (math.log2(k) + 1))


def log_softmax64(x, temperature=1.0):
    """(log p, p) in 64 bits; a row of nothing but -inf has no distribution: log p -inf, p 0."""
    z = x.double() / temperature
    m = z.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    s = (z - m).exp().sum(1, keepdim=True)
    lp = torch.where(s == 0, torch.full_like(z, -math.inf), z - m - s.log())
    return lp, lp.exp()


def entropy64(lp, p):
    return -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(1)


def top64(x, top):
    """Indices of the largest scores, NaN first, equal ones (the two zeros as well) in the order of their index."""
    key = x.double() + 0.0
    key = torch.where(torch.isnan(key), torch.full_like(key, math.inf), key)
    # NaN before +inf: a second, stable sort by "is NaN"
    order = torch.sort(key, dim=1, descending=True, stable=True)[1]
    nan = torch.isnan(x).gather(1, order)
    again = torch.sort(nan.to(torch.int8), dim=1, descending=True, stable=True)[1]
    return order.gather(1, again)[:, :top]


def log_probs64(x, ids=None, temperature=1.0, top=0):
    lp, p = log_softmax64(x, temperature)
    k = x.shape[1]
    out = {"entropy": entropy64(lp, p)}
    if ids is not None:
        on = (ids >= 0) & (ids < k)
        out["logp"] = torch.where(on, lp.gather(1, torch.where(on, ids, 0)[:, None])[:, 0], 0.0)
    if top:
        out["top_ids"] = top64(x, top)
        out["top_logp"] = lp.gather(1, out["top_ids"])
    return out


def log_probs_grad64(x, ids, g_logp, g_entropy, temperature=1.0):
    """(gradient, size of the terms it is the sum of)."""
    lp, p = log_softmax64(x, temperature)
    n, k = x.shape
    grad = torch.zeros_like(p)
    size = torch.zeros_like(p)
    if g_logp is not None:
        on = (ids >= 0) & (ids < k)
        g = torch.where(on, g_logp.double(), 0.0)[:, None]
        hit = torch.zeros_like(p).scatter_(1, torch.where(on, ids, 0)[:, None], on.double()[:, None])
        alive = (p.sum(1, keepdim=True) > 0).double()
        grad += g * (hit * alive - p)
        size += g.abs() * (hit + p)
    if g_entropy is not None:
        g = g_entropy.double()[:, None]
        h = entropy64(lp, p)[:, None]
        grad -= g * torch.where(p == 0, torch.zeros_like(p), p * (lp + h))
        size += g.abs() * torch.where(p == 0, torch.zeros_like(p), p * (lp.abs() + h + math.log(k + 1)))
    # a row that no gradient reaches has none, NaN among its scores or not
    zero = torch.zeros(n, dtype=torch.float64, device=x.device)
    gl = zero if g_logp is None else torch.where((ids >= 0) & (ids < k), g_logp.double(), 0.0)
    gh = zero if g_entropy is None else g_entropy.double()
    off = ((gl == 0) & (gh == 0))[:, None]
    return torch.where(off, 0.0, grad / temperature), torch.where(off, 0.0, size / temperature)


def teacher64(ids, scores, k, temperature):
    used = (ids >= 0) & (ids < k)
    s = torch.where(used, scores.double() / temperature, -math.inf)
    m = s.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = (s - m).exp()
    total = e.sum(1, keepdim=True)
    q = torch.where(total == 0, torch.zeros_like(e), e / total)
    lq = torch.where(q == 0, torch.zeros_like(e), s - m - total.log())
    return q, lq, torch.where(used, ids, 0), used


def distill64(x, ids, scores, weights=None, temperature=1.0):
    """loss, gradient of its sum, and the sizes of the terms that either is the sum of."""
    n, k = x.shape
    lp, p = log_softmax64(x, temperature)
    q, lq, at, used = teacher64(ids, scores, k, temperature)
    w = torch.ones((n,), dtype=torch.float64, device=x.device) if weights is None else weights.double()
    lpj = lp.gather(1, at)
    terms = torch.where(q == 0, torch.zeros_like(q), q * (lq - lpj))
    sizes = torch.where(q == 0, torch.zeros_like(q), q * (lq.abs() + lpj.abs() + 4))
    off = (w == 0) | (q.sum(1) == 0)
    t2 = temperature * temperature
    loss = torch.where(off, torch.zeros_like(w), w * t2 * terms.sum(1))
    size = torch.where(off, torch.zeros_like(w), w.abs() * t2 * sizes.sum(1))
    dead = off | (p.sum(1) == 0)
    qk = torch.zeros_like(p).scatter_add_(1, at, torch.where(used, q, torch.zeros_like(q)))
    grad = torch.where(dead[:, None], torch.zeros_like(p), (p - qk) * (w * temperature)[:, None])
    gsize = torch.where(dead[:, None], torch.zeros_like(p), (p + qk) * (w.abs() * temperature)[:, None])
    return loss, size, grad, gsize


# ---- tolerances -------------------------------------------------------------------------------------------------
def _in_32_bits(want):
    """Values beyond the largest float32 are infinite in the results' type."""
    return torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * math.inf, want)


def check_logp(got, want, k, name="logp"):
    want = _in_32_bits(want)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want.cpu())), f"{name}: NaN in other places"
    assert torch.equal(got[~fin & ~torch.isnan(want)].double(), want[~fin & ~torch.isnan(want)]), f"{name}: infinities"
    d = (got.double() - want)[fin].abs()
    tol = row_error(k) + 5 * U * want[fin].abs()
    assert (d <= tol).all(), f"{name}: off by {float(d.max()):.3g}, {float((d / tol).max()):.3g} of the bound"


def check_entropy(got, want, k):
    # H = ln S - U / S ln 2: both parts at most ln k, U with the relative error of S and 1 rounding a term more
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want.cpu()))
    d = (got.double() - want).abs()
    tol = 2 * row_error(k) * (1 + math.log(k + 1)) + 2 * U * want.abs()
    ok = (d <= tol) | torch.isnan(want)
    assert ok.all(), f"entropy: off by {float(d.max()):.3g}, {float((d / tol).max()):.3g} of the bound"


def check_grad(got, want, size, k):
    """`size`: of the terms that the gradient is the sum of; each is off by row_error and its own t's rounding (t of a
    probability that is not negligible is above -60: 3 * 60 ln 2 + 16 roundings), the sum rounded once to the type, to
    half a step of its subnormals at least; what is below 2^-126 in 32 bits may be 0."""
    info = torch.finfo(got.dtype)
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want.cpu()))
    d = (got.double() - want).abs()
    tol = (row_error(k) + 144 * U) * size + info.eps / 2 * want.abs() + max(info.tiny * info.eps / 2, 2.0 ** -126)
    ok = (d <= tol) | torch.isnan(want)
    assert ok.all(), f"gradient: off by {float(d.max()):.3g}, {float((d / tol).max()):.3g} of the bound"


def check_loss(got, want, size, k):
    """Every term q (ln q - ln p): both logarithms off as check_logp allows, q by 64 roundings and its t's, up to 256
    terms added in a tree."""
    want = _in_32_bits(want)
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want.cpu()))
    inf = torch.isinf(want)
    assert torch.equal(got[inf].double(), want[inf])
    d = (got.double() - want)[~inf].abs()
    tol = (row_error(k) + 256 * U) * size[~inf]
    ok = (d <= tol) | torch.isnan(want[~inf])
    assert ok.all(), f"loss: off by {float(d.max()):.3g}, {float((d / tol).max()):.3g} of the bound"
