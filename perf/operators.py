"""Timed cases of the operators on rows of class scores: log probabilities and distillation.

`log_probs`: of every row of scores, at a temperature, the log probability of a given class, the
entropy, and the classes with the highest scores; and the gradient of the first two.  `distill`: the
divergence of every row from the distribution over a teacher's top classes, and its gradient.

`run` computes them in plain torch operations in 32 bits while `own` is false and calls the library's
operators where it is true; `exact` computes the same outputs in 64 bits."""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORED = -100          # the id of a row without a label, and of an unused teacher entry


# ------------------------------------------------------------------------------------------ the cases
def _log_probs(name, rows, classes, dtype, top, temperature=1.0, entropy=True, grad=False, pad=0, masked=0.0,
               ignored=0.0):
    """`pad`: scores between the end of a row and the next; `masked`: share of classes whose score is -inf;
    `ignored`: share of rows without a label; `grad`: the gradient as well."""
    return {"name": name, "op": "log_probs", "rows": rows, "classes": classes, "dtype": dtype, "top": top,
            "temperature": temperature, "entropy": entropy, "grad": grad, "pad": pad, "masked": masked,
            "ignored": ignored}


def _distill(name, rows, classes, dtype, top, temperature=1.0, grad=True, pad=0, masked=0.0, ignored=0.0):
    """`top`: teacher entries of a row; `ignored`: share of rows of weight 0 (the end of a padded batch) and of unused
    teacher entries; the rest as above."""
    return {"name": name, "op": "distill", "rows": rows, "classes": classes, "dtype": dtype, "top": top,
            "temperature": temperature, "grad": grad, "pad": pad, "masked": masked, "ignored": ignored}


def listed():
    return [
        # the shot classifier's scores of the benchmark's 10 000-frame clip, with the runner-up class
        _log_probs("clip_frames", 10000, 3, "f32", 2),
        # one token of one sequence: a call whose latency is what counts
        _log_probs("one_token", 1, 32000, "bf16", 5),
        # one token each of a batch of sequences, with alternatives, below temperature 1
        _log_probs("token_batch", 64, 131072, "bf16", 20, temperature=0.7),
        # scoring of whole texts: every position's token and its alternatives; the largest forward call
        _log_probs("score_texts", 4096, 128000, "bf16", 20),
        # scores in 32 bits with an odd number of classes, part of them masked, rows cut out of a wider buffer
        _log_probs("masked_odd", 777, 50021, "f32", 8, pad=27, masked=0.3),
        # a policy-gradient step: log probabilities and an entropy bonus, forward and backward
        _log_probs("policy_step", 2048, 65536, "bf16", 0, grad=True),
        # the same on a ragged batch in fp16 with unlabelled rows
        _log_probs("policy_odd", 515, 32003, "f16", 0, temperature=1.3, grad=True, ignored=0.2),
        # a batch of frames of a student of the shot classifier against all three of its scores
        _distill("clip_student", 256, 3, "f32", 3, temperature=2.0),
        # evaluation of a student: the loss alone, 32 bits, many teacher entries
        _distill("student_eval", 1000, 50021, "f32", 100, grad=False),
        # a training step with a padded batch
        _distill("student_step", 2048, 32000, "bf16", 20, temperature=2.0, ignored=0.15),
        # few rows over a long class axis
        _distill("student_long", 8, 262144, "f32", 50),
        # the largest training step
        _distill("student_large", 4096, 131072, "bf16", 64),
    ]


MOST = 4096 * 128000          # scores of a drawn case at most


def _between(rng, low, high):
    """A whole number, its logarithm spread evenly over the range."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    classes = _between(rng, 2, 262144)
    rows = _between(rng, 1, min(200000, max(1, MOST // classes)))
    op = rng.choice(["log_probs", "distill"])
    grad = rng.random() < 0.5
    top = 0 if op == "log_probs" and grad else _between(rng, 1, min(64 if op == "log_probs" else 128, classes))
    case = {"rows": rows, "classes": classes, "dtype": rng.choice(sorted(DTYPES)), "top": top, "grad": grad,
            "temperature": rng.choice([1.0, 1.0, 0.5, 0.8, 2.0, 3.5]), "pad": rng.choice([0, 0, 1, 24, 77]),
            "masked": rng.choice([0.0, 0.0, 0.2, 0.6]), "ignored": rng.choice([0.0, 0.1, 0.4])}
    build = _log_probs if op == "log_probs" else _distill
    case = build(None, **case)
    if op == "log_probs":
        case["entropy"] = grad or rng.random() < 0.7
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------ inputs
def _distinct(n, k, count, gen):
    """`count` different classes for each row: a start of the row's own and a step without a common factor with k."""
    start = torch.randint(0, k, (n, 1), generator=gen, device="cuda")
    step = max(1, int(k * 0.38196601))
    while math.gcd(step, k) != 1:
        step += 1
    return (start + step * torch.arange(count, device="cuda")) % k


def _scores(case, gen):
    """Rows of scores as a trained classifier gives them: a spread of 2 around a level of the row, a few high ones."""
    n, k = case["rows"], case["classes"]
    dtype = DTYPES[case["dtype"]]
    buf = torch.empty((n, k + case["pad"]), dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // (k + case["pad"]))
    for a in range(0, n, step):
        part = torch.randn((min(step, n - a), k + case["pad"]), generator=gen, device="cuda")
        part.mul_(2.0).add_(3.0 * torch.randn((part.shape[0], 1), generator=gen, device="cuda"))
        buf[a:a + step] = part
    x = buf[:, :k]
    # the classes the row is about
    high = _distinct(n, k, min(4, k), gen)
    lift = 4.0 + 3.0 * torch.rand(high.shape, generator=gen, device="cuda")
    x.scatter_(1, high, (x.gather(1, high).float() + lift).to(dtype))
    if case["masked"]:
        for a in range(0, n, step):
            b = min(n, a + step)
            mask = torch.rand((b - a, k), generator=gen, device="cuda") < case["masked"]
            mask.scatter_(1, high[a:b], False)
            x[a:b].masked_fill_(mask, float("-inf"))
    return x, high


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, k, top = case["rows"], case["classes"], case["top"]
    x, high = _scores(case, gen)
    state = {"case": case, "scores": x}
    if case["op"] == "log_probs":
        # mostly one of the likely classes, now and then any of them
        ids = high[:, 0].clone()
        if not case["masked"]:
            rare = torch.rand((n,), generator=gen, device="cuda") < 0.25
            ids = torch.where(rare, torch.randint(0, k, (n,), generator=gen, device="cuda"), ids)
        if case["ignored"]:
            ids.masked_fill_(torch.rand((n,), generator=gen, device="cuda") < case["ignored"], IGNORED)
        state["ids"] = ids
        if case["grad"]:
            state["grad_logp"] = torch.randn((n,), generator=gen, device="cuda")
            state["grad_entropy"] = 0.1 * torch.rand((n,), generator=gen, device="cuda")
    else:
        ids = _distinct(n, k, top, gen)
        kind = torch.float32 if case["dtype"] == "f32" else DTYPES[case["dtype"]]
        teacher = 2.0 * torch.randn((n, top), generator=gen, device="cuda") + 6.0
        state["teacher_scores"] = teacher.sort(1, descending=True)[0].to(kind)
        weights = 0.5 + torch.rand((n,), generator=gen, device="cuda")
        if case["ignored"]:
            weights.masked_fill_(torch.rand((n,), generator=gen, device="cuda") < case["ignored"], 0.0)
            unused = torch.rand((n, top), generator=gen, device="cuda") < case["ignored"]
            unused[:, 0] = False
            ids = ids.masked_fill(unused, IGNORED)
        if case["masked"]:
            # a teacher names no class that is masked for the student
            safe = ids.clamp(min=0)
            old = x.gather(1, safe)
            x.scatter_(1, safe, torch.where(torch.isinf(old), torch.zeros_like(old), old))
        state["teacher_ids"], state["weights"] = ids, weights
    if own:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cut-detection_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from cutdet import api
        state["engine"] = api.default_engine(x.device)
    return state


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if case["op"] == "log_probs":
        return (_log_probs_own if own else _log_probs_plain)(state, case)
    return (_distill_own if own else _distill_plain)(state, case)


def _log_probs_own(state, case):
    eng, x, ids = state["engine"], state["scores"], state["ids"]
    got = eng.log_probs(x, ids, top=case["top"], temperature=case["temperature"], entropy=case["entropy"])
    out = {"logp": got["logp"]}
    if case["entropy"]:
        out["entropy"] = got["entropy"]
    if case["top"]:
        out["top_logp"], out["top_ids"] = got["top_logp"], got["top_ids"]
    if case["grad"]:
        out["grad"] = eng.log_probs_backward(x, ids, got["stats"], got["entropy"], state["grad_logp"],
                                             state["grad_entropy"], temperature=case["temperature"])
    return out


def _distill_own(state, case):
    got = state["engine"].distill(state["scores"], state["teacher_ids"], state["teacher_scores"], state["weights"],
                                  temperature=case["temperature"], grad=case["grad"])
    return {"loss": got["loss"], "grad": got["grad"]} if case["grad"] else {"loss": got["loss"]}


def _order_keys(x):
    """Whole numbers in the order of the scores, equal scores in the reverse order of their index, all different."""
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    return (bits << 32) | (x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device))


def _log_probs_plain(state, case):
    x, ids, t = state["scores"].float(), state["ids"], case["temperature"]
    n, k = x.shape
    z = x / t
    z = z - z.amax(1, keepdim=True)
    logp = z - z.exp().sum(1, keepdim=True).log()
    p = logp.exp()
    labelled = (ids >= 0) & (ids < k)
    safe = torch.where(labelled, ids, 0)
    out = {"logp": torch.where(labelled, logp.gather(1, safe[:, None])[:, 0], 0.0)}
    if case["entropy"]:
        weighted = torch.where(p > 0, p * logp, 0.0)
        out["entropy"] = -weighted.sum(1)
    if case["top"]:
        keys = _order_keys(x).topk(case["top"], dim=1)[0]
        out["top_ids"] = k - 1 - (keys & 0xFFFFFFFF)
        out["top_logp"] = logp.gather(1, out["top_ids"])
    if case["grad"]:
        g_l = torch.where(labelled, state["grad_logp"], 0.0)[:, None]
        g_h = state["grad_entropy"][:, None]
        grad = -p * g_l - g_h * torch.where(p > 0, p * (logp + out["entropy"][:, None]), 0.0)
        grad.scatter_add_(1, safe[:, None], g_l)
        out["grad"] = (grad / t).to(state["scores"].dtype)
    return out


def _distill_plain(state, case):
    x, t = state["scores"].float(), case["temperature"]
    ids, w = state["teacher_ids"], state["weights"]
    k = x.shape[1]
    z = x / t
    z = z - z.amax(1, keepdim=True)
    logp = z - z.exp().sum(1, keepdim=True).log()
    used = (ids >= 0) & (ids < k)
    safe = torch.where(used, ids, 0)
    s = torch.where(used, state["teacher_scores"].float() / t, float("-inf"))
    s = s - s.amax(1, keepdim=True)
    logq = s - s.exp().sum(1, keepdim=True).log()
    q = logq.exp()
    terms = torch.where(q > 0, q * (logq - logp.gather(1, safe)), 0.0)
    out = {"loss": torch.where(w != 0, w * t * t * terms.sum(1), 0.0)}
    if case["grad"]:
        grad = logp.exp().scatter_add_(1, safe, torch.where(used, -q, 0.0))
        out["grad"] = torch.where(w[:, None] != 0, grad * (w * t)[:, None], 0.0).to(state["scores"].dtype)
    return out


# ------------------------------------------------------------------------------------------ work and truth
def work(case):
    n, k, top = case["rows"], case["classes"], case["top"]
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    scores = n * k * size
    if case["op"] == "log_probs":
        bytes_ = scores + 8 * n + 4 * n + (4 * n if case["entropy"] else 0) + 12 * n * top
        flops = n * k * (6 if case["entropy"] else 4)
        if case["grad"]:
            bytes_ += scores + 8 * n
            flops += n * k * 6
    else:
        live = n * (1.0 - case["ignored"])           # rows of weight 0 need not be read
        bytes_ = live * k * size + n * (4 + 4) + n * top * (8 + size)
        flops = live * k * 4
        if case["grad"]:
            bytes_ += scores
            flops += live * k * 4
    return {"bytes": int(bytes_), "flops": int(flops)}


def exact(case, seed):
    state = prepare(case, seed)
    parts = []
    step = max(1, (1 << 25) // case["classes"])
    for a in range(0, case["rows"], step):
        rows = slice(a, a + step)
        part = {key: value[rows] for key, value in state.items() if torch.is_tensor(value)}
        parts.append((_exact_log_probs if case["op"] == "log_probs" else _exact_distill)(part, case))
    return {key: torch.cat([part[key] for part in parts]) for key in parts[0]}


def _exact_log_probs(part, case):
    z = part["scores"].double() / case["temperature"]
    n, k = z.shape
    lse = torch.logsumexp(z, 1)
    ids, line = part["ids"], torch.arange(n, device=z.device)
    has = ids.ge(0).logical_and(ids.lt(k))
    label = ids.clamp(0, k - 1)
    out = {"logp": (z[line, label] - lse) * has}
    p = torch.softmax(z, 1)
    mean = (p * z.clamp(min=-1e30)).sum(1)           # -inf only where p is 0
    entropy = lse - mean
    if case["entropy"]:
        out["entropy"] = entropy
    if case["top"]:
        values, order = torch.sort(z, dim=1, descending=True, stable=True)
        out["top_logp"] = values[:, :case["top"]] - lse[:, None]
        out["top_ids"] = order[:, :case["top"]].contiguous()
    if case["grad"]:
        g_l = (part["grad_logp"].double() * has)[:, None]
        g_h = part["grad_entropy"].double()[:, None]
        grad = -p * (g_l + g_h * (z.clamp(min=-1e30) - mean[:, None]))
        grad[line, label] += g_l[:, 0]
        out["grad"] = grad / case["temperature"]
    return out


def _exact_distill(part, case):
    t = case["temperature"]
    z = part["scores"].double() / t
    ids, w = part["teacher_ids"], part["weights"].double()
    unused = ids.lt(0).logical_or(ids.ge(z.shape[1]))
    at = ids.masked_fill(unused, 0)
    q = torch.softmax((part["teacher_scores"].double() / t).masked_fill(unused, float("-inf")), 1)
    log_ratio = torch.log(q.clamp(min=1e-300)) - (z.gather(1, at) - torch.logsumexp(z, 1, keepdim=True))
    loss = w * t * t * (q * log_ratio.masked_fill(q == 0, 0.0)).sum(1)
    out = {"loss": loss.masked_fill(w == 0, 0.0)}
    if case["grad"]:
        grad = torch.softmax(z, 1)
        grad.scatter_add_(1, at, -q)
        out["grad"] = (grad * (w * t)[:, None]).masked_fill((w == 0)[:, None], 0.0)
    return out
