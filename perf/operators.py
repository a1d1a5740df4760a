"""Cases of the class / vocabulary operators: drawing a class from scores, distillation from a teacher's
top logits, and the embedding lookup with its gradient.

``run`` computes a case in plain torch operations, or, where ``own`` is set, through ``ser_amd``.
"""

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding stream, the usual truncation: latency is all there is
        {"name": "sample_one", "op": "sample", "rows": 1, "classes": 50001, "dtype": "bf16",
         "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "mixed": False},
        # a serving batch whose requests each bring their own settings, some of them greedy
        {"name": "sample_mixed_batch", "op": "sample", "rows": 64, "classes": 65536, "dtype": "f16",
         "temperature": 0.7, "top_k": 40, "top_p": 0.9, "min_p": 0.02, "mixed": True},
        # a large batch over a large vocabulary, nucleus and min-p without top-k
        {"name": "sample_nucleus_large", "op": "sample", "rows": 512, "classes": 131072, "dtype": "bf16",
         "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.01, "mixed": False},
        # rollouts for training: the untruncated distribution, 32-bit scores, an odd vocabulary
        {"name": "sample_full_f32", "op": "sample", "rows": 256, "classes": 100003, "dtype": "f32",
         "temperature": 0.6, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mixed": False},
        # the fast profile's eight classes, one row per clip of a prepared corpus, taught by the accurate profile
        {"name": "distill_emotions", "op": "distill_step", "rows": 46080, "classes": 8, "teacher": 3, "dtype": "f32",
         "temperature": 2.0},
        # a short ragged batch of transcript tokens, loss and gradient through autograd
        {"name": "distill_short_autograd", "op": "distill_autograd", "rows": 37, "classes": 50001, "teacher": 20,
         "dtype": "bf16", "temperature": 1.0},
        # a training step's worth of tokens, loss and gradient in one call
        {"name": "distill_step_large", "op": "distill_step", "rows": 4096, "classes": 50001, "teacher": 64,
         "dtype": "bf16", "temperature": 2.0},
        # 32-bit logits of a large vocabulary through autograd
        {"name": "distill_autograd_f32", "op": "distill_autograd", "rows": 1024, "classes": 131072, "teacher": 128,
         "dtype": "f32", "temperature": 1.5},
        # one token of each of a few decoding streams
        {"name": "embed_decode", "op": "embed", "tokens": 8, "classes": 50001, "width": 1280, "dtype": "f16"},
        # a packed batch of prompts
        {"name": "embed_prompts", "op": "embed", "tokens": 65536, "classes": 131072, "width": 1024, "dtype": "bf16"},
        # the table's gradient for a small training batch; the width is the feature vector's, which is odd
        {"name": "embed_gradient_odd", "op": "embed_gradient", "tokens": 3001, "classes": 5003, "width": 187,
         "dtype": "f32"},
        # the table's gradient for a large training batch
        {"name": "embed_gradient_large", "op": "embed_gradient", "tokens": 32768, "classes": 50001, "width": 1024,
         "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo..hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "distill_step", "distill_autograd", "embed", "embed_gradient"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "sample":
        classes = _spread(rng, 16, 131072)
        rows = _spread(rng, 1, max(1, min(2048, (512 * 131072 // 2) // classes)))
        return {"op": op, "rows": rows, "classes": classes, "dtype": dtype,
                "temperature": round(rng.uniform(0.3, 1.5), 3),
                "top_k": rng.choice([0, 1, _spread(rng, 1, 1000), _spread(rng, 1, 100)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.1, 0.99), 3)]),
                "min_p": rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]), "mixed": rng.random() < 0.4}
    if op in ("distill_step", "distill_autograd"):
        classes = _spread(rng, 2, 131072)
        rows = _spread(rng, 1, max(1, min(65536, (4096 * 50001 // 2) // classes)))
        return {"op": op, "rows": rows, "classes": classes, "teacher": min(classes, _spread(rng, 1, 256)),
                "dtype": dtype, "temperature": rng.choice([1.0, 2.0, round(rng.uniform(0.5, 4.0), 3)])}
    width = _spread(rng, 16, 4096)
    classes = _spread(rng, 8, max(8, min(131072, (1 << 26) // width)))
    tokens = _spread(rng, 1, max(1, min(65536, (1 << 26) // width)))
    return {"op": op, "tokens": tokens, "classes": classes, "width": width, "dtype": dtype}


# --------------------------------------------------------------------------------------------- inputs
def _scores(gen, rows, classes, dtype):
    """Scores as a trained head gives them: most classes far below a handful of likely ones."""
    x = torch.randn((rows, classes), generator=gen, device="cuda") * 2.0
    lift = torch.randint(0, classes, (rows, min(24, classes)), generator=gen, device="cuda")
    x.scatter_add_(1, lift, torch.rand(lift.shape, generator=gen, device="cuda") * 9.0)
    return x.to(_DTYPES[dtype])


def _tokens(gen, count, classes):
    """Token ids whose frequencies fall off as in text, the frequent ones spread over the table; every 37th
    place is padding (-1)."""
    r = torch.rand((count,), generator=gen, device="cuda", dtype=torch.float64)
    rank = (torch.exp(r * math.log(classes + 1.0)) - 1.0).long().clamp_(0, classes - 1)
    step = 7919 if classes % 7919 else 7907
    tok = (rank * step + 11) % classes
    tok[36::37] = -1
    return tok


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    if op == "sample":
        n = case["rows"]
        s = {"op": op, "logits": _scores(gen, n, case["classes"], case["dtype"]),
             "uniform": torch.rand((n,), generator=gen, device="cuda")}
        for key in ("temperature", "top_k", "top_p", "min_p"):
            s[key] = case[key]
        if case["mixed"]:
            at = torch.arange(n, device="cuda")
            s["temperature"] = torch.where(at % 4 == 3, 0.0, case["temperature"] * (0.5 + (at % 5) * 0.25)).float()
            s["top_k"] = torch.where(at % 3 == 1, 0, case["top_k"] + at % 7).to(torch.int32)
            s["top_p"] = torch.where(at % 5 == 2, 1.0, torch.full((n,), case["top_p"], device="cuda")).float()
            s["min_p"] = torch.where(at % 2 == 1, 0.0, torch.full((n,), case["min_p"], device="cuda")).float()
        return s
    if op in ("distill_step", "distill_autograd"):
        n, v, k = case["rows"], case["classes"], case["teacher"]
        logits = _scores(gen, n, v, case["dtype"])
        near = 0.6 * logits.float() + 1.5 * torch.randn((n, v), generator=gen, device="cuda")
        top, index = torch.topk(near, k, dim=1)
        weight = torch.rand((n,), generator=gen, device="cuda") / n
        weight[12::13] = 0.0   # padded places of the batch
        if op == "distill_autograd":
            logits.requires_grad_(True)
        return {"op": op, "logits": logits, "index": index, "top": top.to(logits.dtype), "weight": weight,
                "temperature": case["temperature"]}
    d, v, n = case["width"], case["classes"], case["tokens"]
    s = {"op": op, "tokens": _tokens(gen, n, v), "scale": math.sqrt(d), "classes": v}
    if op == "embed":
        s["table"] = (torch.randn((v, d), generator=gen, device="cuda") * 0.02).to(_DTYPES[case["dtype"]])
    else:
        s["grad"] = (torch.randn((n, d), generator=gen, device="cuda") * 0.01).to(_DTYPES[case["dtype"]])
    return s


# ----------------------------------------------------------------------------------------- plain forms
def _column(value, like, rows):
    """A setting as one 32-bit value per row (a column), whether one number or one for each row was given."""
    if not isinstance(value, torch.Tensor):
        value = torch.full((rows,), value, device=like.device, dtype=torch.float32)
    return value.double().unsqueeze(1)


def _plain_sample(s):
    # 64 bits: the draw is a comparison of a cumulative sum with a number, and every class is next to a border
    n, v = s["logits"].shape
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), -math.inf, x)
    best = x.max(dim=1, keepdim=True)
    alive = x > -math.inf
    far = torch.where(x == best.values, 0.0, x.double() - best.values.double())
    temperature = _column(s["temperature"], x, n)
    greedy = ~((temperature > 0) & (temperature < math.inf))
    weight = torch.where(alive, torch.exp(far / torch.where(greedy, 1.0, temperature)), 0.0)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    w = weight.gather(1, order)
    rank = torch.arange(v, device=x.device).unsqueeze(0)
    top_k, top_p, min_p = _column(s["top_k"], x, n), _column(s["top_p"], x, n), _column(s["min_p"], x, n)
    w = torch.where((top_k >= 1) & (rank >= top_k), 0.0, w)
    before = torch.cumsum(w, 1) - w
    keep = (w > 0) & ((rank == 0) | (before < top_p * w.sum(1, keepdim=True)) | ~(top_p < 1))
    keep &= (w >= min_p.clamp(max=1.0)) | ~(min_p > 0)
    keep &= (rank == 0) | ~greedy
    kept = torch.zeros_like(weight).scatter_(1, order, torch.where(keep, w, 0.0))
    upto = torch.cumsum(kept, 1)
    passed = upto > s["uniform"].double().unsqueeze(1) * upto[:, -1:]
    token = torch.where(passed.any(1), passed.int().argmax(1), v - 1 - kept.flip(1).gt(0).int().argmax(1))
    total = torch.where(alive, torch.exp(far), 0.0).sum(1)
    logprob = far.gather(1, token.unsqueeze(1)).squeeze(1) - torch.log(total)
    dead = ~alive.any(1)
    return torch.where(dead, -1, token), torch.where(dead, -math.inf, logprob).float()


def _plain_distill(s):
    x, index, t = s["logits"].detach().float(), s["index"], s["temperature"]
    z = x / t
    peak = z.max(dim=1, keepdim=True).values
    lse = peak + torch.log(torch.exp(z - peak).sum(1, keepdim=True))
    top = s["top"].float() / t
    top = top - top.max(dim=1, keepdim=True).values
    logp = top - torch.log(torch.exp(top).sum(1, keepdim=True))
    p = torch.exp(logp)
    loss = t * t * (p * (logp - z.gather(1, index) + lse)).sum(1)
    grad = torch.exp(z - lse).scatter_add_(1, index, -p) * (t * s["weight"].unsqueeze(1))
    return loss, grad.to(s["logits"].dtype)


def _plain_embed(s):
    tok, table = s["tokens"], s["table"]
    inside = ((tok >= 0) & (tok < table.shape[0])).unsqueeze(1)
    rows = table[tok.clamp(0, table.shape[0] - 1)].float() * s["scale"]
    return torch.where(inside, rows, 0.0).to(table.dtype)


def _plain_embed_gradient(s):
    tok, grad = s["tokens"], s["grad"]
    inside = ((tok >= 0) & (tok < s["classes"])).unsqueeze(1)
    total = torch.zeros((s["classes"], grad.shape[1]), device=grad.device)
    total.index_add_(0, tok.clamp(0, s["classes"] - 1), torch.where(inside, grad.float(), 0.0))
    return (total * s["scale"]).to(grad.dtype)


def run(state):
    op = state["op"]
    if own:
        import ser_amd

        if op == "sample":
            return ser_amd.sample_tokens(state["logits"], state["uniform"], temperature=state["temperature"],
                                         top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
        if op == "distill_step":
            return ser_amd.distillation_step(state["logits"], state["index"], state["top"],
                                             temperature=state["temperature"], row_weight=state["weight"])
        if op == "distill_autograd":
            loss = ser_amd.distillation_loss(state["logits"], state["index"], state["top"],
                                             temperature=state["temperature"])
            (grad,) = torch.autograd.grad(loss, state["logits"], grad_outputs=state["weight"])
            return loss.detach(), grad
        if op == "embed":
            return ser_amd.embed_tokens(state["tokens"], state["table"], scale=state["scale"])
        return ser_amd.embedding_gradient(state["grad"], state["tokens"], state["classes"], scale=state["scale"])
    if op == "sample":
        return _plain_sample(state)
    if op in ("distill_step", "distill_autograd"):
        return _plain_distill(state)
    return _plain_embed(state) if op == "embed" else _plain_embed_gradient(state)


# ------------------------------------------------------------------------------------------ accounting
def work(case):
    op, size = case["op"], _SIZE[case["dtype"]]
    if op == "sample":
        n, v = case["rows"], case["classes"]
        # one exponential and one sum for the log-probability, one of each for the draw
        return {"bytes": n * (v * size + 4 + 12 + (16 if case["mixed"] else 0)), "flops": 6 * n * v}
    if op in ("distill_step", "distill_autograd"):
        n, v, k = case["rows"], case["classes"], case["teacher"]
        # each logit read once and each gradient written once, also where autograd calls twice
        return {"bytes": n * (2 * v * size + k * (8 + size) + 8), "flops": n * (8 * v + 10 * k)}
    d, v, n = case["width"], case["classes"], case["tokens"]
    if op == "embed":
        return {"bytes": n * (2 * d * size + 8), "flops": n * d}
    return {"bytes": n * (d * size + 8) + v * d * size, "flops": (n + v) * d}


# ------------------------------------------------------------------------------------- 64-bit answers
def _exact_sample(s):
    import numpy as np

    logits = s["logits"].double().cpu().numpy()
    n, v = logits.shape

    def per_row(value):
        return value.cpu().numpy() if isinstance(value, torch.Tensor) else np.full(n, value, np.float32)

    t, k, p, m = (per_row(s[key]).astype(np.float64) for key in ("temperature", "top_k", "top_p", "min_p"))
    u = s["uniform"].double().cpu().numpy()
    token, logprob = np.zeros(n, np.int64), np.zeros(n, np.float64)
    for r in range(n):
        x = logits[r]
        top = x.max()
        if t[r] > 0:
            w = np.exp((x - top) / t[r])
            by = np.argsort(-x, kind="stable")
            if k[r] >= 1:
                by = by[: int(k[r])]
            ranked = w[by]
            if p[r] < 1:
                reached = np.concatenate([[0.0], np.cumsum(ranked)[:-1]])
                by = by[: max(1, int(np.count_nonzero(reached < p[r] * ranked.sum())))]
            if m[r] > 0:
                by = by[w[by] >= m[r]]
            by = np.sort(by)
            share = np.cumsum(w[by])
            token[r] = by[min(len(by) - 1, int(np.searchsorted(share, u[r] * share[-1], side="right")))]
        else:
            token[r] = int(np.argmax(x))
        logprob[r] = x[token[r]] - top - math.log(np.exp(x - top).sum())
    return torch.from_numpy(token), torch.from_numpy(logprob)


def _exact_distill(s):
    t = float(s["temperature"])
    student = torch.log_softmax(s["logits"].detach().double() / t, dim=1)
    teacher = torch.log_softmax(s["top"].double() / t, dim=1)
    loss = t * t * (teacher.exp() * (teacher - student.gather(1, s["index"]))).sum(1)
    target = torch.zeros_like(student).scatter_add_(1, s["index"], teacher.exp())
    return loss, (student.exp_() - target) * (t * s["weight"].double().unsqueeze(1))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        return _exact_sample(s) if case["rows"] * case["classes"] <= 1 << 26 else None
    if op in ("distill_step", "distill_autograd"):
        return _exact_distill(s)
    tok = s["tokens"]
    if op == "embed":
        rows = torch.zeros((tok.numel(), case["width"]), dtype=torch.float64, device=tok.device)
        real = tok >= 0
        rows[real] = s["table"].double()[tok[real]] * s["scale"]
        return rows
    real = tok >= 0
    total = torch.zeros((case["classes"], case["width"]), dtype=torch.float64, device=tok.device)
    total.index_put_((tok[real],), s["grad"].double()[real] * s["scale"], accumulate=True)
    return total
