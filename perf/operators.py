"""What is measured of the operators on a row of logits: the log probabilities of given tokens with entropy and top
alternatives, and the distillation loss against a teacher's top logits, each with its gradient.

``own`` False: the operators in elementary torch operations (fp32, rounded once at the end); True: the calls that a user
makes of the package."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one masked position answered with its five best tokens: latency
        {"name": "fill-mask one", "op": "logprobs", "rows": 1, "vocab": 30522, "pad": 0, "dtype": "f32", "tokens": 1,
         "top": 5, "entropy": True, "scale": 1.0, "masked": False},
        # a decoding step of a batch: long vocabulary, twenty alternatives, temperature
        {"name": "decode step", "op": "logprobs", "rows": 48, "vocab": 131072, "pad": 0, "dtype": "bf16", "tokens": 1,
         "top": 20, "entropy": True, "scale": 1.25, "masked": True},
        # every position of one document scored (the whole-model workload's length and vocabulary)
        {"name": "score document", "op": "logprobs", "rows": 4096, "vocab": 30522, "pad": 0, "dtype": "f32", "tokens": 1,
         "top": 5, "entropy": True, "scale": 1.0, "masked": False},
        # log likelihoods alone over a corpus batch; odd vocabulary, rows that start at any element
        {"name": "corpus odd bf16", "op": "logprobs", "rows": 8192, "vocab": 50257, "pad": 0, "dtype": "bf16", "tokens": 1,
         "top": 0, "entropy": False, "scale": 1.0, "masked": False},
        # cloze questions with 64 candidate answers each, padded rows
        {"name": "cloze choices", "op": "logprobs", "rows": 512, "vocab": 30522, "pad": 6, "dtype": "f32", "tokens": 64,
         "top": 0, "entropy": False, "scale": 1.0, "masked": False},
        # the byte-level model of the C++ driver: short rows, very many
        {"name": "byte model", "op": "logprobs", "rows": 32768, "vocab": 256, "pad": 0, "dtype": "f32", "tokens": 1,
         "top": 4, "entropy": True, "scale": 1.0, "masked": False},
        # training on log probabilities with an entropy term: forward and backward
        {"name": "train bf16", "op": "logprobs_train", "rows": 4096, "vocab": 30522, "pad": 0, "dtype": "bf16", "tokens": 1,
         "top": 0, "entropy": True, "scale": 1.0, "masked": False},
        # the same in fp32 with an odd vocabulary and two tokens a row (a preferred and a rejected one)
        {"name": "train odd f32", "op": "logprobs_train", "rows": 1500, "vocab": 50257, "pad": 0, "dtype": "f32",
         "tokens": 2, "top": 0, "entropy": False, "scale": 0.8, "masked": False},
        # the masked positions of one short text distilled: few rows
        {"name": "distill few rows", "op": "distill", "rows": 20, "vocab": 30522, "pad": 0, "dtype": "f32", "slots": 8,
         "scale": 0.5, "masked": False},
        # a training step's loss and gradient in one call
        {"name": "distill step bf16", "op": "distill", "rows": 8192, "vocab": 30522, "pad": 0, "dtype": "bf16", "slots": 32,
         "scale": 0.5, "masked": False},
        # loss first, gradient once the weights of the rows are known; odd vocabulary
        {"name": "distill apart f32", "op": "distill_apart", "rows": 2048, "vocab": 50257, "pad": 0, "dtype": "f32",
         "slots": 100, "scale": 1.0, "masked": False},
        # the largest: long vocabulary, rows that do not fit a work-group's registers
        {"name": "distill long vocab", "op": "distill", "rows": 4096, "vocab": 131072, "pad": 0, "dtype": "bf16",
         "slots": 64, "scale": 0.25, "masked": True},
    ]


MOST = 4096 * 131072   # logits of the largest listed case


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "logprobs_train", "distill", "distill", "distill_apart"])
    dtype = rng.choice(["f32", "bf16"])
    vocab = _spread(rng, 200, 160000)
    # (half of the largest listed case's logits: that one is 16-bit with one read and one write of each)
    rows = max(1, min(_spread(rng, 1, 32768), MOST // (4 * vocab)))
    case = {"op": op, "rows": rows, "vocab": vocab, "pad": rng.choice([0, 0, rng.randrange(1, 64)]), "dtype": dtype,
            "scale": rng.choice([1.0, round(rng.uniform(0.2, 2.0), 3)]), "masked": rng.random() < 0.3}
    if op.startswith("logprobs"):
        case["tokens"] = rng.choice([1, 1, rng.randrange(2, 100)])
        case["entropy"] = rng.random() < 0.5
        case["top"] = rng.choice([0, rng.randrange(1, 65)]) if op == "logprobs" else 0
    else:
        case["slots"] = _spread(rng, 1, 256) if vocab > 256 else rng.randrange(1, 65)
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    stride = vocab + case["pad"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def whole(high, *shape):
        return torch.randint(0, high, shape, generator=g, device="cuda", dtype=torch.int32)

    # a language model's logits: a wide bulk, and a few tokens of each row that stand out
    logits = torch.empty((rows, stride), device="cuda", dtype=dtype)[:, :vocab]
    logits.copy_(normal(rows, vocab).mul_(2.2))
    if case["masked"]:   # a mask over the vocabulary, as constrained answers have: those logits are -inf
        logits.masked_fill_((whole(8, vocab) == 0)[None], -math.inf)
        logits[:, 0] = 0.0
    # (the workspace: cut rows meet in it; a program keeps one per stream)
    state = {"case": dict(case), "logits": logits, "workspace": torch.zeros(1 << 20, device="cuda", dtype=torch.uint8)}
    if case["op"].startswith("logprobs"):
        n = case["tokens"]
        tokens = whole(vocab, rows, n)
        # seven in ten rows know their token
        known = (whole(10, rows) < 7)[:, None]
        at = tokens[:, :1].long()
        logits.scatter_(1, at, torch.where(known, torch.full_like(at, 9, dtype=dtype), logits.gather(1, at)))
        state["tokens"] = tokens[:, 0].contiguous() if n == 1 else tokens
        if case["op"] == "logprobs_train":
            state["d_logprob"] = normal(*state["tokens"].shape) / rows
            state["d_entropy"] = normal(rows) * (0.1 / rows) if case["entropy"] else None
    else:
        k = case["slots"]
        rank = torch.arange(k, device="cuda")
        step = vocab // 7 if vocab > 1000 else 1
        while math.gcd(step, vocab) > 1:   # the slots of a row name different tokens
            step += 1
        ids = (whole(vocab, rows, 1).long() + rank * step) % vocab
        teacher = 9.0 - 1.5 * torch.log1p(rank.float()) + 0.5 * normal(rows, k)
        # the student has learnt some of it
        logits.scatter_(1, ids, (0.7 * teacher + normal(rows, k)).to(dtype))
        # one row in eight has a shorter list, one in sixteen is padding: no slot, weight zero
        short = (whole(8, rows) == 0)[:, None] & (rank >= (k + 1) // 2)[None]
        padding = whole(16, rows) == 0
        state["teacher_ids"] = ids.int().masked_fill(short | padding[:, None], -1)
        state["teacher_logits"] = teacher
        state["d_loss"] = torch.full((rows,), 1.0 / rows, device="cuda").masked_fill(padding, 0.0)
    return state


# ---------------------------------------------------------------------------------------------- plain form
def _log_softmax(logits, scale):
    x = logits.float() * scale
    t = x - x.amax(1, keepdim=True)
    return t - t.exp().sum(1, keepdim=True).log()


def _slots(ids, vocab):
    valid = (ids >= 0) & (ids < vocab)
    return valid, torch.where(valid, ids, 0).long()


def _top(logits, logp, k):
    """Descending logits, ties to the lowest index: one order over (value, index) in a whole number."""
    bits = (logits.float() + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32)
    order += (1 << 32) - 1 - torch.arange(logits.shape[1], device=logits.device)
    ids = (1 << 32) - 1 - (torch.topk(order, k, dim=1).values & 0xFFFFFFFF)
    return ids.int(), logp.gather(1, ids)


def _plain_logprobs(s, train):
    case, logits = s["case"], s["logits"]
    tokens = s["tokens"].reshape(case["rows"], -1)
    logp = _log_softmax(logits, case["scale"])
    valid, at = _slots(tokens, case["vocab"])
    out = {"logprob": torch.where(valid, logp.gather(1, at), 0.0).reshape(s["tokens"].shape)}
    if case["entropy"] or train:
        p = logp.exp()
    if case["entropy"]:
        out["entropy"] = -torch.where(p > 0, p * logp, 0.0).sum(1)
    if case["top"]:
        out["top_ids"], out["top_logprobs"] = _top(logits, logp, case["top"])
    if train:
        g = torch.where(valid, s["d_logprob"].reshape(tokens.shape), 0.0)
        d = -p * g.sum(1, keepdim=True)
        if case["entropy"]:
            d -= torch.where(p > 0, p * (logp + out["entropy"][:, None]), 0.0) * s["d_entropy"][:, None]
        d.scatter_add_(1, at, g)
        out["d_logits"] = (d * case["scale"]).to(logits.dtype)
    return out


def _plain_distill(s):
    case, logits = s["case"], s["logits"]
    logp = _log_softmax(logits, case["scale"])
    valid, at = _slots(s["teacher_ids"], case["vocab"])
    z = torch.where(valid, s["teacher_logits"] * case["scale"], -1e30)
    t = z - z.amax(1, keepdim=True)
    e = torch.where(valid, t.exp(), 0.0)
    total = e.sum(1, keepdim=True)
    some = total > 0
    total = torch.where(some, total, 1.0)
    q = e / total
    row = torch.where(q > 0, q * (t - total.log() - logp.gather(1, at)), 0.0).sum(1)
    d = torch.where(some, logp.exp(), 0.0)
    d.scatter_add_(1, at, -q)
    d *= (s["d_loss"] / case["scale"])[:, None]
    return {"row_loss": row / case["scale"] ** 2, "d_logits": d.to(logits.dtype)}


# ---------------------------------------------------------------------------------------------- the package
def _package():
    import importlib
    return importlib.import_module("sf-bert_amd")


def _own_logprobs(s, train):
    sfb, case = _package(), s["case"]
    got = sfb.token_logprobs(s["logits"], s["tokens"], top_k=case["top"], scale=case["scale"], entropy=case["entropy"],
                             workspace=s["workspace"])
    out = {"logprob": got["logprob"]}
    if case["entropy"]:
        out["entropy"] = got["entropy"]
    if case["top"]:
        out["top_ids"], out["top_logprobs"] = got["top_ids"], got["top_logprobs"]
    if train:
        out["d_logits"] = sfb.token_logprobs_backward(s["logits"], s["tokens"], got["stats"], d_logprob=s["d_logprob"],
                                                      entropy=got["entropy"] if case["entropy"] else None,
                                                      d_entropy=s["d_entropy"], scale=case["scale"])
    return out


def _own_distill(s):
    sfb, case = _package(), s["case"]
    if case["op"] == "distill":
        got = sfb.distillation_loss(s["logits"], s["teacher_ids"], s["teacher_logits"], scale=case["scale"],
                                    d_loss=s["d_loss"], workspace=s["workspace"])
        return {"row_loss": got["row_loss"], "d_logits": got["d_logits"]}
    got = sfb.distillation_loss(s["logits"], s["teacher_ids"], s["teacher_logits"], scale=case["scale"],
                                workspace=s["workspace"])
    d = sfb.distillation_loss_backward(s["logits"], s["teacher_ids"], s["teacher_logits"], got["stats"], s["d_loss"],
                                       scale=case["scale"])
    return {"row_loss": got["row_loss"], "d_logits": d}


def run(state):
    op = state["case"]["op"]
    if op.startswith("logprobs"):
        train = op == "logprobs_train"
        return _own_logprobs(state, train) if own else _plain_logprobs(state, train)
    return _own_distill(state) if own else _plain_distill(state)


def work(case):
    rows, vocab, size = case["rows"], case["vocab"], 2 if case["dtype"] == "bf16" else 4
    row = vocab * size
    if case["op"].startswith("logprobs"):
        small = 8 * case["tokens"] + 4 * case["entropy"] + 8 * case["top"]
        if case["op"] == "logprobs":   # multiply, subtract, exp, add; the entropy's product and sum
            return {"bytes": rows * (row + small), "flops": rows * vocab * (6 if case["entropy"] else 4)}
        # forward and backward are two calls with the caller's work between them: the logits are read in both
        return {"bytes": rows * (3 * row + 2 * small), "flops": rows * vocab * (14 if case["entropy"] else 9)}
    small = 8 * case["slots"] + 8
    if case["op"] == "distill":
        return {"bytes": rows * (2 * row + small), "flops": rows * vocab * 7}
    return {"bytes": rows * (3 * row + 2 * small), "flops": rows * vocab * 9}


# ---------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    x = s["logits"].double() * case["scale"]
    vocab = case["vocab"]
    lse = torch.logsumexp(x, 1, keepdim=True)
    p = torch.exp(x - lse)
    if case["op"].startswith("logprobs"):
        tokens = s["tokens"].reshape(case["rows"], -1).long()
        inside = (tokens >= 0) & (tokens < vocab)
        picked = torch.gather(x, 1, tokens.clamp(0, vocab - 1)) - lse
        out = {"logprob": torch.where(inside, picked, torch.zeros_like(picked)).reshape(s["tokens"].shape)}
        if case["entropy"]:
            # H = lse - sum p x, with p x = 0 where p = 0
            entropy = lse - torch.nan_to_num(p * x, nan=0.0).sum(1, keepdim=True)
            out["entropy"] = entropy[:, 0]
        if case["top"]:
            out["top_ids"] = None
            out["top_logprobs"] = torch.topk(x, case["top"], dim=1).values - lse
        if case["op"] == "logprobs_train":
            g = s["d_logprob"].double().reshape(tokens.shape) * inside
            grad = torch.zeros_like(x).scatter_add_(1, tokens.clamp(0, vocab - 1), g) - p * g.sum(1, keepdim=True)
            if case["entropy"]:
                grad -= s["d_entropy"].double()[:, None] * torch.nan_to_num(p * (x - lse + entropy), nan=0.0)
            out["d_logits"] = grad * case["scale"]
        return out
    ids = s["teacher_ids"].long()
    inside = (ids >= 0) & (ids < vocab)
    z = s["teacher_logits"].double() * case["scale"]
    z = torch.where(inside, z, torch.full_like(z, -math.inf))
    any_slot = inside.any(1, keepdim=True)
    q = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)
    logq = z - torch.logsumexp(z, 1, keepdim=True)
    logp = torch.gather(x, 1, ids.clamp(0, vocab - 1)) - lse
    row = torch.where(inside & any_slot, q * (logq - logp), torch.zeros_like(q)).sum(1)
    grad = p * any_slot
    grad = grad.scatter_add_(1, ids.clamp(0, vocab - 1), -q) * s["d_loss"].double()[:, None]
    return {"row_loss": row / case["scale"] ** 2, "d_logits": grad / case["scale"]}
