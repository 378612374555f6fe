"""Cases of the operators on rows of logits (token log probabilities, distillation from a teacher's top logits, their
gradients) against plain implementations in 64 bits.  `S` is the binding (capi of the device library or of its host
build), `dev(array, bf16)` puts a numpy array where that library reads it.

Tolerances, with u = 2^-24 (half a step of fp32, relative).  The factor c = scale log2(e) and the products (x - m) c are
off by at most 4 u relative, so an exponent t is off by 4 u |t|; 2^t adds 2 u; a thread's sum of n terms adds n u (every
rounding in the same direction) and joining the threads 16 u.  With T the largest |t| of the row's finite logits (the
reference lags the maximum by at most 8), a log probability is off by at most u (n + 5 (T + 8) + 48).  The entropy is
that times its own two terms' size (l and the mean of |t|); a probability has the same error relative, gradients follow."""
import numpy as np

U = 2.0 ** -24
ERR = {"null": 1, "shape": 4, "dtype": 5, "align": 6, "arg": 8, "workspace": 9}
LOWEST = {False: np.finfo(np.float32).min, True: np.float32(-3.3895314e38)}   # lowest fp32, lowest bf16


def round_bf16(x):
    import oracle_lib as orc
    return orc.round_bf16(np.ascontiguousarray(x, np.float32))


KINDS = ["normal", "peaked", "ties", "masked", "lowest", "all lowest", "rising", "empty", "huge", "constant", "nan", "inf",
         "zeros", "late peak"]
MASKS_AND_TIES = ["spread ties", "late ties", "open half", "open half, lowest", "ten left", "ten and masked", "masked"]


def logits_of(kind, vocab, rng, bf16):
    x = rng.standard_normal(vocab).astype(np.float32) * 2.5
    if kind == "peaked":
        x[rng.integers(vocab)] += 40.0
    elif kind == "ties":
        x = rng.integers(-2, 3, vocab).astype(np.float32)
    elif kind == "masked":        # a mask that leaves a few tokens
        keep = rng.random(vocab) < 5.0 / vocab
        keep[rng.integers(vocab)] = True
        x[~keep] = -np.inf
    elif kind == "lowest":        # a mask made of the type's lowest value
        x[rng.random(vocab) < 0.7] = LOWEST[bf16]
    elif kind == "all lowest":
        x[:] = LOWEST[bf16]
    elif kind == "rising":        # every vector raises the maximum; the largest stand side by side
        x = np.linspace(-60.0, 60.0, vocab).astype(np.float32)
    elif kind == "empty":
        x[:] = -np.inf
    elif kind == "huge":          # far from zero: differences of a few units of large logits
        x = (np.round(x) + 3000.0).astype(np.float32)
    elif kind == "constant":
        x[:] = 1.5
    elif kind == "nan":
        x[rng.integers(vocab)] = np.nan
        x[0] = np.inf
    elif kind == "inf":
        x[rng.integers(vocab)] = np.inf
    elif kind == "zeros":         # +0 and -0 are equal
        x = np.where(rng.random(vocab) < 0.5, np.float32(0.0), np.float32(-0.0))
    elif kind == "late peak":
        x[-1] = 30.0
    elif kind == "spread ties":   # the largest but for two is one value all over the row
        x *= 0.1
        x[5::37] = 7.0
        x[rng.integers(0, vocab, 2)] = 9.0
    elif kind == "late ties":     # and at its end
        x *= 0.1
        x[vocab // 8 * 7:] = 7.0
    elif kind == "open half":     # nothing but masked logits in the first half
        x[:vocab // 2] = -np.inf
    elif kind == "open half, lowest":
        x[:vocab // 2] = LOWEST[True]
    elif kind == "ten left":
        keep = rng.integers(0, vocab, 10)
        x, kept = np.full(vocab, LOWEST[True], np.float32), x[keep]
        x[keep] = kept
    elif kind == "ten and masked":   # masked logits of two kinds
        keep = rng.integers(0, vocab, 10)
        x, kept = np.full(vocab, LOWEST[True], np.float32), x[keep]
        x[::3] = -np.inf
        x[keep] = kept
    elif kind.startswith("behind "):   # a mask of any value
        keep = rng.integers(0, vocab, 10)
        x, kept = np.full(vocab, float(kind[7:]), np.float32), x[keep]
        x[keep] = kept
    elif kind.startswith("all of "):   # a row whose logits are all masked
        x[:] = float(kind[7:])
    elif kind == "falling":
        x = np.linspace(60.0, -60.0, vocab).astype(np.float32)
    elif kind == "first ones large":   # a vocabulary in the order of its tokens' frequencies
        x[:700] += 30.0
    elif kind == "coarse":   # more equal largest logits than any list holds, far fewer than half of the row
        x = np.floor(np.abs(x))
        x[vocab // 3:vocab // 3 + 1500] = 20.0
    elif kind.startswith("around "):   # neighbours among the numbers of that size
        x = np.float32(float(kind[7:])) * (1 + rng.integers(0, 4, vocab) * np.float32(2.0 ** -7 if bf16 else 2.0 ** -23))
    return round_bf16(x) if bf16 else x.astype(np.float32)


def matrix(vocab, seed, bf16, kinds=KINDS):
    rng = np.random.default_rng(seed)
    return np.stack([logits_of(k, vocab, rng, bf16) for k in kinds])


def on_device(dev, x, bf16, pad):
    """The rows `pad` elements further apart than they are long, NaN in between."""
    rows, vocab = x.shape
    if not pad:
        return dev(x, bf16)
    base = np.full((rows, vocab + pad), np.nan, np.float32)
    base[:, :vocab] = x
    return dev(base, bf16)[:, :vocab]


def host(t):
    return t.float().cpu().numpy().astype(np.float64) if t.is_floating_point() else t.cpu().numpy()


# ---------------------------------------------------------------------------------------------------------------
# plain implementations, 64 bits
# ---------------------------------------------------------------------------------------------------------------
def plain_log_softmax(x, scale):
    with np.errstate(all="ignore"):
        t = x.astype(np.float64) * scale
        m = t.max(1, keepdims=True)
        lp = t - m - np.log(np.exp(t - m).sum(1, keepdims=True))
        lp[np.isnan(x).any(1) | (x == np.inf).any(1)] = np.nan
        lp[(x == -np.inf).all(1)] = -np.inf
    return lp


def plain_entropy(lp):
    with np.errstate(all="ignore"):
        p = np.exp(lp)
        return -np.where(p > 0, p * lp, np.where(np.isnan(p), np.nan, 0.0)).sum(1)


def plain_top(x, k):
    """Falling, NaN first, ties to the lowest index."""
    out = np.zeros((x.shape[0], k), np.int64)
    for r, row in enumerate(x):
        key = np.where(np.isnan(row), np.float64(4e38), np.where(row == np.inf, 3.9e38, row.astype(np.float64)))
        out[r] = np.argsort(-key, kind="stable")[:k]
    return out


def plain_gradient(x, lp, ids, coef, d_entropy, scale):
    """s ( sum c - p C - g p (ln p + H) ); zeros for rows without coefficients and rows of nothing but -inf."""
    rows, vocab = x.shape
    out = np.zeros((rows, vocab))
    for r in range(rows):
        c = coef[r] * ((ids[r] >= 0) & (ids[r] < vocab))
        g = 0.0 if d_entropy is None else d_entropy[r]
        if (not c.any() and g == 0) or (x[r] == -np.inf).all():
            continue
        with np.errstate(all="ignore"):
            p = np.exp(lp[r])
            out[r] = -p * c.sum()
            if g:
                out[r] -= g * np.where(p > 0, p * (lp[r] + plain_entropy(lp[r:r + 1])[0]), np.where(np.isnan(p), np.nan, 0.0))
            inside = (ids[r] >= 0) & (ids[r] < vocab)
            np.add.at(out[r], ids[r][inside], c[inside])
    return out * scale


def plain_teacher(ids, z, vocab, scale):
    used = (ids >= 0) & (ids < vocab)
    t = np.where(used, z.astype(np.float64) * scale, -np.inf)
    with np.errstate(all="ignore"):
        m = t.max(1, keepdims=True)
        e = np.where(t == -np.inf, 0.0, np.exp(t - m))
        total = e.sum(1, keepdims=True)
        q = np.where(total > 0, e / total, 0.0)
        logq = np.where(q > 0, t - m - np.log(total), 0.0)
    return q, logq


def plain_distill(x, ids, z, scale):
    lp = plain_log_softmax(x, scale)
    q, logq = plain_teacher(ids, z, x.shape[1], scale)
    at = np.take_along_axis(lp, np.clip(ids, 0, x.shape[1] - 1).astype(np.int64), 1)
    with np.errstate(all="ignore"):
        return np.where(q > 0, q * (logq - at), 0.0).sum(1) / scale ** 2, lp, q


# ---------------------------------------------------------------------------------------------------------------
# error bounds
# ---------------------------------------------------------------------------------------------------------------
def log_bound(x, scale, threads=64):
    """Per row: how far a log probability may be off (absolute)."""
    with np.errstate(all="ignore"):
        finite = np.isfinite(x)
        hi = np.where(finite, x, -np.inf).max(1)
        # logits more than 150 powers of two below the maximum have probability 0 and no part in the sum
        t = np.where(finite, (hi[:, None] - x.astype(np.float64)) * scale * np.log2(np.e), 0.0)
        T = np.where(t < 150, t, 0).max(1)
    n = (x.shape[1] + threads - 1) // threads + 16
    return U * (n + 5 * (T + 8) + 48)


def same(got, want, tol, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    tol = np.broadcast_to(np.asarray(tol, np.float64), want.shape)
    with np.errstate(over="ignore"):
        want = want.astype(np.float32).astype(np.float64)   # (past fp32's range: infinite)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), what
    off = np.abs(got[fine] - want[fine])
    bad = off > tol[fine]
    assert not bad.any(), (what, float(off[bad].max()), float(tol[fine][bad].min()), np.argwhere(fine)[bad][:4].tolist())


def logprob_tol(x, scale, want):
    """(a token far below the maximum: its own exponent's error)"""
    return log_bound(x, scale)[:, None] + 8 * U * np.where(np.isfinite(want), np.abs(want), 0.0)


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def alike(ids, vocab):
    """Few different tokens, most of them several times, and with equal lower 13 bits where the vocabulary has such."""
    return (ids % 3 % vocab + 8192 * (ids // 3 % max((vocab - 3) // 8192 + 1, 1))).astype(np.int32)


def tokens_of(rng, rows, vocab, n, few=False):
    ids = rng.integers(0, vocab, (rows, n)).astype(np.int32)
    if few:
        ids = alike(ids, vocab)
    if n > 2:
        ids[:, 1] = ids[:, 0]          # the same token twice
        ids[::2, 2] = -100             # no token
        ids[1::2, 2] = vocab
    return ids


def logprobs(S, dev, vocab, bf16, pad=0, n=1, k=4, scale=1.0, workspace=None, kinds=KINDS, seed=1, repeat=1, entropy=True,
             few=False):
    rng = np.random.default_rng(seed)
    x = matrix(vocab, seed + 1, bf16, kinds)
    rows = x.shape[0]
    ids = tokens_of(rng, rows, vocab, n, few)
    t = on_device(dev, x, bf16, pad)
    lp = plain_log_softmax(x, scale)
    tok = dev(ids[:, 0].copy() if n == 1 else ids)
    first = None
    for _ in range(repeat):
        got = S.token_logprobs(t, tok, top_k=k, scale=scale, entropy=entropy, workspace=workspace)
        if first is None:
            first = got
        for name in got:   # the same bits from every launch
            assert np.array_equal(host(got[name]), host(first[name]), equal_nan=True), name
    inside = (ids >= 0) & (ids < vocab)
    want = np.where(inside, np.take_along_axis(lp, np.clip(ids, 0, vocab - 1).astype(np.int64), 1), 0.0)
    same(host(got["logprob"]).reshape(rows, n), want, logprob_tol(x, scale, want), "logprob")
    if entropy:
        with np.errstate(all="ignore"):
            p = np.exp(lp)
            size = np.where(p > 0, p * np.abs(lp), 0.0).sum(1) + 18 + np.log(vocab)
        same(host(got["entropy"]), plain_entropy(lp), log_bound(x, scale) * size, "entropy")
    else:
        assert "entropy" not in got
    if k:
        top = plain_top(x, k)
        assert np.array_equal(host(got["top_ids"]), top), [KINDS[r] for r in range(rows) if not np.array_equal(host(got["top_ids"])[r], top[r])]
        want = np.take_along_axis(lp, top, 1)
        same(host(got["top_logprobs"]), want, logprob_tol(x, scale, want), "top")
    return t, tok, x, ids, lp, got


def gradient_tol(x, scale, lp, weight, want, bf16):
    """weight: what multiplies p (its error is log_bound relative); bf16: half a step of the result."""
    with np.errstate(all="ignore"):
        p = np.where(np.isfinite(lp), np.exp(lp), 0.0)
        spread = np.where(np.isfinite(lp), np.abs(lp), 0.0)
    tol = (log_bound(x, scale)[:, None] + 8 * U * spread) * p * weight[:, None] + 8 * U * (np.abs(np.nan_to_num(want)) + 1e-30) \
        + 4 * U * weight[:, None] * (p + (np.abs(np.nan_to_num(want)) > 0))
    return tol + (2.0 ** -8 * np.abs(np.nan_to_num(want)) + 2.0 ** -127 if bf16 else 2.0 ** -126)


def logprobs_backward(S, dev, vocab, bf16, pad=0, n=1, scale=1.0, entropy=True, in_place=False, kinds=KINDS, seed=5, few=False):
    t, tok, x, ids, lp, got = logprobs(S, dev, vocab, bf16, pad, n, 0, scale, kinds=kinds, seed=seed, entropy=entropy, few=few)
    rng = np.random.default_rng(seed + 100)
    rows = x.shape[0]
    g = rng.standard_normal((rows, n)).astype(np.float32)
    g[0] = 0.0
    ge = rng.standard_normal(rows).astype(np.float32) if entropy else None
    if entropy:
        ge[0] = 0.0       # row 0 takes no part
    coef = dev(g[:, 0].copy() if n == 1 else g)
    d = S.token_logprobs_backward(t, tok, got["stats"], d_logprob=coef, entropy=got.get("entropy"),
                                  d_entropy=None if ge is None else dev(ge), scale=scale, out=t if in_place else None)
    want = plain_gradient(x, lp, ids, g.astype(np.float64), ge, scale)
    with np.errstate(all="ignore"):
        H = np.nan_to_num(plain_entropy(lp))
    weight = scale * (np.abs(g).sum(1) + (np.abs(ge) * (20 + 2 * H) if entropy else 0.0))
    same(host(d), want, gradient_tol(x, scale, lp, weight, want, bf16), "d_logits")
    assert (host(d)[0] == 0).all()
    return d


def teacher_of(rng, rows, vocab, slots, teacher_bf16, few=False):
    ids = rng.integers(0, vocab, (rows, slots)).astype(np.int32)
    if few:
        ids = alike(ids, vocab)
    z = (rng.standard_normal((rows, slots)) * 2 + 3).astype(np.float32)
    if slots > 3:
        ids[:, 1] = ids[:, 0]           # the same token twice
        ids[::2, 2] = -1                # unused slots
        ids[1::2, 2] = vocab
        z[::3, 3] = -np.inf             # a slot without probability
    ids[2] = -1                         # a row without a slot
    if rows > 4:
        z[4] = -np.inf                  # and one whose slots have no probability
    return ids, (round_bf16(z) if teacher_bf16 else z)


def distillation(S, dev, vocab, bf16, pad=0, slots=8, scale=0.5, teacher_bf16=False, in_place=False, workspace=None,
                 kinds=KINDS, seed=9, repeat=1, few=False):
    rng = np.random.default_rng(seed)
    x = matrix(vocab, seed + 1, bf16, kinds)
    rows = x.shape[0]
    ids, z = teacher_of(rng, rows, vocab, slots, teacher_bf16, few)
    w = rng.standard_normal(rows).astype(np.float32)
    w[-1] = 0.0
    loss, lp, q = plain_distill(x, ids, z, scale)
    want = plain_gradient(x, lp, ids, -q * (w / np.float64(scale) ** 2)[:, None], None, scale)
    t, tid, tz, tw = on_device(dev, x, bf16, pad), dev(ids), dev(z, teacher_bf16), dev(w)
    apart = S.distillation_loss(t, tid, tz, scale=scale, workspace=workspace)
    assert "d_logits" not in apart
    d_apart = S.distillation_loss_backward(t, tid, tz, apart["stats"], tw, scale=scale)
    for _ in range(repeat):
        got = S.distillation_loss(t, tid, tz, scale=scale, d_loss=tw, out=t if in_place else None, workspace=workspace)
    size = np.where(np.isfinite(lp), np.abs(lp), 0.0).max(1) + 10
    with np.errstate(all="ignore"):
        at = np.take_along_axis(lp, np.clip(ids, 0, vocab - 1).astype(np.int64), 1)
        size = np.where(q > 0, q * np.nan_to_num(np.abs(at), posinf=0.0), 0.0).sum(1) + 20 + np.abs(np.nan_to_num(z, neginf=0.0)).max(1) * scale * 2
    tol = (log_bound(x, scale) + 8 * U * size + U * (slots + 40) * size) / scale ** 2
    weight = np.abs(w) / scale
    gtol = gradient_tol(x, scale, lp, weight, want, bf16)
    # q's own error: 5 u |t| + (slots + 40) u relative
    gtol = gtol + (U * (5 * 40 * scale + slots + 40) * weight)[:, None] * (np.abs(np.nan_to_num(want)) > 0)
    for name, g, d in (("apart", apart, d_apart), ("together", got, got["d_logits"])):
        same(host(g["row_loss"]), loss, tol, name + " row_loss")
        same(host(d), want, gtol, name + " d_logits")
    assert (host(got["d_logits"])[2] == 0).all() and (host(d_apart)[-1] == 0).all()
    assert host(got["row_loss"])[2] == 0
    return got


def teacher_to_student(S, dev, vocab=700, rows=6, slots=12, scale=0.5):
    """As they are used together: the teacher's top alternatives become the student's targets; loss and gradient, checked
    against differences of the 64-bit loss; the student's log probabilities and their gradient by differences too."""
    rng = np.random.default_rng(77)
    teacher, student = (rng.standard_normal((rows, vocab)).astype(np.float32) * 2 for _ in range(2))
    top = S.token_logprobs(dev(teacher), top_k=slots)
    assert "logprob" not in top and "entropy" not in top
    ids, z = top["top_ids"], top["top_logprobs"]   # log probabilities serve as logits: they differ by a constant
    w = np.full(rows, 1.0 / rows, np.float32)
    ts = dev(student)
    got = S.distillation_loss(ts, ids, z, scale=scale, d_loss=dev(w))
    ids_h, z_h = host(ids), host(z)
    assert np.array_equal(ids_h, plain_top(teacher, slots))
    loss, _, _ = plain_distill(student, ids_h, z_h, scale)
    same(host(got["row_loss"]), loss, 2e-5, "row_loss")
    d = host(got["d_logits"])
    direction = rng.standard_normal((rows, vocab))
    step = 1e-4
    up, down = (plain_distill((student + sign * step * direction), ids_h, z_h, scale)[0] @ w for sign in (1.0, -1.0))
    assert abs((up - down) / (2 * step) - (d * direction).sum()) < 1e-5   # step^2 and fp32 rounding of d: 1e-7 each
    tok = dev(ids_h[:, 0].astype(np.int32).copy())
    lp = S.token_logprobs(ts, tok, scale=scale, entropy=True)
    ge = np.full(rows, 0.3, np.float32)
    d = host(S.token_logprobs_backward(ts, tok, lp["stats"], d_logprob=dev(w), entropy=lp["entropy"], d_entropy=dev(ge), scale=scale))

    def value(x):
        a = plain_log_softmax(x, scale)
        return a[np.arange(rows), ids_h[:, 0]] @ w.astype(np.float64) + plain_entropy(a) @ ge.astype(np.float64)
    up, down = value(student + step * direction), value(student - step * direction)
    assert abs((up - down) / (2 * step) - (d * direction).sum()) < 1e-5


def parts_left_out(S, dev):
    """Every combination of what a call can be asked for; the entropy's gradient alone."""
    x = matrix(300, 3, False, KINDS[:6])
    rows = x.shape[0]
    t, tok = dev(x), dev(np.arange(rows, dtype=np.int32))
    whole = S.token_logprobs(t, tok, top_k=3, entropy=True)
    for tokens in (None, tok, tok.reshape(rows, 1)):
        for k in (0, 3):
            for entropy in (False, True):
                got = S.token_logprobs(t, tokens, top_k=k, entropy=entropy)
                assert set(got) == {"stats"} | ({"logprob"} if tokens is not None else set()) | \
                    ({"top_ids", "top_logprobs"} if k else set()) | ({"entropy"} if entropy else set())
                for name in got:
                    assert np.array_equal(host(got[name]).reshape(-1), host(whole[name]).reshape(-1)), name
                if tokens is not None:
                    assert got["logprob"].shape == tokens.shape
    ge = np.linspace(-1, 1, rows).astype(np.float32)
    d = S.token_logprobs_backward(t, None, whole["stats"], entropy=whole["entropy"], d_entropy=dev(ge))
    lp = plain_log_softmax(x, 1.0)
    want = plain_gradient(x, lp, np.full((rows, 1), -1), np.zeros((rows, 1)), ge, 1.0)
    with np.errstate(all="ignore"):
        weight = np.abs(ge) * (20 + 2 * np.nan_to_num(plain_entropy(lp)))
    same(host(d), want, gradient_tol(x, 1.0, lp, weight, want, False), "entropy's gradient")


def far_apart(S, dev, vocab, bf16, workspace=None):
    """Logits whose distance is past the largest fp32, though its product with a small scale, or its quotient by a large
    one, is not."""
    rng = np.random.default_rng(61)
    low, x = LOWEST[bf16], np.zeros((3, vocab), np.float32)
    x[:2, vocab // 3] = -low
    x[:, vocab // 2] = low
    x[1, 2::5] = low
    x[2] = low
    x[2, vocab - 1] = -low
    t = dev(x, bf16)
    ids = np.tile(np.int32([vocab // 3, vocab // 2, 0, vocab - 1]), (3, 1))
    for scale in (1e-4, 1e-3):
        lp = plain_log_softmax(x, scale)
        got = S.token_logprobs(t, dev(ids), top_k=3, scale=scale, entropy=True, workspace=workspace)
        want = np.take_along_axis(lp, ids.astype(np.int64), 1)
        assert np.isfinite(want).all() and want.min() < -1e34
        same(host(got["logprob"]), want, logprob_tol(x, scale, want), "logprob")
        assert (host(got["entropy"]) == 0).all()   # one token has all of the probability
        assert np.array_equal(host(got["top_ids"]), plain_top(x, 3))
        want = np.take_along_axis(lp, plain_top(x, 3), 1)
        same(host(got["top_logprobs"]), want, logprob_tol(x, scale, want), "top_logprobs")
    z = rng.standard_normal((3, 4)).astype(np.float32)
    for scale in (2.5, 40.0):   # loss: sum q (distance) / scale, 8 roundings of it beside the slots' 4
        loss, lp, q = plain_distill(x, ids, z, scale)
        assert np.isfinite(loss.astype(np.float32)).all() and loss.max() > 1e30
        w = dev(np.ones(3, np.float32))
        for d_loss in (None, w):
            got = S.distillation_loss(t, dev(ids), dev(z), scale=scale, d_loss=d_loss, workspace=workspace)
            # (q's error: 5 u |t| + (slots + 40) u relative, |t| the teacher's largest exponent)
            same(host(got["row_loss"]), loss, U * (12 + 44 + 5 * 8 * scale) * np.abs(loss), "row_loss")


def far_masks(S, dev, vocab, bf16, mask, scale, workspace=None):
    """Masks that are neither -inf nor the type's lowest value, but far below the other logits: what is behind them has
    probability 0."""
    kinds = ["behind %r" % mask] * 2 + ["normal", "masked", "behind %r" % mask, "empty"]
    logprobs(S, dev, vocab, bf16, 1, n=2, k=min(vocab, 12), scale=scale, workspace=workspace, kinds=kinds, seed=110)
    logprobs(S, dev, vocab, bf16, 0, n=1, k=0, scale=scale, workspace=workspace, kinds=kinds, seed=111, entropy=False)
    distillation(S, dev, vocab, bf16, 0, slots=6, scale=scale, workspace=workspace, kinds=kinds, seed=112)


def far_from_zero(S, dev, vocab, bf16, value, scale, workspace=None):
    """Logits so far from zero that neighbouring scaled values are hundreds of powers of two apart, as a mask, as whole
    rows and as the row's largest."""
    kinds = ["behind %r" % value, "all of %r" % value, "normal", "around %r" % value, "masked", "all of %r" % value,
             "behind %r" % value]
    logprobs(S, dev, vocab, bf16, 1, n=2, k=min(vocab, 12), scale=scale, workspace=workspace, kinds=kinds, seed=120)
    logprobs(S, dev, vocab, bf16, 0, n=1, k=0, scale=scale, workspace=workspace, kinds=kinds, seed=121, entropy=False)
    logprobs_backward(S, dev, vocab, bf16, 0, n=2, scale=scale, kinds=kinds, seed=122)
    distillation(S, dev, vocab, bf16, 0, slots=6, scale=scale, workspace=workspace, kinds=kinds, seed=123)


def large_weights(S, dev, vocab, bf16, scale, weight, workspace=None, slots=9):
    """Gradients d_loss / scale (p - q) that are ordinary numbers where d_loss / scale^2 is past the largest fp32."""
    rng = np.random.default_rng(140)
    x = (rng.standard_normal((5, vocab)) * 2 / scale).astype(np.float32)
    x = round_bf16(x) if bf16 else x
    ids = rng.integers(0, vocab, (5, slots)).astype(np.int32)
    ids[:, 1] = ids[:, 0]
    z = (rng.standard_normal((5, slots)) * 2 / scale).astype(np.float32)
    w = (np.float64(weight) * (1 + rng.random(5))).astype(np.float32)
    w[3] = 0.0
    _, lp, q = plain_distill(x, ids, z, scale)
    want = plain_gradient(x, lp, ids, -q * (w / np.float64(scale) ** 2)[:, None], None, scale)
    assert np.isfinite(want.astype(np.float32)).all()
    tol = gradient_tol(x, scale, lp, np.abs(w) / scale, want, bf16)
    # named entries: q's own error, 5 u |t| + (slots + 40) u relative, |t| <= 40
    named = np.zeros(want.shape)
    np.put_along_axis(named, ids.astype(np.int64), 1.0, 1)
    tol = tol + (U * (5 * 40 + slots + 40) * np.abs(w) / scale)[:, None] * named
    t, tid, tz, tw = dev(x, bf16), dev(ids), dev(z), dev(w)
    got = S.distillation_loss(t, tid, tz, scale=scale, d_loss=tw, workspace=workspace)
    same(host(got["d_logits"]), want, tol, "together")
    same(host(S.distillation_loss_backward(t, tid, tz, got["stats"], tw, scale=scale)), want, tol, "apart")


def one_row_of_many(S, dev, rows=1, apart=64, vocab=50):
    """Rows far apart (one position of every sequence): the gradient has their distance, but a single row has none."""
    base = dev(np.random.default_rng(150).standard_normal((rows, apart * vocab)).astype(np.float32))
    x = base[:, (apart - 2) * vocab:(apart - 1) * vocab]
    assert x.stride(0) == apart * vocab
    tok, w = dev(np.arange(rows, dtype=np.int32)), dev(np.ones(rows, np.float32))
    lp = S.token_logprobs(x, tok)
    d = S.token_logprobs_backward(x, tok, lp["stats"], d_logprob=w)
    both = S.distillation_loss(x, tok[:, None], w[:, None], d_loss=w)
    for got in (d, both["d_logits"], S.distillation_loss_backward(x, tok[:, None], w[:, None], both["stats"], w)):
        assert got.shape == x.shape
        assert got.untyped_storage().nbytes() == 4 * vocab * (1 if rows == 1 else rows * apart)
    p = np.exp(plain_log_softmax(host(x).astype(np.float32), 1.0))
    p[np.arange(rows), np.arange(rows)] -= 1
    assert np.abs(host(d) + p).max() < 1e-6 and np.abs(host(both["d_logits"]) - p).max() < 1e-6


def refusals(S, dev):
    """Calls that are turned away, with the status that says why."""
    import pytest
    import torch
    x = dev(np.zeros((3, 40), np.float32))
    tok = dev(np.zeros(3, np.int32))
    stats = dev(np.zeros((3, 2), np.float32))
    row = dev(np.zeros(3, np.float32))
    ids, z = dev(np.zeros((3, 5), np.int32)), dev(np.zeros((3, 5), np.float32))

    def turned_away(status, call):
        with pytest.raises(S.SfbError) as e:
            call()
        assert e.value.status == ERR[status], (status, e.value)

    turned_away("shape", lambda: S.token_logprobs(x[0], tok))                       # one dimension
    turned_away("shape", lambda: S.token_logprobs(x[:0], tok[:0]))                  # no rows
    turned_away("shape", lambda: S.token_logprobs(x[:, :0], tok))                   # no columns
    turned_away("shape", lambda: S.token_logprobs(x.t(), tok))                      # columns apart
    turned_away("shape", lambda: S.token_logprobs(x[:1].expand(3, 40), tok))        # rows on top of each other
    turned_away("shape", lambda: S.token_logprobs(x, tok[:2]))
    turned_away("shape", lambda: S.token_logprobs(x, top_k=41))                     # more than the vocabulary
    turned_away("shape", lambda: S.token_logprobs(dev(np.zeros((1, 100), np.float32)), top_k=65))
    turned_away("shape", lambda: S.token_logprobs(x, dev(np.zeros((3, 257), np.int32))))
    turned_away("shape", lambda: S.token_logprobs(x, tok.reshape(3, 1, 1)))
    turned_away("shape", lambda: S.token_logprobs(x, tok[0]))
    turned_away("shape", lambda: S.token_logprobs(x, top_k=-1))
    turned_away("shape", lambda: S.distillation_loss(x, ids[0], z[0]))
    turned_away("shape", lambda: S.token_logprobs_backward(x, tok, stats, d_logprob=row[:2]))
    turned_away("dtype", lambda: S.token_logprobs(x.double(), tok))
    turned_away("dtype", lambda: S.token_logprobs(x, tok.long()))
    turned_away("align", lambda: S.token_logprobs(x[:, 1:], tok))                   # first element off 16 bytes
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e-5, 1e5):
        turned_away("arg", lambda: S.token_logprobs(x, tok, scale=scale))
        turned_away("arg", lambda: S.distillation_loss(x, ids, z, scale=scale))
    turned_away("arg", lambda: S.token_logprobs_backward(x, tok, stats))            # nothing to differentiate
    turned_away("null", lambda: S.token_logprobs_backward(x, None, stats, d_logprob=row))
    turned_away("null", lambda: S.token_logprobs_backward(x, tok, stats, d_logprob=row, d_entropy=row))   # needs the entropy
    turned_away("null", lambda: S.token_logprobs_backward(x, tok, None, d_logprob=row))
    turned_away("shape", lambda: S.token_logprobs_backward(x, tok, row, d_logprob=row))
    turned_away("shape", lambda: S.token_logprobs_backward(x, tok, stats, d_logprob=row, out=dev(np.zeros((3, 41), np.float32))))
    turned_away("shape", lambda: S.token_logprobs_backward(x, tok, stats, d_logprob=row, out=dev(np.zeros((3, 48), np.float32))[:, :40]))
    turned_away("shape", lambda: S.distillation_loss(x, ids[:, :0], z[:, :0]))
    turned_away("shape", lambda: S.distillation_loss(x, ids, z[:, :4].contiguous()))
    turned_away("shape", lambda: S.distillation_loss(x, dev(np.zeros((3, 257), np.int32)), dev(np.zeros((3, 257), np.float32))))
    turned_away("dtype", lambda: S.distillation_loss(x, ids, z.double()))
    turned_away("dtype", lambda: S.distillation_loss(x, ids.long(), z))
    turned_away("null", lambda: S.distillation_loss(x, ids, z, out=x))              # a gradient without d_loss
    turned_away("shape", lambda: S.distillation_loss(x, ids, z, d_loss=row[:2]))
    turned_away("shape", lambda: S.distillation_loss_backward(x, ids, z, row, row))
    turned_away("null", lambda: S.distillation_loss_backward(x, ids, z, stats, None))
    small = dev(np.zeros(4096, np.uint8))
    turned_away("workspace", lambda: S.token_logprobs(x, tok, workspace=small))
    turned_away("workspace", lambda: S.distillation_loss(x, ids, z, workspace=small))
    big = dev(np.zeros(S.LOGIT_WORKSPACE_BYTES + 16, np.uint8))
    turned_away("align", lambda: S.token_logprobs(x, tok, workspace=big[4:]))
    assert torch.equal(x, torch.zeros_like(x))
