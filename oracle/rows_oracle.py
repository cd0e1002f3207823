"""The builtins on rows and weights - layer norm, log probabilities, AdamW - from their formulas in 64 bits.
TEST INFRASTRUCTURE ONLY.  numpy float32 in, float32 out."""
import numpy as np


def _f32(x):
    return np.asarray(x, np.float64).astype(np.float32)


def flayernorm(x, gamma, beta, eps):
    """(out, mean, rstd) over the last dimension."""
    a = np.asarray(x, np.float64)
    mean = a.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(((a - mean) ** 2).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
    out = (a - mean) * rstd * np.asarray(gamma, np.float64) + np.asarray(beta, np.float64)
    return _f32(out), _f32(mean[..., 0]), _f32(rstd[..., 0])


def flayernorm_grad(gradient, x, gamma, mean, rstd):
    """(dx, dgamma, dbeta)."""
    cols = x.shape[-1]
    g, a = (np.asarray(t, np.float64).reshape(-1, cols) for t in (gradient, x))
    m, r = (np.asarray(t, np.float64).reshape(-1, 1) for t in (mean, rstd))
    h, q = (a - m) * r, g * np.asarray(gamma, np.float64)
    dx = r * (q - q.mean(1, keepdims=True) - h * (q * h).mean(1, keepdims=True))
    return _f32(dx).reshape(x.shape), _f32((g * h).sum(0)), _f32(g.sum(0))


def flogprob(logits, ids, top=0):
    """(logprob, entropy, logsumexp, top ids, top logprobs); finite logits and ids of classes or below zero."""
    a, ids = np.asarray(logits, np.float64), np.asarray(ids).astype(np.int64)
    m = a.max(1, keepdims=True)
    e = np.exp(a - m)
    lse = m + np.log(e.sum(1, keepdims=True))
    l = a - lse
    lp = np.where(ids < 0, 0.0, l[np.arange(len(ids)), np.maximum(ids, 0)])
    order = np.argsort(-a, axis=1, kind="stable")[:, :top]
    return _f32(lp), _f32(-(np.exp(l) * l).sum(1)), _f32(lse[:, 0]), order, _f32(np.take_along_axis(l, order, 1))


def flogprob_grad(logits, ids, logsumexp, entropy, g_logprob, g_entropy):
    a, ids = np.asarray(logits, np.float64), np.asarray(ids).astype(np.int64)
    l = a - np.asarray(logsumexp, np.float64)[:, None]
    g = np.where(ids < 0, 0.0, np.asarray(g_logprob, np.float64))
    d = -np.exp(l) * g[:, None]
    if g_entropy is not None:
        d -= np.exp(l) * np.asarray(g_entropy, np.float64)[:, None] * (l + np.asarray(entropy, np.float64)[:, None])
    d[np.arange(len(ids)), np.maximum(ids, 0)] += g
    return _f32(d)


def fadamw(w, g, m, v, step, lr, beta1, beta2, eps, decay):
    """(weights, first, second) with moments in 32 bits, whose products and sums are rounded one by one."""
    f = np.float32
    w, g, m, v = (np.asarray(t, f) for t in (w, g, m, v))
    b1, b2 = f(beta1), f(beta2)
    m = m * b1 + g * (f(1) - b1)
    v = v * b2 + g * (f(1) - b2) * g
    c1, c2, lr = 1 - float(b1) ** step, 1 - float(b2) ** step, float(f(lr))
    update = lr / c1 * m.astype(np.float64) / (np.sqrt(v.astype(np.float64) / c2) + float(f(eps)))
    return _f32(w.astype(np.float64) * (1 - lr * float(f(decay))) - update), m, v


def to_e4m3(y):
    """float32 to e4m3 codes: to nearest even, saturating at 448; NaN is 0x7f."""
    y = np.asarray(y, np.float32)
    a = np.minimum(np.where(np.isnan(y), 0, np.abs(y)).astype(np.float64), 448.0)
    exponent = np.maximum(np.frexp(a)[1] - 1, -6)            # of the step 2^(exponent - 3); -6 for what is subnormal
    a = np.minimum(np.rint(a / 2.0 ** (exponent - 3)) * 2.0 ** (exponent - 3), 448.0)
    exponent = np.maximum(np.frexp(a)[1] - 1, -6)
    code = np.where(a < 2.0 ** -6, a * 2.0 ** 9, (exponent + 7) * 8 + (a / 2.0 ** exponent - 1) * 8)
    code = np.where(np.isnan(y), 0x7f, code).astype(np.uint8)
    return code | np.where(np.signbit(y) & ~np.isnan(y), 0x80, 0).astype(np.uint8)


def from_e4m3(code):
    code = np.asarray(code, np.uint8)
    exponent, digits = (code >> 3 & 15).astype(int), (code & 7).astype(np.float64)
    a = np.where(exponent == 0, digits * 2.0 ** -9, (1 + digits / 8) * 2.0 ** (exponent - 7))
    a = np.where((code & 0x7f) == 0x7f, np.nan, a)
    return np.where(code & 0x80, -a, a).astype(np.float32)


def fadamw8(w, g, first, first_scales, second, second_scales, step, lr, beta1, beta2, eps, decay):
    """(weights, first, first scales, second, second scales) with moments as e4m3 codes in blocks of 128, one scale each."""
    f, n = np.float32, np.size(w)
    w, g = np.asarray(w, f), np.asarray(g, f)

    def blocks(x):
        x = np.ravel(x)
        return np.concatenate([x, np.zeros(-len(x) % 128, x.dtype)]).reshape(-1, 128)

    def held(x, never_zero):
        largest = np.abs(x).max(1)
        scale = np.where(largest < f(2.0 ** -100), f(0), largest * f(1 / 448)).astype(f)
        by = np.where(scale == 0, f(0), f(1) / np.where(scale == 0, f(1), scale)).astype(f)
        code = to_e4m3(x * by[:, None])
        if never_zero:
            code[(code == 0) & (x > 0) & (scale > 0)[:, None]] = 1
        return code.ravel()[:n], scale

    b1, b2 = f(beta1), f(beta2)
    m = from_e4m3(blocks(first)) * np.asarray(first_scales, f).ravel()[:, None]
    u = from_e4m3(blocks(second)) * np.asarray(second_scales, f).ravel()[:, None]
    m = m * b1 + blocks(g) * (f(1) - b1)
    u = np.sqrt(u * u * b2 + blocks(g) * (f(1) - b2) * blocks(g))
    m64, u64 = (x.ravel()[:n].reshape(w.shape).astype(np.float64) for x in (m, u))
    c1, c2, lr = 1 - float(b1) ** step, 1 - float(b2) ** step, float(f(lr))
    new = _f32(w.astype(np.float64) * (1 - lr * float(f(decay))) - lr / c1 * m64 / (u64 / np.sqrt(c2) + float(f(eps))))
    return (new, *held(m, False), *held(u, True))


def _tokens(ids, offsets):
    """The sequence of each token of [offsets[0], offsets[-1]), and which of them count."""
    offsets = np.asarray(offsets).astype(np.int64)
    of = np.repeat(np.arange(len(offsets) - 1), np.diff(offsets))
    counts = ~(np.asarray(ids)[offsets[0]:offsets[-1]] < 0) if len(of) else np.zeros(0, bool)
    return of, counts, slice(int(offsets[0]), int(offsets[0]) + len(of))


def policy_loss64(logprob, old, reference, entropy, advantage, ids, offsets, clip_low, clip_high, kl_weight, entropy_weight, by_sequence=False,
                  per_token=False, count=0.0):
    """(loss[5], g_logprob, g_entropy, size) in 64 bits; NaN outside the sequences.  size: per token, what the terms of its gradient come to by
    magnitude, and the same for the five sums, for bounds of rounding errors."""
    f = lambda v: float(np.float32(v))  # noqa: E731
    low, high, beta, alpha = f(clip_low), f(clip_high), f(kl_weight), f(entropy_weight)
    of, counts, span = _tokens(ids, offsets)
    n, sequences = len(ids), len(offsets) - 1
    per = np.bincount(of[counts], minlength=sequences)
    units = f(count) if count > 0 else max((per > 0).sum() if by_sequence else counts.sum(), 1)
    w = counts / units / (np.maximum(per, 1)[of] if by_sequence else 1)
    pick = lambda t: np.where(counts, np.asarray(t, np.float64)[span], 0.0)  # noqa: E731
    lp, a = pick(logprob), np.asarray(advantage, np.float64)
    a = np.where(counts, a[span] if per_token else a[of], 0.0)
    d = lp - pick(old)
    with np.errstate(over="ignore", invalid="ignore"):
        free = np.exp(d) * a
        over, under = d > np.log1p(high), (d < np.log1p(-low) if low < 1 else np.zeros(len(d), bool))
        cut = (over & (a > 0)) | (under & (a < 0))
        surrogate = np.where(cut, np.where(over, 1 + high, 1 - low) * a, free)
        slope = np.where(cut, 0.0, -free)
        q = pick(reference) - lp if reference is not None else np.zeros(len(lp))
        kl = np.where(np.abs(q) < 1e-3, q * q * (0.5 + q / 6 + q * q / 24), np.expm1(q) - q)
        beta = beta if reference is not None else 0.0
        h = pick(entropy) if entropy is not None else np.zeros(len(lp))
        alpha = alpha if entropy is not None else 0.0
        # (a term of weight zero is none, whatever its arrays hold)
        grown = np.expm1(q) if beta != 0 else np.zeros(len(q))
        g = np.where(counts, (slope - beta * grown) * w, 0.0)
        parts = [np.where(counts, t * w, 0.0) for t in (surrogate, kl, h, cut * 1.0)]
        sums = [t.sum() for t in parts]
        # (an exponential has its argument's rounding times the argument)
        sizes = [np.abs(t * by).sum() for t, by in zip(parts, (1 + np.abs(d) * ~cut, 1 + np.abs(q), 1.0, 1.0))]
        loss = np.array([sum(by * t for by, t in ((-1.0, sums[0]), (beta, sums[1]), (-alpha, sums[2])) if by != 0), *sums])
        size = np.array([beta * sizes[1] + sizes[0] + alpha * sizes[2], *sizes])
        token = w * (np.abs(slope) * (1 + np.abs(d)) + np.abs(beta * grown) + (np.abs(beta * q * np.exp(q)) if beta != 0 else 0.0))
    spread = lambda v: np.concatenate([np.full(span.start, np.nan), v, np.full(n - span.stop, np.nan)])  # noqa: E731
    return loss, spread(g), spread(-alpha * w), (size, spread(np.where(counts, token, 0.0)))


def _over(old, new):
    """Gradients outside the sequences stay as they were."""
    return np.where(np.isnan(new) & ~np.isnan(old), old, new) if old is not None else new


def preference_loss64(logprob, reference, ids, offsets, beta, smoothing, margin, average=False, count=0.0):
    """(loss[3], rewards, g_logprob, size) in 64 bits; NaN outside the sequences.  size: the sum of each sequence by magnitude."""
    f = lambda v: float(np.float32(v))  # noqa: E731
    beta, e, margin = f(beta), f(smoothing), f(margin)
    of, counts, span = _tokens(ids, offsets)
    n, sequences = len(ids), len(offsets) - 1
    ratio = np.asarray(logprob, np.float64)[span] - (np.asarray(reference, np.float64)[span] if reference is not None else 0.0)
    ratio = np.where(counts, ratio, 0.0)
    per = np.maximum(np.bincount(of[counts], minlength=sequences), 1) if average else np.ones(sequences)
    total = np.bincount(of, weights=ratio, minlength=sequences) / per
    rewards = beta * total
    gap = rewards[0::2] - rewards[1::2]
    z = gap - margin
    units = f(count) if count > 0 else max(len(gap), 1)
    # (a side of weight zero is none, also where z is infinite)
    loss = sum(by * np.logaddexp(0, side) for by, side in ((1 - e, -z), (e, z)) if by != 0)
    with np.errstate(over="ignore"):
        slope = (e / (1 + np.exp(-z)) - (1 - e) / (1 + np.exp(z))) * beta / units
    g = np.where(counts, (np.stack([slope, -slope], 1).ravel() / per)[of], 0.0)
    out = np.array([loss.sum(), (gap > 0).sum(), gap.sum()]) / units
    return out, rewards, np.concatenate([np.full(span.start, np.nan), g, np.full(n - span.stop, np.nan)]), z


def fpolicy_loss(logprob, old, reference, entropy, advantage, ids, offsets, clip_low, clip_high, kl_weight, entropy_weight, count, by_sequence,
                 g_logprob, g_entropy, per_token=None):
    """(loss[5], g_logprob, g_entropy) as the builtin of a program gives them.  per_token: whether the advantage is one for each token; None: its size tells."""
    tokens = len(ids)
    if per_token is None:
        if tokens == len(offsets) - 1 and tokens > 1:
            raise ValueError("fpolicy_loss: as many sequences as tokens: whose are the advantages?")
        per_token = np.size(advantage) == tokens
    if np.size(advantage) != (tokens if per_token else len(offsets) - 1):
        raise ValueError("fpolicy_loss: shapes do not agree")
    loss, g, ge, _ = policy_loss64(logprob, old, reference, entropy, advantage, ids, offsets, clip_low, clip_high, kl_weight, entropy_weight, bool(by_sequence),
                                   per_token, count)
    return _f32(loss), _f32(_over(g_logprob, g)), _f32(_over(g_entropy, ge))


def fpreference_loss(logprob, reference, ids, offsets, beta, smoothing, margin, count, average, g_logprob):
    """(loss[3], rewards, g_logprob)."""
    loss, rewards, g, _ = preference_loss64(logprob, reference, ids, offsets, beta, smoothing, margin, bool(average), count)
    return _f32(loss), _f32(rewards), _f32(_over(g_logprob, g))


def muon64(w, g, m, lr, momentum, nesterov, steps, decay, scale, a=3.4445, b=-4.7750, c=2.0315):
    """(weights, momentum, update) of one matrix in 64 bits; update: the orthogonalised matrix."""
    f = lambda v: float(np.float32(v))  # noqa: E731
    mu, lr = f(momentum), f(lr)
    g, m = np.asarray(g, np.float64), np.asarray(m, np.float64)
    m = mu * m + g
    u = g + mu * m if nesterov else m
    size = np.sqrt((u * u).sum())
    x = u / size if size != 0 else u
    x = x if x.shape[0] <= x.shape[1] else x.T
    for _ in range(int(steps)):
        gram = x @ x.T
        x = f(a) * x + (f(b) * gram + f(c) * gram @ gram) @ x
    x = x if x.shape == g.shape else x.T
    return np.asarray(w, np.float64) * (1 - lr * f(decay)) - lr * f(scale) * x, m, x


def fmuon(w, g, m, lr, momentum, nesterov, steps, decay, scale):
    """(weights, momentum) of matrices [..., rows, cols]."""
    shape = np.shape(w)
    flat = [np.reshape(t, (-1, *shape[-2:])) for t in (w, g, m)]
    r = [muon64(*t, lr, momentum, nesterov, steps, decay, scale)[:2] for t in zip(*flat)]
    return _f32(np.stack([x[0] for x in r]).reshape(shape)), _f32(np.stack([x[1] for x in r]).reshape(shape))
