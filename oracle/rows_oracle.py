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
