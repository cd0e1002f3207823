"""What stands around the matrix products of a training or answering step, as cases that can be timed and compared:

  norm           layer norm of every row: a single token's row up to a full batch of hidden activations
  norm_grad      its backward pass with the weights' gradients
  logprob        log probability of a given token or class per row, the row's entropy and its likeliest alternatives
  logprob_grad   the gradient at the logits
  adamw          one AdamW step over all weights of a network, its moments held in 32 or in 8 bits

`run` computes them in elementary torch operations or, where `own` is true, with the builtins of this package.
All tensors are float32 but ids (int64) and moments in 8 bits (e4m3 codes with a float32 scale for each block of 128).
"""
import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-5                                # layer norm
BETA1, BETA2, ADAM_EPS, DECAY, RATE = 0.9, 0.999, 1e-8, 0.01, 1e-3
BLOCK = 128                               # values per scale of an 8-bit moment
LEAST = 2.0 ** -100                       # a block whose largest value is below this is held as zeros
INV_MAX = 0.0022321429569274187           # float32 nearest to 1 / 448, the largest e4m3 value


def listed():
    return [
        # one hidden vector of a serving step
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 4096},
        # the hidden activations of the benchmark's full batch
        {"name": "norm_65536x4096", "kind": "norm", "rows": 65536, "cols": 4096},
        # the same in training
        {"name": "norm_grad_65536x4096", "kind": "norm_grad", "rows": 65536, "cols": 4096},
        # a batch and a width that are no multiples of anything
        {"name": "norm_grad_ragged", "kind": "norm_grad", "rows": 2001, "cols": 1511},
        # a sampled token's log probability and twenty alternatives, as a server reports them
        {"name": "logprob_token", "kind": "logprob", "rows": 1, "classes": 131072, "top": 20, "masked": False},
        # scoring prompts of a padded batch: odd vocabulary, part of it masked, some alternatives
        {"name": "logprob_prompt", "kind": "logprob", "rows": 2048, "classes": 50001, "top": 5, "masked": True},
        # the classes of the benchmark's network, one row per sample
        {"name": "logprob_classes", "kind": "logprob", "rows": 65536, "classes": 10, "top": 0, "masked": False},
        # the loss gradient of a training batch of tokens
        {"name": "logprob_grad_8192x32000", "kind": "logprob_grad", "rows": 8192, "classes": 32000, "entropy": False, "masked": False},
        # with an entropy term, as policy gradients have, on a ragged and partly padded batch
        {"name": "logprob_grad_ragged", "kind": "logprob_grad", "rows": 999, "classes": 10007, "entropy": True, "masked": True},
        # the benchmark's network with its norm: four tensors
        {"name": "adamw_mlp", "kind": "adamw", "bits": 32, "layers": 0, "width": 784, "inner": 4096, "classes": 10},
        # a token model's weights: one large table, many matrices, many vectors
        {"name": "adamw_many", "kind": "adamw", "bits": 32, "layers": 16, "width": 1024, "inner": 4096, "classes": 32768},
        # the same with its moments in 8 bits
        {"name": "adamw8_many", "kind": "adamw", "bits": 8, "layers": 16, "width": 1024, "inner": 4096, "classes": 32768},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _size(rng, lo, hi):
    """Half of them multiples of 16, as widths usually are, half as they come."""
    v = _log(rng, lo, hi)
    return min(hi, max(16, (v + 8) // 16 * 16)) if rng.random() < 0.5 else v


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "logprob", "logprob", "logprob_grad", "adamw", "adamw"])
    if kind in ("norm", "norm_grad"):
        cols = _size(rng, 24, 32768)
        return {"kind": kind, "rows": _log(rng, 1, min(65536, (1 << 28) // cols)), "cols": cols}
    if kind == "adamw":
        width = _size(rng, 24, 1024)
        return {"kind": kind, "bits": rng.choice([32, 8]), "layers": rng.randint(0, 16), "width": width,
                "inner": _size(rng, 32, 4096), "classes": _log(rng, 10, 32768)}
    classes = _size(rng, 2, 131072)
    case = {"kind": kind, "rows": _log(rng, 1, min(65536, (1 << 27) // classes)), "classes": classes, "masked": rng.random() < 0.5}
    if kind == "logprob":
        return {**case, "top": min(classes, rng.choice([0, 1, 5, 20, 32]))}
    return {**case, "entropy": rng.random() < 0.5}


# ---- inputs

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(g, *shape, scale=1.0, mean=0.0):
    return torch.empty(shape, device=DEVICE).normal_(mean, scale, generator=g)


def _logits(g, case):
    """Logits as a trained model gives them: a broad bell and, in most rows, a favourite; `masked`: an eighth of the classes
    is shut out in every third row, and one row is shut out altogether."""
    rows, classes = case["rows"], case["classes"]
    x = _normal(g, rows, classes, scale=2.0)
    at = torch.randint(0, classes, (rows,), device=DEVICE, generator=g)
    r = torch.arange(rows, device=DEVICE)
    x[r, at] += _normal(g, rows, scale=3.0, mean=8.0)
    ids = torch.where(torch.rand(rows, device=DEVICE, generator=g) < 0.7, at,
                      torch.randint(0, classes, (rows,), device=DEVICE, generator=g))
    if case["masked"]:
        shut = torch.rand(classes, device=DEVICE, generator=g) < 0.125
        shut[0] = False
        x[::3].masked_fill_(shut, -math.inf)
        if rows > 2:
            x[rows // 2] = -math.inf
        ids[1:][torch.rand(rows - 1, device=DEVICE, generator=g) < 0.2] = -1      # padding
    return x, ids


def _tensors(case):
    """The shapes of a network's weights: a table and a norm, and per layer four square matrices, two to and from the inner
    width, and two norms of two vectors.  No layers: the benchmark's two matrices and their norm."""
    w, i, c = case["width"], case["inner"], case["classes"]
    if case["layers"] == 0:
        return [(w, i), (i, c), (i,), (i,)]
    return [(c, w), (w,), (w,)] + case["layers"] * (4 * [(w, w)] + [(w, i), (i, w)] + 4 * [(w,)])


def _views(flat, shapes):
    """A network's tensors in one allocation, each on a boundary of 128 values, as memory pools place them."""
    at = [0]
    for t in shapes:
        at.append(at[-1] + -(-math.prod(t) // BLOCK) * BLOCK)
    return [flat[a:a + math.prod(t)].view(t) for a, t in zip(at, shapes)]


def _blocks(t):
    """Its values in rows of one block, the last one filled up with zeros."""
    return torch.nn.functional.pad(t.reshape(-1), (0, -t.numel() % BLOCK)).view(-1, BLOCK)


def _in_8_bits(flat):
    """Moments as e4m3 codes and a scale for each block."""
    x = flat.view(-1, BLOCK)
    scale = x.abs().amax(1) * INV_MAX
    return (x / torch.where(scale > 0, scale, 1.0)[:, None]).to(torch.float8_e4m3fn).view(-1), scale


def prepare(case, seed):
    g, kind = _generator(seed), case["kind"]
    new = lambda *s, **k: torch.empty(s, device=DEVICE, **k)  # noqa: E731
    s = {"case": case}
    if kind in ("norm", "norm_grad"):
        rows, cols = case["rows"], case["cols"]
        # rows of their own place and size, as activations have
        s["x"] = _normal(g, rows, cols).mul_(torch.rand((rows, 1), device=DEVICE, generator=g) + 0.5).add_(_normal(g, rows, 1))
        s["gamma"], s["beta"] = _normal(g, cols, scale=0.1, mean=1.0), _normal(g, cols, scale=0.1)
        if kind == "norm":
            s["out"], s["mean"], s["rstd"] = new(rows, cols), new(rows), new(rows)
        else:
            s["gradient"] = _normal(g, rows, cols, scale=1e-2)
            s["mean"] = s["x"].mean(1)
            s["rstd"] = 1 / torch.sqrt(s["x"].var(1, unbiased=False) + EPS)
            s["dx"], s["dgamma"], s["dbeta"] = new(rows, cols), new(cols), new(cols)
        return s
    if kind in ("logprob", "logprob_grad"):
        rows = case["rows"]
        s["logits"], s["ids"] = _logits(g, case)
        if kind == "logprob":
            s["out"] = {"logprob": new(rows), "entropy": new(rows), "logsumexp": new(rows)}
            if case["top"]:
                s["out"]["top_ids"] = new(rows, case["top"], dtype=torch.int64)
                s["out"]["top_logprob"] = new(rows, case["top"])
        else:
            s["lse"], s["entropy"] = new(rows), new(rows)
            for a in range(0, rows, 1024):                   # what the forward pass left, here in 64 bits
                l = s["logits"][a:a + 1024].double()
                lse = torch.logsumexp(l, 1)
                l = l - torch.where(torch.isinf(lse), 0.0, lse)[:, None]
                s["lse"][a:a + 1024] = lse.float()
                s["entropy"][a:a + 1024] = -torch.nan_to_num(l.exp() * l).sum(1).float()
            s["g_logprob"] = torch.full((rows,), -1.0 / rows, device=DEVICE) * (torch.rand(rows, device=DEVICE, generator=g) + 0.5)
            s["g_entropy"] = _normal(g, rows, scale=0.1 / rows) if case["entropy"] else None
            s["dlogits"] = new(rows, case["classes"])
        return s
    shapes = _tensors(case)
    s["step"], s["shapes"] = 10 + seed % 1000, shapes
    total = sum(-(-math.prod(t) // BLOCK) * BLOCK for t in shapes)
    flat = {"w": (0.02, 0), "g": (1e-3, 0), "m": (3e-4, 0), "v": (1e-3, 0)}
    flat = {k: _normal(g, total, scale=a, mean=b) for k, (a, b) in flat.items()}
    flat["v"].square_()
    for t in (_views(flat[k], shapes)[0] for k in "gmv"):
        t[::2] = 0                                           # rows of the table that no batch has had
    s["weights"], s["gradients"] = _views(flat["w"], shapes), _views(flat["g"], shapes)
    s["out"] = {"weights": flat["w"]}
    if case["bits"] == 8:
        flat["v"].sqrt_()                                    # held as its root
        for k, name in (("m", "first"), ("v", "second")):
            codes, scales = _in_8_bits(flat[k])
            s["out"][name], s["out"][name + "_scales"] = codes, scales
            s[name] = _views(codes, shapes)
            s[name + "_scales"] = torch.split(scales, [-(-math.prod(t) // BLOCK) for t in shapes])
    else:
        s["out"]["first"], s["out"]["second"] = flat["m"], flat["v"]
        s["first"], s["second"] = _views(flat["m"], shapes), _views(flat["v"], shapes)
    return s


# ---- the plain forms, in 32 bits

def _norm(s):
    x = s["x"]
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1 / torch.sqrt((d * d).mean(1) + EPS)
    return {"out": d * rstd[:, None] * s["gamma"] + s["beta"], "mean": mean, "rstd": rstd}


def _norm_grad(s):
    h = (s["x"] - s["mean"][:, None]) * s["rstd"][:, None]
    dy = s["gradient"]
    q = dy * s["gamma"]
    dx = s["rstd"][:, None] * (q - q.mean(1, keepdim=True) - h * (q * h).mean(1, keepdim=True))
    return {"dx": dx, "dgamma": (dy * h).sum(0), "dbeta": dy.sum(0)}


def _logprob(s):
    x, ids, top = s["logits"], s["ids"], s["case"]["top"]
    m = x.amax(1)
    dead = m == -math.inf                                    # nothing in the row has any probability
    d = x - torch.where(dead, 0.0, m)[:, None]
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    given = torch.gather(d, 1, ids.clamp(0)[:, None])[:, 0] - log_total
    out = {"logprob": torch.where(ids < 0, 0.0, torch.where(dead, -math.inf, given)),
           "entropy": torch.where(dead, 0.0, log_total - torch.where(e > 0, e * d, 0.0).sum(1) / total),
           "logsumexp": m + torch.where(dead, 0.0, log_total)}
    if top:
        # of equal logits the one of the lowest index: a key of the value's order and the index, no two alike
        bits = (x + 0.0).view(torch.int32).to(torch.int64)
        order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
        key = order * (1 << 31) - torch.arange(x.shape[1], device=x.device)
        out["top_ids"] = torch.topk(key, top, 1).indices
        best = torch.gather(d, 1, out["top_ids"]) - log_total[:, None]
        out["top_logprob"] = torch.where(dead[:, None], -math.inf, best)
    return out


def _logprob_grad(s):
    x, ids, lse = s["logits"], s["ids"], s["lse"]
    dead = lse == -math.inf
    g = torch.where((ids < 0) | dead, 0.0, s["g_logprob"])
    l = x - torch.where(dead, 0.0, lse)[:, None]
    p = torch.exp(l)
    if s["g_entropy"] is None:
        d = p * -g[:, None]
    else:
        d = p * (-g[:, None] - s["g_entropy"][:, None] * torch.where(p > 0, l + s["entropy"][:, None], 0.0))
    return d.scatter_add_(1, ids.clamp(0)[:, None], g[:, None])


def _rounded(v):
    return torch.tensor(v, dtype=torch.float32).item()


def _moments(m, v, g):
    """The new moments; every product and every sum is rounded to float32."""
    b1, b2 = _rounded(BETA1), _rounded(BETA2)
    return m * b1 + g * (1 - b1), v * b2 + g * (1 - b2) * g


def _updated(w, m, v, step):
    b1, b2 = _rounded(BETA1), _rounded(BETA2)
    w.mul_(1 - RATE * DECAY).sub_(m / (torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** step)) + ADAM_EPS) * (RATE / (1 - b1 ** step)))


def _adamw32(w, g, m, v, step):
    new_m, new_v = _moments(m, v, g)
    m.copy_(new_m), v.copy_(new_v)
    _updated(w, m, v, step)


def _store8(codes, scales, x, never_zero):
    """x, in rows of a block, as codes and scales; `never_zero`: what is above zero gets the least code at least."""
    largest = x.abs().amax(1)
    scale = torch.where(largest < LEAST, 0.0, largest * INV_MAX)
    q = (x * torch.where(scale > 0, torch.reciprocal(scale), 0.0)[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    if never_zero:
        q = torch.where((x > 0) & (q == 0) & (scale > 0)[:, None], 1, q).to(torch.uint8)
    codes.view(-1).view(torch.uint8).copy_(q.view(-1)[:codes.numel()]), scales.copy_(scale)


def _adamw8(w, g, first, second, first_scales, second_scales, step):
    n = g.numel()
    u = _blocks(second.float()) * second_scales[:, None]
    m, v = _moments(_blocks(first.float()) * first_scales[:, None], u * u, _blocks(g))
    _store8(first, first_scales, m, False), _store8(second, second_scales, torch.sqrt(v), True)
    _updated(w.view(-1), m.view(-1)[:n], v.view(-1)[:n], step)


# ---- one pass

def _builtins():
    global _device_builtins
    if _device_builtins is None:
        from __graft_entry__ import load_package
        load_package()
        from polarai_framework_b200.device_builtins import DeviceBuiltins
        _device_builtins = DeviceBuiltins()
    return _device_builtins


_device_builtins = None


def run(state):
    s, kind = state, state["case"]["kind"]
    if kind == "adamw":
        s["step"] += 1
        lists = [s[k] for k in ("weights", "gradients", "first", "second", "first_scales", "second_scales") if k in s]
        if own:
            _builtins().fadamw(*lists, step=s["step"], lr=RATE, beta1=BETA1, beta2=BETA2, eps=ADAM_EPS, weight_decay=DECAY)
        else:
            one = _adamw8 if s["case"]["bits"] == 8 else _adamw32
            [one(*t, s["step"]) for t in zip(*lists)]
        return s["out"]
    if not own:
        return {"norm": _norm, "norm_grad": _norm_grad, "logprob": _logprob, "logprob_grad": _logprob_grad}[kind](s)
    d = _builtins()
    if kind == "norm":
        d.flayernorm(s["x"], s["gamma"], s["beta"], EPS, s["out"], s["mean"], s["rstd"])
        return {k: s[k] for k in ("out", "mean", "rstd")}
    if kind == "norm_grad":
        d.flayernorm_grad(s["gradient"], s["x"], s["gamma"], s["mean"], s["rstd"], s["dx"], s["dgamma"], s["dbeta"])
        return {k: s[k] for k in ("dx", "dgamma", "dbeta")}
    if kind == "logprob":
        o = s["out"]
        d.flogprob(s["logits"], s["ids"], o["logprob"], o["entropy"], o["logsumexp"], o.get("top_ids"), o.get("top_logprob"))
        return o
    return d.flogprob_grad(s["logits"], s["ids"], s["lse"], s["entropy"], s["g_logprob"], s["g_entropy"], s["dlogits"])


# ---- what a pass cannot do without, and what the definitions give in 64 bits

def work(case):
    kind = case["kind"]
    if kind == "adamw":
        sizes = [math.prod(t) for t in _tensors(case)]
        n, blocks = sum(sizes), sum(-(-t // BLOCK) for t in sizes)
        return {"bytes": 28 * n if case["bits"] == 32 else 16 * n + 16 * blocks, "flops": 14 * n}
    rows = case["rows"]
    if kind in ("norm", "norm_grad"):
        cols = case["cols"]
        if kind == "norm":
            return {"bytes": 8 * rows * cols + 8 * rows + 8 * cols, "flops": 8 * rows * cols}
        return {"bytes": 12 * rows * cols + 8 * rows + 12 * cols, "flops": 16 * rows * cols}
    n = rows * case["classes"]
    if kind == "logprob":
        return {"bytes": 4 * n + (20 + 12 * case["top"]) * rows, "flops": 6 * n}
    return {"bytes": 8 * n + (24 if case["entropy"] else 16) * rows, "flops": 5 * n}


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "adamw":
        return _exact_adamw(s)
    if kind == "norm":
        x = s["x"].double()
        variance, mean = torch.var_mean(x, 1, correction=0)
        inv = (variance + EPS).rsqrt()
        return {"out": torch.addcmul(s["beta"].double(), x.sub_(mean[:, None]).mul_(inv[:, None]), s["gamma"].double()),
                "mean": mean, "rstd": inv}
    if kind == "norm_grad":
        inv, dy = s["rstd"].double(), s["gradient"].double()
        h = (s["x"].double() - s["mean"].double()[:, None]).mul_(inv[:, None])
        gamma, cols = s["gamma"].double(), case["cols"]
        a, b = dy @ gamma / cols, (dy * h) @ gamma / cols
        dgamma, dbeta = torch.einsum("rc,rc->c", dy, h), dy.sum(0)
        dx = (dy.mul_(gamma) - torch.addcmul(a[:, None], h, b[:, None])).mul_(inv[:, None])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    x, ids = s["logits"].double(), s["ids"]
    if kind == "logprob":
        lse = torch.logsumexp(x, 1)
        empty = torch.isneginf(lse)
        l = torch.where(empty[:, None], -math.inf, x - lse[:, None])
        out = {"logprob": torch.where(ids >= 0, l[torch.arange(len(ids), device=x.device), ids.clamp(min=0)], 0.0),
               "entropy": torch.special.entr(l.exp()).sum(1), "logsumexp": lse}
        if case["top"]:
            out["top_ids"] = None
            out["top_logprob"] = torch.topk(l, case["top"], 1).values
        return out
    lse = s["lse"].double()[:, None]
    l = torch.where(torch.isneginf(lse), -math.inf, x.sub_(lse))
    weight = torch.where(ids >= 0, s["g_logprob"].double(), 0.0) * ~torch.isneginf(lse[:, 0])
    p = l.exp()
    dx = -weight[:, None] * p
    if s["g_entropy"] is not None:
        dx += s["g_entropy"].double()[:, None] * (torch.special.entr(p) - p * s["entropy"].double()[:, None])
    at = (torch.arange(len(ids), device=x.device), ids.clamp(min=0))
    dx[at] += weight
    return dx


def _f32(x):
    """A result in 64 bits rounded as the definition of the moments says."""
    return x.float().double()


def _exact_adamw(s):
    b1, b2, t = _rounded(BETA1), _rounded(BETA2), s["step"] + 1
    # every tensor starts a block of its own, so that one pass over the allocation is one over the tensors; what lies between
    # them counts as zeros
    used = torch.zeros_like(s["out"]["weights"], dtype=torch.bool)
    [v.fill_(True) for v in _views(used, s["shapes"])]
    whole = lambda tensors: torch.cat([torch.nn.functional.pad(v.flatten().float(), (0, -v.numel() % BLOCK))  # noqa: E731
                                       for v in tensors]).double()
    g, w, eight = whole(s["gradients"]), s["out"]["weights"].double(), "first_scales" in s
    m, v = whole(s["first"]), whole(s["second"])
    if eight:
        m = _f32(m * s["out"]["first_scales"].double().repeat_interleave(BLOCK))
        v = _f32(_f32(v * s["out"]["second_scales"].double().repeat_interleave(BLOCK)).square())
    # the moments' roundings are part of the definition: codes hang on them
    m = _f32(_f32(m * b1) + _f32(g * (1 - b1)))
    v = _f32(_f32(v * b2) + _f32(_f32(g * (1 - b2)) * g))
    step = RATE / (1 - b1 ** t) * m / (torch.sqrt(v / (1 - b2 ** t)) + ADAM_EPS)
    out = {"weights": torch.where(used, w * (1 - RATE * DECAY) - step, w)}
    if eight:
        out["first"], out["first_scales"] = _exact_codes(m, False)
        out["second"], out["second_scales"] = _exact_codes(_f32(v.sqrt()), True)
        for k in ("first", "second"):
            out[k] = torch.where(used, out[k], s["out"][k].double())
    else:
        out["first"] = torch.where(used, m, s["out"]["first"].double())
        out["second"] = torch.where(used, v, s["out"]["second"].double())
    return out


def _exact_codes(x, never_zero):
    x = x.view(-1, BLOCK)
    top = x.abs().max(1, keepdim=True).values
    scale = _f32(top * INV_MAX) * (top >= LEAST)
    y = torch.nan_to_num(_f32(x * _f32(1 / scale)), 0.0, 0.0, 0.0)
    # to the nearest of e4m3: steps of an eighth of the power of two below, 2^-9 at least; ties to even
    unit = torch.exp2(torch.frexp(y)[1].double().sub(4).clamp(min=-9))
    q = torch.round(y / unit) * unit
    if never_zero:
        q = torch.where((x > 0) & (scale > 0), q.clamp(min=2.0 ** -9), q)
    return q.flatten(), scale.flatten()
