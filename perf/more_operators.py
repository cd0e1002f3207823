"""What ends a training step of a token policy, as cases that can be timed and compared:

  policy      clipped policy loss of sampled tokens with a KL term and an entropy term, and its gradients
  preference  loss of pairs of answers by the ratios of their probabilities to a reference's, and its gradient
  muon        one step of orthogonalised momentum over the matrices of a network

`run` computes them in elementary torch operations or, where `own` is true, with the builtins of this package.
All tensors are float32 but ids and offsets (int64, or int32 in some cases).  Sequences lie behind one another: sequence s has the tokens
[offsets[s], offsets[s + 1]); an id below zero marks a token that does not count (a prompt's, or padding).
"""
import math

import torch

own = False

DEVICE = "cuda:0"
CLIP_LOW, CLIP_HIGH, KL, ENTROPY = 0.2, 0.28, 0.04, 0.003
BETA = 0.1                                # of the preference loss
RATE, MOMENTUM, DECAY, STEPS = 0.02, 0.95, 0.1, 5
A, B, C = 3.4445, -4.7750, 2.0315         # of the orthogonalisation's polynomial


def listed():
    return [
        # a few short answers, as an online learner's smallest update has
        {"name": "policy_few", "kind": "policy", "tokens": 600, "sequences": 5, "behind": 0, "reference": True, "entropy": True,
         "by_sequence": False, "advantage": "sequence", "gradient": True, "bits": 64},
        # a batch of sampled answers, each answer of the same weight
        {"name": "policy_batch", "kind": "policy", "tokens": 131072, "sequences": 256, "behind": 0, "reference": True, "entropy": True,
         "by_sequence": True, "advantage": "sequence", "gradient": True, "bits": 64},
        # the loss alone on an odd, partly padded batch with an advantage per token
        {"name": "policy_ragged", "kind": "policy", "tokens": 77777, "sequences": 1001, "behind": 501, "reference": False, "entropy": False,
         "by_sequence": False, "advantage": "token", "gradient": False, "bits": 32},
        # all answers of a large sampling round at once
        {"name": "policy_large", "kind": "policy", "tokens": 8388608, "sequences": 4096, "behind": 0, "reference": True, "entropy": False,
         "by_sequence": False, "advantage": "token", "gradient": True, "bits": 64},
        # four pairs of answers
        {"name": "preference_few", "kind": "preference", "tokens": 1500, "pairs": 4, "behind": 0, "reference": True, "average": False, "smoothing": 0.0,
         "margin": 0.0, "gradient": True, "bits": 64},
        # a batch of pairs with uncertain labels
        {"name": "preference_batch", "kind": "preference", "tokens": 400001, "pairs": 300, "behind": 77, "reference": True, "average": False,
         "smoothing": 0.1, "margin": 0.0, "gradient": True, "bits": 64},
        # pairs of long answers without a reference, by the mean over their tokens
        {"name": "preference_long", "kind": "preference", "tokens": 4194304, "pairs": 64, "behind": 0, "reference": False, "average": True,
         "smoothing": 0.0, "margin": 0.05, "gradient": True, "bits": 32},
        # the two matrices of the benchmark's network
        {"name": "muon_mlp", "kind": "muon", "shapes": "784x4096 4096x10", "count": 1},
        # many small matrices
        {"name": "muon_small", "kind": "muon", "shapes": "64x64 64x128 128x64", "count": 12},
        # matrices that are multiples of nothing, wide and tall ones
        {"name": "muon_ragged", "kind": "muon", "shapes": "301x514 999x301 1511x777", "count": 2},
        # a token model's layers
        {"name": "muon_layers", "kind": "muon", "shapes": "1024x1024 1024x1024 1024x1024 1024x1024 1024x4096 4096x1024", "count": 16},
        # one large projection
        {"name": "muon_wide", "kind": "muon", "shapes": "4096x16384", "count": 1},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _size(rng, lo, hi):
    """Half of them multiples of 16, as widths usually are, half as they come."""
    v = _log(rng, lo, hi)
    return min(hi, max(16, (v + 8) // 16 * 16)) if rng.random() < 0.5 else v


def draw(rng):
    kind = rng.choice(["policy", "preference", "muon"])
    flag = lambda: rng.random() < 0.5  # noqa: E731
    if kind == "policy":
        tokens = _log(rng, 1, 1 << 23)
        return {"kind": kind, "tokens": tokens, "sequences": _log(rng, 1, max(1, min(tokens, 65536))), "behind": rng.choice([0, tokens // 16]),
                "reference": flag(), "entropy": flag(), "by_sequence": flag(), "advantage": rng.choice(["token", "sequence"]),
                "gradient": rng.random() < 0.75, "bits": rng.choice([32, 64])}
    if kind == "preference":
        tokens = _log(rng, 2, 1 << 22)
        return {"kind": kind, "tokens": tokens, "pairs": _log(rng, 1, max(1, min(tokens // 2, 16384))), "behind": rng.choice([0, tokens // 16]),
                "reference": flag(), "average": flag(), "smoothing": rng.choice([0.0, 0.1]), "margin": rng.choice([0.0, 0.05]),
                "gradient": rng.random() < 0.75, "bits": rng.choice([32, 64])}
    if rng.random() < 0.5:                                   # a network's matrices
        w, i, layers = _size(rng, 16, 1024), _size(rng, 32, 4096), rng.randint(1, 16)
        return {"kind": kind, "shapes": f"{w}x{w} {w}x{i} {i}x{w}", "count": layers}
    return {"kind": kind, "shapes": f"{_size(rng, 1, 4096)}x{_size(rng, 1, 16384)}", "count": 1}


def _shapes(case):
    """The matrices of a step, layer by layer."""
    return [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split()] * case["count"]


def _views(flat, shapes):
    """A network's matrices in one allocation, each on a boundary of 128 values, as memory pools place them."""
    at = [0]
    for t in shapes:
        at.append(at[-1] + -(-math.prod(t) // 128) * 128)
    return [flat[a:a + math.prod(t)].view(t) for a, t in zip(at, shapes)]


# ---- inputs

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(g, *shape, scale=1.0, mean=0.0):
    return torch.empty(shape, device=DEVICE).normal_(mean, scale, generator=g)


def _sequences(g, tokens, sequences, behind, bits):
    """Offsets of sequences of random lengths, some of them empty, in all tokens but the last `behind`, and ids: a sequence's first third
    does not count, nor does anything of every seventh sequence."""
    used = tokens - behind
    cuts = torch.randint(0, used + 1, (max(sequences - 1, 0),), device=DEVICE, generator=g).sort().values
    if sequences > 8:
        cuts[sequences // 2] = cuts[sequences // 2 - 1]      # (an empty one at least)
    ends = torch.tensor([0, used], device=DEVICE)
    offsets = torch.cat([ends[:1], cuts, ends[1:]])
    at = torch.arange(tokens, device=DEVICE)
    s = torch.searchsorted(offsets, at, right=True).sub_(1).clamp_(0, sequences - 1)
    ids = torch.randint(0, 32000, (tokens,), device=DEVICE, generator=g)
    ids[(at - offsets[s]) * 3 < offsets[s + 1] - offsets[s] - 2] = -1
    ids[(s % 7 == 6) | (at >= used)] = -1
    dtype = torch.int64 if bits == 64 else torch.int32
    return ids.to(dtype), offsets.to(dtype)


def prepare(case, seed):
    g, kind = _generator(seed), case["kind"]
    s = {"case": case}
    if kind == "muon":
        shapes = _shapes(case)
        total = sum(-(-math.prod(t) // 128) * 128 for t in shapes)
        flat = [_normal(g, total, scale=a) for a in (0.02, 0.5, 0.5)]
        s["weights"], s["gradients"], s["momenta"] = (_views(f, shapes) for f in flat)
        s["out"] = {"weights": flat[0], "momenta": flat[2]}
        for g1, m1 in zip(s["gradients"], s["momenta"]):
            # gradients as they are met: a few directions stand out of the rest
            rank = min(8, *g1.shape)
            few = _normal(g, g1.shape[0], rank) * torch.logspace(0, -1, rank, device=DEVICE) @ _normal(g, rank, g1.shape[1])
            g1.add_(few), m1.add_(few)
        flat[1].mul_(1e-3), flat[2].mul_(8e-3)
        return s
    tokens = case["tokens"]
    sequences = case["sequences"] if kind == "policy" else 2 * case["pairs"]
    s["ids"], s["offsets"] = _sequences(g, tokens, sequences, case["behind"], case["bits"])
    counts = s["ids"] >= 0
    s["logprob"] = -_normal(g, tokens).abs_().mul_(1.5)
    s["logprob"][~counts] = 0.0                              # as log probabilities of rows without an id are held
    s["reference"] = s["logprob"] + _normal(g, tokens, scale=0.1) if case["reference"] else None
    if case["gradient"]:
        s["g_logprob"] = torch.zeros(tokens, device=DEVICE)
    if kind == "preference":
        s["loss"], s["rewards"] = torch.empty(3, device=DEVICE), torch.empty(sequences, device=DEVICE)
        return s
    s["old"] = s["logprob"] + _normal(g, tokens, scale=0.15)
    s["advantage"] = _normal(g, tokens if case["advantage"] == "token" else sequences, mean=0.2)
    s["entropy"] = _normal(g, tokens).abs_() if case["entropy"] else None
    s["loss"] = torch.empty(5, device=DEVICE)
    if case["gradient"] and case["entropy"]:
        s["g_entropy"] = torch.zeros(tokens, device=DEVICE)
    # a token that does not count may hold anything
    s["old"][~counts & (torch.rand(tokens, device=DEVICE, generator=g) < 0.01)] = -math.inf
    return s


# ---- the plain forms, in 32 bits

def _where(s, sequences):
    """The sequence of each token, whether the token counts, and whether it is part of a sequence at all."""
    offsets = s["offsets"].to(torch.int64)
    at = torch.arange(len(s["ids"]), device=DEVICE)
    inside = (at >= offsets[0]) & (at < offsets[-1])
    q = (torch.searchsorted(offsets, at, right=True) - 1).clamp(0, sequences - 1)
    return q, inside & (s["ids"] >= 0), inside


def _policy(s):
    c = s["case"]
    q, counts, inside = _where(s, c["sequences"])
    zero = torch.zeros((), device=DEVICE)
    if c["by_sequence"]:
        per = torch.zeros(c["sequences"], device=DEVICE, dtype=torch.int64).index_add_(0, q, counts.to(torch.int64))
        weight = (1 / (per[q].to(torch.float32) * (per > 0).sum()))
    else:
        weight = 1 / counts.sum().to(torch.float32)
    weight = torch.where(counts, weight, zero)
    lp, old = torch.where(counts, s["logprob"], zero), torch.where(counts, s["old"], zero)
    advantage = s["advantage"] if c["advantage"] == "token" else s["advantage"][q]
    # which side of the clipping border a token is on: in 64 bits
    d = lp.double() - old.double()
    high, low = d > math.log1p(_rounded(CLIP_HIGH)), d < math.log1p(-_rounded(CLIP_LOW))
    clipped = ((advantage > 0) & high) | ((advantage < 0) & low)
    ratio = torch.exp(lp - old)
    bound = torch.where(high, 1 + CLIP_HIGH, 1 - CLIP_LOW)
    surrogate = torch.where(clipped, bound, ratio) * advantage
    out = {}
    g = torch.where(clipped, zero, -ratio * advantage)
    terms = [surrogate * weight]
    if s["reference"] is not None:
        r = torch.where(counts, s["reference"], zero).double() - lp.double()
        e = torch.expm1(r)
        terms.append((e - r).float() * weight)               # exp(r) - 1 - r, of which 32 bits lose the most where r is small
        g = g - KL * e.float()
    else:
        terms.append(zero)
    terms.append(torch.where(counts, s["entropy"], zero) * weight if s["entropy"] is not None else zero)
    terms.append(torch.where(clipped & counts, weight, zero))
    sums = [t.sum(dtype=torch.float64) for t in terms]
    loss = -sums[0] + KL * sums[1] - (ENTROPY * sums[2] if c["entropy"] else 0)
    out["loss"] = torch.stack([loss, *sums]).float()
    if c["gradient"]:
        out["g_logprob"] = torch.where(inside, torch.where(counts, g * weight, zero), s["g_logprob"])
        if c["entropy"]:
            out["g_entropy"] = torch.where(inside, -ENTROPY * weight, s["g_entropy"])
    return out


def _preference(s):
    c = s["case"]
    n = 2 * c["pairs"]
    q, counts, inside = _where(s, n)
    d = s["logprob"].double() - (s["reference"].double() if c["reference"] else 0)
    sums = torch.zeros(n, device=DEVICE, dtype=torch.float64).index_add_(0, q, torch.where(counts, d, 0.0))
    share = torch.ones(n, device=DEVICE)
    if c["average"]:
        per = torch.zeros(n, device=DEVICE, dtype=torch.int64).index_add_(0, q, counts.to(torch.int64))
        share = 1 / per.clamp(min=1).float()
        sums = sums / per.clamp(min=1)
    rewards = (BETA * sums).float()
    gap = (BETA * (sums[0::2] - sums[1::2])).float()         # (long sums that nearly cancel)
    z = gap - c["margin"]
    # -log(sigmoid(z)) and -log(sigmoid(-z))
    more = torch.log1p(torch.exp(-z.abs()))
    right, wrong = more + (-z).clamp(min=0), more + z.clamp(min=0)
    e = c["smoothing"]
    loss = (1 - e) * right + e * wrong
    out = {"loss": torch.stack([loss.sum(), (gap > 0).sum().float(), gap.sum()]) / c["pairs"], "rewards": rewards}
    if c["gradient"]:
        p = 1 / (1 + torch.exp(-z))
        dz = (e * p - (1 - e) * (1 / (1 + torch.exp(z)))) * (BETA / c["pairs"])
        per_sequence = torch.stack([dz, -dz], 1).view(-1) * share
        out["g_logprob"] = torch.where(inside, torch.where(counts, per_sequence[q], 0.0), s["g_logprob"])
    return out


def _rounded(v):
    return torch.tensor(v, dtype=torch.float32).item()


def _muon(s):
    for w, g, m in zip(s["weights"], s["gradients"], s["momenta"]):
        rows, cols = w.shape
        m.mul_(MOMENTUM).add_(g)
        u = g + MOMENTUM * m
        x = u / torch.sqrt((u.double() * u.double()).sum()).float()
        x = x.T if rows > cols else x
        for _ in range(STEPS):
            a = x @ x.T
            x = A * x + (B * a + C * (a @ a)) @ x
        x = x.T if rows > cols else x
        w.mul_(1 - RATE * DECAY).sub_(x * (RATE * math.sqrt(max(1.0, rows / cols))))
    return s["out"]


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
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        return {"policy": _policy, "preference": _preference, "muon": _muon}[kind](s)
    d = _builtins()
    if kind == "muon":
        d.fmuon(s["weights"], s["gradients"], s["momenta"], lr=RATE, momentum=MOMENTUM, nesterov=True, weight_decay=DECAY, steps=STEPS)
        return s["out"]
    if kind == "policy":
        d.fpolicy_loss(s["logprob"], s["old"], s["advantage"], s["ids"], s["offsets"], s["loss"], s.get("g_logprob"), s.get("g_entropy"),
                       reference=s["reference"], entropy=s["entropy"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_weight=KL,
                       entropy_weight=ENTROPY, by_sequence=c["by_sequence"], advantage_per_token=c["advantage"] == "token")
        return {k: s[k] for k in ("loss", "g_logprob", "g_entropy") if k in s}
    d.fpreference_loss(s["logprob"], s["ids"], s["offsets"], s["loss"], s["rewards"], s.get("g_logprob"), reference=s["reference"], beta=BETA,
                       smoothing=c["smoothing"], margin=c["margin"], average=c["average"])
    return {k: s[k] for k in ("loss", "rewards", "g_logprob") if k in s}


# ---- what a pass cannot do without, and what the definitions give in 64 bits

def work(case):
    kind = case["kind"]
    if kind == "muon":
        size = flops = 0
        for rows, cols in _shapes(case):
            small, n = min(rows, cols), rows * cols
            size += n
            # per round: two symmetric products, of which one half is computed, and the product with the matrix
            flops += STEPS * (n * small + small ** 3 + 2 * n * small)
        return {"bytes": 20 * size, "flops": flops}
    n, word = case["tokens"], case["bits"] // 8
    used = n - case["behind"]
    if kind == "policy":
        per = 8 + word + 4 * (case["reference"] + case["entropy"] + (case["advantage"] == "token"))
        per += 4 * case["gradient"] * (1 + case["entropy"])
        return {"bytes": per * used + (word + 4 * (case["advantage"] == "sequence")) * case["sequences"] + 20, "flops": 30 * used}
    per = 4 + word + 4 * case["reference"] + 4 * case["gradient"]
    return {"bytes": per * used + (word + 4) * 2 * case["pairs"] + 12, "flops": 4 * used}


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "muon":
        return _exact_muon(s)
    lengths = s["offsets"].diff().long()
    used, n = case["tokens"] - case["behind"], len(lengths)
    of = torch.repeat_interleave(torch.arange(n, device=DEVICE), lengths)
    live = s["ids"][:used] >= 0
    at, of = live.nonzero()[:, 0], of[live]
    per = torch.bincount(of, minlength=n).double()
    lp = s["logprob"][at].double()
    ref = s["reference"][at].double() if case["reference"] else None

    def spread(values, name):
        g = s[name].double()
        g[:used] = 0
        g[at] = values
        return g

    if kind == "preference":
        ratio = lp - ref if ref is not None else lp
        total = torch.bincount(of, weights=ratio, minlength=n)
        share = 1 / per.clamp(min=1) if case["average"] else torch.ones_like(per)
        rewards = _rounded(BETA) * total * share
        gap = rewards.view(-1, 2)[:, 0] - rewards.view(-1, 2)[:, 1]
        z, e, p = gap - _rounded(case["margin"]), _rounded(case["smoothing"]), case["pairs"]
        softplus = torch.nn.functional.softplus
        loss = (1 - e) * softplus(-z, threshold=1e4) + e * softplus(z, threshold=1e4)
        out = {"loss": torch.stack([loss.mean(), (gap > 0).double().mean(), gap.mean()]), "rewards": rewards}
        if case["gradient"]:
            slope = (e * torch.sigmoid(z) - (1 - e) * torch.sigmoid(-z)) * _rounded(BETA) / p
            out["g_logprob"] = spread((torch.stack([slope, -slope], 1).flatten() * share)[of], "g_logprob")
        return out
    weight = 1 / (per * (per > 0).sum())[of] if case["by_sequence"] else torch.full_like(lp, 1 / max(len(at), 1))
    advantage = s["advantage"].double()
    advantage = advantage[at] if case["advantage"] == "token" else advantage[of]
    d = lp - s["old"][at].double()
    low, high = 1 - _rounded(CLIP_LOW), 1 + _rounded(CLIP_HIGH)
    ratio = d.exp()
    held = d.clamp(math.log(low), math.log(high))
    free, bound = ratio * advantage, torch.where(held == d, ratio, held.exp()) * advantage
    cut = bound < free
    parts = [(torch.minimum(free, bound) * weight).sum()]
    slope = torch.where(cut, 0.0, -free)
    if ref is not None:
        r = ref - lp
        parts.append(((torch.expm1(r) - r) * weight).sum())
        slope = slope - _rounded(KL) * torch.expm1(r)
    else:
        parts.append(torch.zeros_like(parts[0]))
    parts.append((s["entropy"][at].double() * weight).sum() if case["entropy"] else torch.zeros_like(parts[0]))
    parts.append((weight * cut).sum())
    loss = _rounded(KL) * parts[1] - parts[0] - _rounded(ENTROPY) * parts[2]
    out = {"loss": torch.stack([loss, *parts])}
    if case["gradient"]:
        out["g_logprob"] = spread(slope * weight, "g_logprob")
        if case["entropy"]:
            out["g_entropy"] = spread(-_rounded(ENTROPY) * weight, "g_entropy")
    return out


def _exact_muon(s):
    mu, a, b, c = (_rounded(v) for v in (MOMENTUM, A, B, C))
    out = {k: v.double() for k, v in s["out"].items()}       # what lies between the matrices stays as it is
    shapes = [t.shape for t in s["weights"]]
    for w, g, m in zip(_views(out["weights"], shapes), s["gradients"], _views(out["momenta"], shapes)):
        m.mul_(mu).add_(g)
        x = g.double() + mu * m
        x = x / torch.linalg.norm(x)
        tall = x.shape[0] > x.shape[1]
        for _ in range(STEPS):
            # the polynomial of the Gram matrix of the shorter side, by Horner's rule
            gram = x.mT @ x if tall else x @ x.mT
            p = gram @ (b * torch.eye(len(gram), dtype=x.dtype, device=x.device) + c * gram)
            x = a * x + (x @ p if tall else p @ x)
        scale = math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
        w.mul_(1 - _rounded(RATE) * _rounded(DECAY)).sub_(_rounded(RATE) * _rounded(scale) * x)
    return out
