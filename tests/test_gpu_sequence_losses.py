"""The policy loss and the loss of pairs, with their gradients, against the formulas in 64 bits."""
import math

import numpy as np
import pytest

import __graft_entry__ as ge

ge.load_package()
import torch  # noqa: E402
from oracle import rows_oracle as rows  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24                                               # half a step of fp32, relative


@pytest.fixture(scope="module")
def d():
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return DeviceBuiltins()


def offsets_of(rng, tokens, sequences, before=0, behind=0):
    cuts = np.sort(rng.integers(before, tokens - behind + 1, max(sequences - 1, 0)))
    return np.concatenate([[before], cuts, [tokens - behind]]).astype(np.int64)


def batch(seed, tokens, sequences, before=0, behind=0, counted=0.7, empty_rows=True):
    rng = np.random.default_rng(seed)
    f = np.float32
    o = offsets_of(rng, tokens, sequences, before, behind)
    ids = rng.integers(0, 1000, tokens)
    ids[rng.random(tokens) >= counted] = -1
    if empty_rows:                                           # every fifth sequence has no token that counts
        of = np.clip(np.searchsorted(o, np.arange(tokens), side="right") - 1, 0, max(sequences - 1, 0))
        ids[of % 5 == 4] = -1
    lp = (-np.abs(rng.standard_normal(tokens)) * 2).astype(f)
    return {"logprob": lp, "old": (lp + 0.3 * rng.standard_normal(tokens)).astype(f), "reference": (lp + 0.3 * rng.standard_normal(tokens)).astype(f),
            "entropy": np.abs(rng.standard_normal(tokens)).astype(f), "token_advantage": rng.standard_normal(tokens).astype(f),
            "advantage": rng.standard_normal(max(sequences, 1)).astype(f)[:sequences], "ids": ids, "offsets": o}


def up(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0", dtype)


ID = {"f32": torch.float32, "i32": torch.int32, "i64": torch.int64}


def policy(d, b, kind="i64", reference=True, entropy=True, per_token=True, by_sequence=False, gradient=True, count=0.0, shift=0, **o):
    """The device's (loss, g_logprob, g_entropy) and the oracle's with its sizes; `shift`: how many floats the arrays lie off 16 bytes."""
    def placed(a):
        t = torch.empty(len(a) + 4, device="cuda:0")[shift:shift + len(a)]
        return t.copy_(up(a))
    n = len(b["ids"])
    opts = dict(clip_low=0.2, clip_high=0.25, kl_weight=0.1, entropy_weight=0.01)
    opts.update(o)
    a = b["token_advantage"] if per_token else b["advantage"]
    loss = torch.full((5,), math.nan, device="cuda:0")
    g, ge_ = (placed(np.full(n, 7.0, np.float32)) for _ in range(2))
    d.fpolicy_loss(placed(b["logprob"]), placed(b["old"]), placed(a), up(b["ids"], ID[kind]), up(b["offsets"], ID[kind]), loss,
                   g if gradient else None, ge_ if gradient and entropy else None, reference=placed(b["reference"]) if reference else None,
                   entropy=placed(b["entropy"]) if entropy else None, by_sequence=by_sequence, advantage_per_token=per_token, count=count, **opts)
    want = rows.policy_loss64(b["logprob"], b["old"], b["reference"] if reference else None, b["entropy"] if entropy else None, a, b["ids"], b["offsets"],
                              opts["clip_low"], opts["clip_high"], opts["kl_weight"], opts["entropy_weight"], by_sequence, per_token, count)
    return loss.cpu().numpy(), g.cpu().numpy(), ge_.cpu().numpy(), want


def check(got, gradient=True, entropy=True):
    loss, g, ge_, (want, wg, wge, (size, token)) = got
    # a sum: each term has some eight roundings (exponential 2 ulp, its argument, products), and passes through some twenty additions
    assert (np.abs(loss - want) <= 32 * U * size + 1e-44).all(), (loss, want)
    inside = ~np.isnan(wg)
    if gradient:
        # a token: the exponential's two steps and its argument's, the series' few, four products, the weight's two divisions
        assert (np.abs(g - wg)[inside] <= 16 * U * token[inside] + 1e-44).all()
        assert (g[~inside] == 7).all()
    if gradient and entropy:
        assert (np.abs(ge_ - wge)[inside] <= 4 * U * np.abs(wge[inside])).all() and (ge_[~inside] == 7).all()
    if not gradient:
        assert (g == 7).all()


# one CTA: up to 4096 tokens (pairs: 6144) of 2048 sequences; beyond, tiles of 2048 tokens
SIZES = [(1, 1), (2, 1), (3, 7), (31, 2), (33, 5), (1000, 1), (1025, 40), (4095, 2000), (8191, 2048), (8192, 1), (8193, 3), (8192, 2049), (5000, 6000),
         (12289, 1), (20000, 19), (65537, 4000), (100001, 99999), (300007, 2)]


@pytest.mark.parametrize("by_sequence", [False, True])
@pytest.mark.parametrize("tokens,sequences", SIZES)
def test_policy_sizes(d, tokens, sequences, by_sequence):
    for per_token in (False, True):
        check(policy(d, batch(tokens + sequences, tokens, sequences), per_token=per_token, by_sequence=by_sequence))


@pytest.mark.parametrize("tokens,sequences", [(700, 9), (30001, 50)])
@pytest.mark.parametrize("kind", ["f32", "i32", "i64"])
@pytest.mark.parametrize("shift", [0, 1])
def test_policy_id_types_and_alignment(d, kind, shift, tokens, sequences):
    check(policy(d, batch(5, tokens, sequences, before=37, behind=41), kind=kind, shift=shift, per_token=False, by_sequence=True))


@pytest.mark.parametrize("tokens,sequences", [(500, 7), (20011, 33)])
@pytest.mark.parametrize("reference,entropy,gradient", [(False, False, True), (True, False, True), (False, True, True), (True, True, False), (False, False, False)])
def test_policy_parts_left_out(d, reference, entropy, gradient, tokens, sequences):
    check(policy(d, batch(6, tokens, sequences), reference=reference, entropy=entropy, gradient=gradient), gradient, entropy)


@pytest.mark.parametrize("tokens,sequences", [(300, 6), (9000, 20)])
@pytest.mark.parametrize("by_sequence", [False, True])
def test_policy_count_of_a_larger_batch(d, by_sequence, tokens, sequences):
    check(policy(d, batch(7, tokens, sequences), by_sequence=by_sequence, count=12345.0))


@pytest.mark.parametrize("tokens,sequences", [(64, 4), (10000, 4)])
@pytest.mark.parametrize("by_sequence", [False, True])
def test_policy_nothing_counts(d, by_sequence, tokens, sequences):
    b = batch(8, tokens, sequences, before=3, behind=5)
    b["ids"][:] = -1
    for t in ("logprob", "old", "reference", "entropy", "token_advantage"):
        b[t][:] = np.nan
    loss, g, ge_, _ = policy(d, b, by_sequence=by_sequence)
    assert (loss == 0).all() and (g[3:-5] == 0).all() and (ge_[3:-5] == 0).all() and (g[:3] == 7).all() and (g[-5:] == 7).all()


@pytest.mark.parametrize("tokens", [400, 12000])
def test_policy_masked_places_hold_anything(d, tokens):
    b = batch(9, tokens, 11)
    out = b["ids"] < 0
    for t, v in (("logprob", np.nan), ("old", -np.inf), ("reference", np.inf), ("entropy", np.nan), ("token_advantage", -np.inf)):
        b[t][out] = v
    for by_sequence in (False, True):
        check(policy(d, b, by_sequence=by_sequence))


@pytest.mark.parametrize("tokens", [50, 9000])
def test_policy_no_sequences_and_no_tokens(d, tokens):
    b = batch(10, tokens, 1)
    b["offsets"], b["advantage"] = np.array([0]), np.zeros(0, np.float32)
    loss, g, ge_, _ = policy(d, {**b}, per_token=True)
    assert (loss == 0).all() and (g == 7).all()
    empty = batch(11, 0, 3)
    loss, *_ = policy(d, empty, per_token=False)
    assert (loss == 0).all()


@pytest.mark.parametrize("tokens", [512, 16384])
def test_policy_on_the_clipping_border(d, tokens):
    # ratios within a few steps of fp32 of the borders, on both sides: d is decided in 64 bits, as the oracle's
    rng = np.random.default_rng(12)
    b = batch(12, tokens, 4, counted=1.0, empty_rows=False)
    border = np.where(rng.random(tokens) < 0.5, np.log1p(np.float64(np.float32(0.25))), np.log1p(-np.float64(np.float32(0.2))))
    b["logprob"][:] = 0
    old = (-border).astype(np.float32)
    for _ in range(3):
        old = np.where(rng.random(tokens) < 0.5, np.nextafter(old, np.float32(9)), np.where(rng.random(tokens) < 0.5, np.nextafter(old, np.float32(-9)), old))
    b["old"] = old.astype(np.float32)
    got = policy(d, b)
    check(got)
    # beyond the border by a step up with probability 1/2 and that at least in part, clipped there for one sign of the advantage: about
    # 1/2 * 1/2, less what three steps bring back
    assert 0.05 < got[0][4] < 0.45


@pytest.mark.parametrize("tokens", [100, 10000])
def test_policy_far_ratios_and_close_references(d, tokens):
    b = batch(13, tokens, 3, counted=1.0, empty_rows=False)
    b["old"][::2] = b["logprob"][::2] - 60                   # e^60 ratios: clipped where the advantage is above zero
    b["token_advantage"] = np.abs(b["token_advantage"])
    rng = np.random.default_rng(14)
    q = (10.0 ** rng.uniform(-6, 1, tokens) * rng.choice([-1, 1], tokens))
    b["reference"] = (b["logprob"] + q).astype(np.float32)
    check(policy(d, b))
    check(policy(d, b, clip_high=float("inf"), clip_low=1.0))


def test_policy_zero_advantage_has_no_gradient_of_its_own(d):
    b = batch(15, 300, 3)
    b["token_advantage"][:] = 0
    loss, g, *_ = policy(d, b, reference=False)
    assert (g == 0).all() and loss[1] == 0 and loss[4] == 0


def test_policy_long_runs_of_empty_sequences(d):
    # 40000 empty ones in the middle of a tile, 300 of one token, then a long one
    b = batch(16, 30000, 1, counted=0.8, empty_rows=False)
    b["offsets"] = np.concatenate([[0, 100], np.full(40000, 5000), 5000 + np.arange(1, 301), [30000]])
    n = len(b["offsets"]) - 1
    b["advantage"] = np.random.default_rng(16).standard_normal(n).astype(np.float32)
    for by_sequence in (False, True):
        check(policy(d, b, per_token=False, by_sequence=by_sequence))


@pytest.mark.parametrize("tokens", [400, 20000])
def test_policy_gradient_in_the_place_of_an_input(d, tokens):
    b = batch(17, tokens, 9)
    t = {k: up(v) for k, v in b.items()}
    loss, g, ge_ = (torch.empty(n, device="cuda:0") for n in (5, tokens, tokens))
    call = lambda lp, old, h, g, ge_: d.fpolicy_loss(lp, old, t["token_advantage"], t["ids"], t["offsets"], loss, g, ge_, reference=t["reference"],  # noqa: E731
                                                      entropy=h, advantage_per_token=True, kl_weight=0.1, entropy_weight=0.1)
    call(t["logprob"], t["old"], t["entropy"], g, ge_)
    first = loss.clone()
    lp, h = t["logprob"].clone(), t["entropy"].clone()
    call(lp, t["old"], h, lp, h)
    assert torch.equal(lp, g) and torch.equal(h, ge_) and torch.equal(first, loss)


def test_policy_same_bits_each_time_and_beside_another_stream(d):
    b = batch(18, 200003, 700)
    first = policy(d, b, by_sequence=True, per_token=False)[:3]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    again = []
    for s in streams:
        with torch.cuda.stream(s):
            again.append(policy(d, b, by_sequence=True, per_token=False)[:3])
    assert all(np.array_equal(x, y) for r in again for x, y in zip(first, r))


@pytest.mark.parametrize("tokens,sequences", [(900, 10), (50000, 60)])
def test_losses_captured_and_replayed(d, tokens, sequences):
    b = batch(19, tokens, sequences)
    t = {k: up(v) for k, v in b.items()}
    out = [torch.zeros(n, device="cuda:0") for n in (5, tokens, tokens, 3, sequences, tokens)]

    def step():
        d.fpolicy_loss(t["logprob"], t["old"], t["advantage"], t["ids"], t["offsets"], out[0], out[1], out[2], reference=t["reference"],
                       entropy=t["entropy"], kl_weight=0.1, entropy_weight=0.01, by_sequence=True)
        d.fpreference_loss(t["logprob"], t["ids"], t["offsets"], out[3], out[4], out[5], reference=t["reference"], average=True)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    other = batch(20, tokens, sequences)
    for k in t:
        t[k].copy_(up(other[k]))
    graph.replay()
    torch.cuda.synchronize()
    replayed = [o.clone() for o in out]
    [o.zero_() for o in out]
    step()
    assert all(torch.equal(a, b) for a, b in zip(out, replayed))


def test_bad_offsets_stay_inside_the_arrays(d):
    # no results are promised; every access is cut off at the arrays' ends
    for tokens, sequences in ((500, 20), (30000, 50), (30000, 3000)):
        b = batch(21, tokens, sequences)
        rng = np.random.default_rng(21)
        for o in (rng.integers(-5, 3 * tokens, sequences + 1), b["offsets"][::-1].copy(), np.full(sequences + 1, -1), np.full(sequences + 1, 1 << 40)):
            c = {**b, "offsets": o}
            t = {k: up(v) for k, v in c.items()}
            g = torch.empty(tokens, device="cuda:0")
            for by_sequence in (False, True):
                d.fpolicy_loss(t["logprob"], t["old"], t["advantage"], t["ids"], t["offsets"], torch.empty(5, device="cuda:0"), g, by_sequence=by_sequence)
            n = sequences // 2 * 2 + 1
            d.fpreference_loss(t["logprob"], t["ids"], t["offsets"][:n].clone(), torch.empty(3, device="cuda:0"), None, g)
    torch.cuda.synchronize()


# ---- pairs

def preference(d, b, kind="i64", reference=True, gradient=True, rewards=True, count=0.0, shift=0, beta=0.1, smoothing=0.0, margin=0.0, average=False):
    def placed(a):
        t = torch.empty(len(a) + 4, device="cuda:0")[shift:shift + len(a)]
        return t.copy_(up(a))
    n, sequences = len(b["ids"]), len(b["offsets"]) - 1
    loss, r = torch.full((3,), math.nan, device="cuda:0"), torch.full((sequences,), math.nan, device="cuda:0")
    g = placed(np.full(n, 7.0, np.float32))
    d.fpreference_loss(placed(b["logprob"]), up(b["ids"], ID[kind]), up(b["offsets"], ID[kind]), loss, r if rewards else None, g if gradient else None,
                       reference=placed(b["reference"]) if reference else None, beta=beta, smoothing=smoothing, margin=margin, average=average, count=count)
    want, wr, wg, z = rows.preference_loss64(b["logprob"], b["reference"] if reference else None, b["ids"], b["offsets"], beta, smoothing, margin, average, count)
    loss, r, g = loss.cpu().numpy(), r.cpu().numpy(), g.cpu().numpy()
    # a pair's loss: z is rounded once (the loss's slope is 1 at most), then some eight operations; then sums of some twenty additions
    each = np.maximum(np.logaddexp(0, -z), np.logaddexp(0, z)) + np.abs(z)
    units = count if count > 0 else max(len(z), 1)
    assert abs(loss[0] - want[0]) <= 32 * U * each.sum() / units and abs(loss[1] - want[1]) <= 4 * U
    assert abs(loss[2] - want[2]) <= 32 * U * np.abs(z + margin).sum() / units + 1e-44
    if rewards:
        assert (np.abs(r - wr) <= 2 * U * np.abs(wr) + 1e-44).all()
    inside = ~np.isnan(wg)
    if gradient:
        # the sigmoid's relative error: z's rounding times its derivative (|z| at most) and eight operations; with smoothing two parts of
        # opposite sign, 1 together
        part = np.repeat(np.abs(z), 2)[np.repeat(np.arange(sequences), np.diff(b["offsets"]))] if sequences else np.zeros(0)
        whole = np.abs(wg[inside]) if smoothing == 0 else np.where(wg[inside] != 0, beta / units, 0.0)
        assert (np.abs(g - wg)[inside] <= (16 + part) * U * whole + 1e-44).all()
        assert (g[~inside] == 7).all()
    else:
        assert (g == 7).all()
    return loss


PAIRS = [(2, 1), (3, 4), (64, 1), (777, 3), (1500, 4), (8191, 1024), (8192, 1), (8193, 1), (4097, 1030), (9000, 2000), (40961, 5), (100003, 333), (262144, 1),
         (60000, 30000)]


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("tokens,pairs", PAIRS)
def test_pairs_sizes(d, tokens, pairs, average):
    preference(d, batch(tokens + pairs, tokens, 2 * pairs), average=average)


@pytest.mark.parametrize("tokens,pairs", [(600, 5), (50000, 40)])
@pytest.mark.parametrize("kind", ["f32", "i32", "i64"])
@pytest.mark.parametrize("shift", [0, 3])
def test_pairs_id_types_alignment_and_what_lies_around(d, kind, shift, tokens, pairs):
    preference(d, batch(31, tokens, 2 * pairs, before=33, behind=70), kind=kind, shift=shift)


@pytest.mark.parametrize("tokens,pairs", [(600, 5), (50000, 40)])
def test_pairs_options(d, tokens, pairs):
    b = batch(32, tokens, 2 * pairs)
    preference(d, b, smoothing=0.1, margin=0.3)
    preference(d, b, smoothing=1.0)
    preference(d, b, reference=False, average=True, margin=-0.5, beta=2.0)
    preference(d, b, reference=False, beta=5.0)              # gaps of thousands: the loss is one side of it
    preference(d, b, count=1000.0)
    preference(d, b, gradient=False)
    preference(d, b, gradient=False, rewards=False)
    preference(d, b, beta=0.0)


@pytest.mark.parametrize("tokens,pairs", [(2000, 9), (30000, 11), (30000, 9000), (9000, 3000)])
def test_pairs_loss_is_the_same_without_the_gradient(d, tokens, pairs):
    b = batch(36, tokens, 2 * pairs)
    for k in ({}, {"average": True, "smoothing": 0.2}):
        whole = preference(d, b, **k)
        assert (whole == preference(d, b, gradient=False, **k)).all() and (whole == preference(d, b, rewards=False, **k)).all()


@pytest.mark.parametrize("tokens", [1000, 30000])
def test_pairs_masked_places_and_empty_sequences(d, tokens):
    b = batch(33, tokens, 12)
    out = b["ids"] < 0
    b["logprob"][out], b["reference"][out] = np.nan, -np.inf
    preference(d, b), preference(d, b, average=True)
    b["ids"][:] = -1
    loss = preference(d, {**b, "logprob": np.full(tokens, np.nan, np.float32)})
    assert loss[1] == 0 and loss[2] == 0 and abs(loss[0] - math.log(2)) < 4 * U


def test_pairs_boundaries_on_tiles(d):
    # sequences that begin or end where a tile of 4096 does, or fill one
    for cuts in ([0, 4096, 8192, 12288, 16384], [0, 4095, 8192, 8193, 16384], [0, 4097, 4097, 4097, 16384], [0, 1, 2, 16383, 16384], [4096, 4096, 8192, 8192, 12288]):
        b = batch(34, 16384, 4)
        b["offsets"] = np.array(cuts)
        preference(d, b), preference(d, b, average=True)
        check(policy(d, b, per_token=False, by_sequence=True))


def test_pairs_no_pairs_and_no_tokens(d):
    b = batch(35, 9000, 2)
    b["offsets"] = np.array([0])
    loss, r = torch.full((3,), math.nan, device="cuda:0"), torch.empty(0, device="cuda:0")
    d.fpreference_loss(up(b["logprob"]), up(b["ids"]), up(b["offsets"]), loss, r)
    assert (loss == 0).all()
    for pairs in (3, 4000):                                  # all sequences empty
        e = batch(36, 0, 2 * pairs)
        loss = preference(d, e)
        assert abs(loss[0] - math.log(2)) < 4 * U


def test_pairs_same_bits_each_time(d):
    b = batch(37, 150001, 400)
    t = {k: up(v) for k, v in b.items()}
    results = []
    for _ in range(3):
        loss, r, g = torch.empty(3, device="cuda:0"), torch.empty(400, device="cuda:0"), torch.zeros(150001, device="cuda:0")
        d.fpreference_loss(t["logprob"], t["ids"], t["offsets"], loss, r, g, reference=t["reference"])
        results.append((loss, r, g))
    assert all(torch.equal(x, y) for o in results[1:] for x, y in zip(results[0], o))


def test_gradients_against_differences(d):
    # the device's losses of shifted inputs, in a batch small enough for fp32 differences: loss 1, shift 1/64, third derivatives below 2
    b = batch(38, 12, 4, counted=1.0, empty_rows=False)
    b["old"] = (b["logprob"] + np.float32(0.01)).astype(np.float32)   # away from the clipping borders
    h = np.float32(1 / 64)
    got = policy(d, b, by_sequence=True)
    _, _, _, want = got
    grad = got[1]
    for i in range(12):
        shifted = []
        for s in (h, -h):
            c = {**b, "logprob": b["logprob"].copy()}
            c["logprob"][i] += s
            shifted.append(policy(d, c, by_sequence=True)[0][0])
        assert abs((shifted[0] - shifted[1]) / (2 * h) - grad[i]) < 2 * float(h) ** 2 + 64 * U / float(h)
    pair_loss = lambda c: rows.preference_loss64(c["logprob"], c["reference"], c["ids"], c["offsets"], 0.5, 0.1, 0.2)[0][0]  # noqa: E731
    g = torch.zeros(12, device="cuda:0")
    d.fpreference_loss(up(b["logprob"]), up(b["ids"]), up(b["offsets"]), torch.empty(3, device="cuda:0"), None, g, reference=up(b["reference"]), beta=0.5,
                       smoothing=0.1, margin=0.2)
    for i in range(12):
        shifted = []
        for s in (1e-4, -1e-4):
            c = {**b, "logprob": b["logprob"].astype(np.float64)}
            c["logprob"][i] += s
            shifted.append(pair_loss(c))
        assert abs((shifted[0] - shifted[1]) / 2e-4 - g[i].item()) < 1e-6


@pytest.mark.parametrize("tokens", [1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 6143, 6144, 6145])
def test_few_tokens_where_the_threads_shares_change(d, tokens):
    for sequences in (2, 64, 2048):
        b = batch(tokens + sequences, tokens, sequences)
        for by_sequence in (False, True):
            for per_token in (False, True):
                check(policy(d, b, per_token=per_token, by_sequence=by_sequence))
        for average in (False, True):
            preference(d, b, average=average)
    b = batch(tokens, tokens - 50, 12, before=20, behind=30)
    check(policy(d, b, by_sequence=True))
    preference(d, b, average=True)


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_long_sequences_among_many_short_ones(d, seed):
    # a lane looks at sequences of up to 64 tokens, its warp at the others; tiles end at 2048
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, 7, 4000)
    lengths[rng.choice(4000, 12, replace=False)] = [63, 64, 65, 127, 128, 129, 2047, 2048, 2049, 5000, 9000, 1000]
    o = np.concatenate([[0], np.cumsum(lengths)]) + 5 * seed
    tokens = int(o[-1]) + 100
    b = batch(seed, tokens, 4000)
    b["ids"], b["offsets"] = np.where(rng.random(tokens) < 0.6, 3, -1), o
    for by_sequence in (False, True):
        for per_token in (False, True):
            check(policy(d, b, per_token=per_token, by_sequence=by_sequence))
    for average in (False, True):
        preference(d, b, average=average)
        preference(d, b, average=average, gradient=False)
