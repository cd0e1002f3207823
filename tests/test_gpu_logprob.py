"""flogprob and flogprob_grad against their formulas in 64 bits.

Tolerances count roundings of U = 2^-24.  With d = x - max (one rounding, U |d|) an exponential is off by U |d| from d, U |d| more where it is
taken as a power of two, and 4 U of its own; a sum of them by its longest chain of additions, classes / 32 + 40 of them at most, and by
its terms' errors weighted by their probabilities.  The logarithm of the sum is then off by the sum's relative error and 2 U of itself."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def env():
    import torch
    import __graft_entry__ as ge
    ge.load_package()
    from polarai_framework_b200.device_builtins import DeviceBuiltins
    return torch, DeviceBuiltins()


def logits(torch, rows, classes, seed=0, pitch=None, offset=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(rows * 7919 + classes + seed)
    pitch = pitch or classes
    buf = torch.full((rows * pitch + offset,), np.nan, device="cuda")
    x = buf[offset:].view(rows, pitch)[:, :classes]
    x.copy_(torch.randn((rows, classes), device="cuda", generator=g) * scale)
    at = torch.randint(0, classes, (rows,), device="cuda", generator=g)
    x[torch.arange(rows, device="cuda"), at] += 5.0
    ids = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.6, at,
                      torch.randint(0, classes, (rows,), device="cuda", generator=g))
    return x, ids


def expect(torch, x, ids):
    x64 = x.double()
    m = x64.amax(1, keepdim=True)
    d = x64 - m
    e = d.exp()
    p = e / e.sum(1, keepdim=True)
    live = p > 0
    dz = torch.where(live, d, 0.0)
    log_sum = e.sum(1).log()
    lse = m[:, 0] + log_sum
    t = (p * dz).sum(1)
    c = (x.shape[1] / 32 + 40) * U
    off_sum = c + (p * (2 * dz.abs() + 4)).sum(1) * U         # relative, of the sum of exponentials
    off_log = off_sum + 2 * U * log_sum.abs()
    dt = torch.gather(d, 1, ids.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    lp = dt - log_sum
    off_lp = U * dt.abs() + off_log + U * lp.abs()
    # T / S: every term by its exponential, its deviation and the product; the sum's chain; the quotient
    off_t = (c + 5 * U) * t.abs() + (p * dz.abs() * (2 * dz.abs() + 6)).sum(1) * U + off_sum * t.abs()
    ent = log_sum - t
    return {"logprob": (lp, off_lp), "entropy": (ent, off_log + off_t + U * ent.abs()), "logsumexp": (lse, off_log + U * lse.abs()),
            "parts": (d, log_sum, off_log)}


def best(torch, x, top):
    """The `top` largest of each row, ties to the lowest index, NaN above all."""
    a = x.cpu().numpy().astype(np.float64)
    ids = np.lexsort((np.broadcast_to(np.arange(a.shape[1]), a.shape), np.where(np.isnan(a), -np.inf, -a)), axis=1)[:, :top]
    return torch.from_numpy(np.ascontiguousarray(ids)).cuda()


def close(got, want, off):
    both = want == got.double()                              # (infinities)
    d = torch_where(both, got.double() - want)
    assert not d.isnan().any()
    worst = (d.abs() - 1.000001 * off - 1e-37)[~both].max().item() if (~both).any() else 0.0
    assert worst <= 0, (worst, d.abs().max().item())


def torch_where(both, d):
    return d.masked_fill(both, 0.0)


def run(torch, d, x, ids, top, kind=None):
    rows = x.shape[0]
    nan = lambda *s: torch.full(s, np.nan, device="cuda")  # noqa: E731
    kind = kind or torch.int64
    o = {"logprob": nan(rows), "entropy": nan(rows), "logsumexp": nan(rows)}
    o["top_ids"] = torch.full((rows, top), -7, dtype=kind, device="cuda") if top else None
    o["top_logprob"] = nan(rows, top) if top else None
    d.flogprob(x, ids.to(kind), *o.values())
    return o


def check(torch, x, ids, o, top):
    want = expect(torch, x, ids)
    for k in ("logprob", "entropy", "logsumexp"):
        close(o[k], *want[k])
    if top:
        at = best(torch, x, top)
        assert torch.equal(o["top_ids"].long(), at)
        dd, log_sum, off_log = want["parts"]
        dt = torch.gather(dd, 1, at)
        w = dt - log_sum[:, None]
        close(o["top_logprob"], w, U * dt.abs() + off_log[:, None] + U * w.abs())


SIZES = [(1, 1, 1), (7, 2, 2), (100, 3, 1), (65, 10, 0), (1000, 10, 10), (33, 16, 5), (40, 17, 17), (129, 31, 20), (64, 32, 32), (9, 33, 32),
         (50, 100, 5), (20, 257, 32), (300, 1000, 3), (5, 1024, 20), (3, 1025, 1), (70, 2048, 0), (6, 4099, 20), (200, 5000, 5),
         (2, 8191, 32), (150, 10007, 5), (300, 20000, 0), (1, 32768, 20), (3, 50001, 20), (40, 65536, 5), (1, 131072, 20), (2, 200003, 32)]


@pytest.mark.parametrize("rows,classes,top", SIZES)
def test_forward(env, rows, classes, top):
    torch, d = env
    x, ids = logits(torch, rows, classes)
    o = run(torch, d, x, ids, top)
    check(torch, x, ids, o, top)
    # each result alone has the same bits
    if top:
        alone = torch.empty_like(o["top_ids"])
        d.flogprob(x, None, None, None, None, alone)
        assert torch.equal(alone, o["top_ids"])
        values = torch.empty_like(o["top_logprob"])
        d.flogprob(x, None, None, None, None, None, values)
        assert torch.equal(values, o["top_logprob"])
    for k, at in (("logprob", 2), ("entropy", 3), ("logsumexp", 4)):
        alone = torch.empty_like(o[k])
        d.flogprob(x, ids, *[alone if i == at else None for i in range(2, 5)])
        assert torch.equal(alone, o[k]), k


@pytest.mark.parametrize("rows,classes,pitch,offset,top", [(5, 10, 12, 1, 3), (9, 100, 103, 2, 20), (4, 1000, 1024, 3, 5), (3, 5001, 5003, 1, 20),
                                                           (20, 5000, 5120, 0, 2), (2, 70000, 70001, 3, 32)])
def test_rows_apart_and_on_odd_boundaries(env, rows, classes, pitch, offset, top):
    torch, d = env
    x, ids = logits(torch, rows, classes, pitch=pitch, offset=offset)   # NaN between the rows
    for kind in (torch.int64, torch.int32, torch.float32):
        check(torch, x, ids, run(torch, d, x, ids, top, kind), top)


def edge_rows(x, ids, classes):
    """Into the first 13 rows; the third one is shut out altogether."""
    low = float(np.finfo(np.float32).min)
    x[0] = 1.25                                              # all alike
    x[1, ::2] = -np.inf                                      # half of them shut out
    x[2] = -np.inf                                           # all of them
    x[3] = low                                               # all at the type's lowest value
    x[4, classes // 2:] = low
    x[5] = x[5].round()                                 # many ties
    x[6] = x.new_tensor(range(classes)) * 1e-3       # rising, and falling
    x[7] = -x.new_tensor(range(classes)) * 1e-3
    x[8] = 0.0
    x[8, ::3] = -0.0                                         # a zero is a zero
    x[9] = 3e38                                              # the largest
    x[10] = -np.inf
    x[10, classes - 1] = -5.0                                # one left
    x[11, 1:] = x[11, 1:] - 400.0                            # nothing but the first
    x[12, :classes // 2] = low
    x[12, 0] = 80.0
    # (differences of the lowest value and others are beyond fp32, and their exponential is zero all the same)
    ids[1], ids[4], ids[10] = 1, 0, 0
    ids[12] = 0


@pytest.mark.parametrize("classes", [7, 32, 40, 500, 3000, 30000, 140001])
def test_ties_masks_and_values_at_the_edges(env, classes):
    torch, d = env
    top = min(classes, 20)
    x, ids = logits(torch, 14, classes)
    edge_rows(x, ids, classes)
    o = run(torch, d, x, ids, top)
    keep = [i for i in range(14) if i != 2]
    check(torch, x[keep], ids[keep], {k: v[keep] for k, v in o.items()}, top)
    assert o["logprob"][2] == -np.inf and o["entropy"][2] == 0 and o["logsumexp"][2] == -np.inf
    assert o["top_ids"][2].tolist() == list(range(top)) and (o["top_logprob"][2] == -np.inf).all()
    # padding, ids that are none, NaN and infinity
    x, ids = logits(torch, 12, classes, seed=1)
    plain = run(torch, d, x, ids, top)
    ids[0], ids[1], ids[2], ids[3] = -1, -100, classes, 2 ** 40
    x[4, classes // 3], x[5, 1] = np.nan, np.inf
    o = run(torch, d, x, ids, top)
    assert (o["logprob"][:2] == 0).all() and torch.isnan(o["logprob"][2:6]).all()
    assert torch.isnan(o["entropy"][4:6]).all() and torch.isnan(o["logsumexp"][4:6]).all()
    assert o["top_ids"][4, 0] == classes // 3 and o["top_ids"][5, 0] == 1
    assert torch.equal(o["top_ids"], best(torch, x, top))
    for k in ("entropy", "logsumexp", "top_logprob"):
        assert torch.equal(o[k][:4], plain[k][:4]) and torch.equal(o[k][6:], plain[k][6:])
    assert torch.equal(o["logprob"][6:], plain["logprob"][6:])
    f = torch.tensor([0.5, -0.5, np.nan, np.inf, float(classes), 1.0] + [0.0] * 6, device="cuda")
    lp = torch.empty(12, device="cuda")
    d.flogprob(logits(torch, 12, classes, seed=1)[0], f, lp)
    assert torch.isnan(lp[[0, 2, 3, 4]]).all() and lp[1] == 0 and torch.isfinite(lp[5:]).all()


@pytest.mark.parametrize("rows", [600, 1003])
@pytest.mark.parametrize("classes", [17, 33, 48, 49, 100, 125, 126, 200, 253, 254, 256, 509, 510, 1024])
def test_edges_among_many_rows(env, rows, classes):
    torch, d = env
    for top, at in ((5, 0), (12, 301), (min(classes, 32), rows - 14)):   # the edges in front, in the middle, at the end
        x, ids = logits(torch, rows, classes, offset=at % 4)
        edge_rows(x[at:], ids[at:], classes)
        nan = rows // 3
        x[nan, classes - 1] = np.nan
        o = run(torch, d, x, ids, top)
        keep = torch.tensor([i for i in range(rows) if i not in (at + 2, nan)], device="cuda")
        check(torch, x[keep], ids[keep], {k: v[keep] for k, v in o.items()}, top)
        assert o["logprob"][at + 2] == -np.inf and o["top_ids"][at + 2].tolist() == list(range(top))
        assert torch.isnan(o["logprob"][nan]) and torch.equal(o["top_ids"][nan:nan + 1], best(torch, x[nan:nan + 1], top))


def expect_grad(torch, x, ids, lse, ent, g, ge):
    x64 = x.double()
    l = x64 - lse.double()[:, None]
    p = l.exp()
    live = p > 0
    lz = torch.where(live, l, 0.0)
    g64 = torch.where(ids < 0, 0.0, g.double())[:, None]
    ge64 = ge.double()[:, None] if ge is not None else torch.zeros_like(g64)
    h = ent.double()[:, None]
    dx = p * (-g64 - torch.where(live, ge64 * (lz + h), 0.0))
    hot = torch.zeros_like(dx).scatter_(1, ids.clamp(0)[:, None], g64)
    # p: U |l| from the difference, as much from the power of two, 4 U of its own; the factor's terms; product, factor and sum
    size = p * (g64.abs() + ge64.abs() * (lz.abs() + h.abs()))
    off = U * ((2 * lz.abs() + 10) * size + 2 * hot.abs() + (dx + hot).abs())
    return dx + hot, off


@pytest.mark.parametrize("rows,classes,pitch,dpitch,offset", [
    (1, 1, 1, 1, 0), (300, 10, 10, 10, 0), (5, 3, 3, 3, 1), (64, 32, 32, 32, 0), (9, 33, 33, 33, 0), (7, 100, 104, 100, 0), (11, 1000, 1000, 1001, 2),
    (40, 1024, 1024, 1024, 0), (5, 4097, 4097, 4097, 3), (33, 5000, 5000, 5000, 0), (3, 5001, 5003, 5007, 1), (99, 10007, 10007, 10007, 0),
    (20, 32000, 32000, 32000, 0), (2, 131072, 131072, 131072, 0), (2, 70001, 70004, 70001, 0)])
def test_backward(env, rows, classes, pitch, dpitch, offset):
    torch, d = env
    x, ids = logits(torch, rows, classes, pitch=pitch, offset=offset)
    gen = torch.Generator(device="cuda").manual_seed(rows)
    g, ge = torch.randn(rows, device="cuda", generator=gen), torch.randn(rows, device="cuda", generator=gen)
    if rows > 4:
        ids[1], g[2], ge[2] = -1, 0.0, 0.0
        ge[3] = 0.0
    lse = torch.logsumexp(x.double(), 1)
    ent = (lse - ((x.double() - lse[:, None]).exp() * x.double()).sum(1)).float()
    lse = lse.float()
    for with_entropy in (False, True):
        for kind in (torch.int64, torch.int32, torch.float32) if with_entropy else (torch.int64,):
            out = torch.full((rows * dpitch + offset,), 77.0, device="cuda")
            dx = out[offset:].view(rows, dpitch)[:, :classes]
            d.flogprob_grad(x, ids.to(kind), lse, ent if with_entropy else None, g, ge if with_entropy else None, dx)
            want, off = expect_grad(torch, x, ids, lse, ent, g, ge if with_entropy else None)
            close(dx, want, off)
            out[offset:].view(rows, dpitch)[:, :classes] = 77.0
            assert (out == 77.0).all()                       # nothing between the rows was written
    buf = x.clone(memory_format=torch.preserve_format) if pitch == classes else None
    if buf is not None:
        dx = torch.empty_like(buf)
        d.flogprob_grad(buf, ids, lse, ent, g, ge, dx)
        d.flogprob_grad(buf, ids, lse, ent, g, ge, buf)      # in place
        assert torch.equal(buf, dx)


@pytest.mark.parametrize("classes", [9, 64, 3000, 30001])
def test_backward_at_the_edges(env, classes):
    torch, d = env
    x, ids = logits(torch, 10, classes)
    x[0] = -np.inf                                           # a row without any probability
    x[1, : classes // 2] = -np.inf
    ids[1] = 0                                               # given a class that is shut out
    x[2], x[3] = np.nan, np.nan                              # rows that nothing reaches
    ids[2] = -1
    x[4, 3] = np.nan
    ids[5] = classes
    ids[6] = -1
    g, ge = torch.ones(10, device="cuda"), torch.full((10,), 0.5, device="cuda")
    g[3] = 0
    ge[2], ge[3], ge[5], ge[6] = 0, 0, 0, 0
    ids[3] = classes + 5
    lse = torch.logsumexp(x.double(), 1)
    p = (x.double() - lse[:, None]).exp()
    ent = -torch.where(p > 0, p * (x.double() - lse[:, None]), 0.0).sum(1).float()
    lse = lse.float()
    dx = torch.full((10, classes), 77.0, device="cuda")
    d.flogprob_grad(x, ids, lse, ent, g, ge, dx)
    assert not dx[[0, 2, 3, 6]].any() and torch.isnan(dx[5]).all()
    assert torch.isnan(dx[4]).all()
    rows = [1, 7, 8, 9]
    want, off = expect_grad(torch, x[rows], ids[rows], lse[rows], ent[rows], g[rows], ge[rows])
    close(dx[rows], want, off)
    assert dx[1, 0] == 1.0 and not dx[1, 1:classes // 2].any()


def test_gradient_against_differences(env):
    torch, d = env
    x, ids = logits(torch, 4, 23)
    o = run(torch, d, x, ids, 0)
    g, ge = torch.tensor([1.0, -0.5, 0.0, 2.0], device="cuda"), torch.tensor([0.0, 1.5, -1.0, 0.25], device="cuda")
    dx = torch.empty_like(x)
    d.flogprob_grad(x, ids, o["logsumexp"], o["entropy"], g, ge, dx)
    x64, t = x.double().cpu(), ids.cpu()

    def value():
        l = x64 - torch.logsumexp(x64, 1, keepdim=True)
        return (g.double().cpu() * l[torch.arange(4), t] - ge.double().cpu() * (l.exp() * l).sum(1)).sum().item()

    for r in range(4):
        for c in range(23):
            at = x64[r, c].item()
            x64[r, c] = at + 1e-5
            up = value()
            x64[r, c] = at - 1e-5
            down = value()
            x64[r, c] = at
            # third derivatives times 1e-10 and 2^-53 of the value over 2e-5; the kernel: some 40 U of factors below 60
            assert abs((up - down) / 2e-5 - dx[r, c].item()) < 2e-4


def test_streams_and_captures(env):
    torch, d = env
    for rows, classes in ((2, 40000), (300, 700), (5000, 10)):
        x, ids = logits(torch, rows, classes)
        want = run(torch, d, x, ids, 5)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append([run(torch, d, x, ids, 5) for _ in range(5)])
        torch.cuda.synchronize()
        assert all(torch.equal(o[k], want[k]) for r in got for o in r for k in o)
        o = {k: torch.zeros_like(v) for k, v in want.items()}
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            d.flogprob(x, ids, *o.values())
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o[k], want[k]) for k in o)


def test_rows_beyond_32_bits_of_offset(env):
    torch, d = env
    rows, classes = 70000, 65536                             # 4.6 G logits
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("not enough free memory")
    x = torch.empty((rows, classes), device="cuda")
    x[:2] = logits(torch, 2, classes)[0]
    x[2:] = x[0]
    x[-1] = x[1]
    ids = torch.full((rows,), 5, device="cuda")
    o = run(torch, d, x, ids, 2)
    for k in o:
        assert torch.equal(o[k][-1], o[k][1]) and torch.equal(o[k][2:-1], o[k][:1].expand_as(o[k][2:-1])), k
    g = torch.ones(rows, device="cuda")
    two = torch.empty((2, classes), device="cuda")
    d.flogprob_grad(x[:2], ids[:2], o["logsumexp"][:2], None, g[:2], None, two)
    d.flogprob_grad(x, ids, o["logsumexp"], None, g, None, x)
    assert torch.equal(x[-1], two[1]) and torch.equal(x[-2], two[0]) and torch.equal(x[:2], two)
