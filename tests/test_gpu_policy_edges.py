"""The operators over decisions where their inputs are special: references that rule the action
out, NaN among the rows' numbers, advantages of zero, certain preferences, rows of every kernel
next to the border of the clip, and how exact the losses are."""
import zlib

import numpy as np
import policy_reference as ref64
import pytest

pytestmark = pytest.mark.gpu

# rows of a thread, of some lanes, of a workgroup, in pieces (float32)
WIDTHS = [4, 40, 5000, 40000]


def _normal(*shape, key):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr((shape, key)).encode()))
    return torch.randn(shape, generator=g, device="cuda")


def _rows(n, k, dtype="float32", scale=2.0):
    import torch

    print(f"case n={n} k={k} {dtype}", flush=True)
    z = (_normal(n, k, key="z") * scale).to(getattr(torch, dtype))
    y = torch.arange(n, device="cuda") * 7 % k
    return z, y


def _logp(z, y):
    import torch

    return torch.log_softmax(z.double(), 1).gather(1, y[:, None])[:, 0]


def _unlikely(n, k):
    """Rows whose taken class has log-probability -70 exactly: exp(-70) is lost beside 1, also in
    64 bits, and so is what its probability takes from its gradient."""
    import torch

    z = torch.full((n, k), -200.0, device="cuda")
    y = torch.arange(n, device="cuda") % (k - 1)
    z[:, k - 1] = 0.0
    z.scatter_(1, y[:, None], -70.0)
    return z, y


# ---------------------------------------------------------------------------
# The KL term
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_references_that_rule_the_action_out(ws, device, k, dtype):
    """log-probability -infinity, or nearly: the estimate grows without bound, its slope is -1."""
    import torch
    from dpgbdt import ops

    z, y = _rows(12, k, dtype)
    logp = _logp(z, y)
    reference = (logp - 0.1).float()
    reference[::4] = -float("inf")
    reference[1::4] = -1e8
    reference[2::4] = -1e30
    old, adv = logp.float(), torch.zeros(12, device="cuda")
    out = ops.policy_loss(ws, z, y, old, adv, reference=reference, kl=0.5,
                          hessian=dtype == "float32")
    d = reference.double() - logp
    far = torch.arange(12, device="cuda") % 4 != 3
    assert torch.equal(out.kl[far], (-1.0 - d).float()[far])
    assert torch.equal(out.loss[far], (0.5 * (-1.0 - d)).float()[far])
    rows = ref64.Rows(z, y)
    c = -0.5 * np.expm1(d.cpu().numpy())
    # the slope: 0.5 of one rounding of e^d - 1, and of logp's error times e^d
    slope = 0.5 * (2.0 ** -22 + np.exp(d.cpu().numpy()) * rows.logp_bound())
    g, off = rows.grad(c, np.zeros(12))
    ref64.close(out.grad, g, off + slope[:, None], "grad")
    if out.hess is not None:
        h, off = rows.hess(c, np.zeros(12))
        ref64.close(out.hess, h, off + slope[:, None], "hess")


@pytest.mark.parametrize("k", WIDTHS)
def test_kl_term_to_its_last_bits(ws, device, k):
    """e^d - 1 - d and e^d - 1 over the range of d, each to 2^-22 of itself: d is exact here (see
    _unlikely), and each is a few roundings of 2^-24 away from its result."""
    import torch
    from dpgbdt import ops

    size = torch.logspace(-3, np.log10(60.0), 32, device="cuda")
    reference = torch.cat([size, -size, torch.tensor([0.5, -0.5, 1.0, -1.0], device="cuda")]) - 70.0
    z, y = _unlikely(len(reference), k)
    zero = torch.zeros_like(reference)
    out = ops.policy_loss(ws, z, y, zero - 70.0, zero, reference=reference, kl=0.5)
    d = reference.cpu().double().numpy() + 70.0
    assert np.abs(d).max() > 59.0 and (d != 0).all()
    want = np.where(np.abs(d) < 0.5, d * d * _tangent_rest(d), np.expm1(d) - d)
    ref64.close(out.kl, want, 2.0 ** -22 * want, "kl")
    ref64.close(out.loss, 0.5 * want, 2.0 ** -23 * want, "loss")
    slope = 0.5 * np.expm1(d)
    ref64.close(out.grad.gather(1, y[:, None])[:, 0], -slope, 2.0 ** -22 * np.abs(slope), "slope")


def _tangent_rest(d):
    """(e^d - 1 - d) / d^2 by its series, for |d| < 0.5."""
    total, term = np.zeros_like(d), np.full_like(d, 0.5)
    for i in range(3, 24):
        total += term
        term = term * d / i
    return total


# ---------------------------------------------------------------------------
# The ratio
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("k", WIDTHS)
def test_ratio_to_its_last_bits(ws, device, k):
    """Log-ratios that 32 bits do not hold, of both signs: loss and slope are two roundings away
    from the ratio of exact numbers (see _unlikely)."""
    import torch
    from dpgbdt import ops

    old = -torch.cat([torch.linspace(0.3, 20.0, 40, device="cuda"),
                      torch.linspace(70.3, 130.0, 40, device="cuda")])
    z, y = _unlikely(len(old), k)
    x = -70.0 - old.cpu().double().numpy()
    assert (np.float32(x) != x).sum() > 30
    adv = torch.where(old > -70.0, 1.5, -1.5)  # the side on which nothing is clipped
    out = ops.policy_loss(ws, z, y, old, adv)
    want = -np.exp(x) * adv.cpu().double().numpy()
    ref64.close(out.loss, want, 2.0 ** -23 * np.abs(want), "loss")
    ref64.close(out.grad.gather(1, y[:, None])[:, 0], want, 2.0 ** -22 * np.abs(want), "slope")


@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_advantages_of_zero(ws, device, k, dtype):
    """Nothing is lost or gained, however large the ratio."""
    import torch
    from dpgbdt import ops

    z, y = _rows(8, k, dtype)
    logp = _logp(z, y)
    old = (logp - torch.tensor([0.0, 1.0, 88.0, 89.0, 100.0, 700.0, 800.0, 1e30],
                               device="cuda")).float()
    zero = torch.zeros(8, device="cuda")
    for adv in (zero, -zero):
        out = ops.policy_loss(ws, z, y, old, adv, hessian=dtype == "float32")
        assert not out.loss.any() and not out.grad.any()
        if out.hess is not None:
            assert (out.hess == 1e-16).all()


# ---------------------------------------------------------------------------
# NaN
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("what", ["old", "advantage", "weight", "reference"])
def test_nan_of_a_row_reaches_its_gradient(ws, device, k, dtype, what):
    """On either side of either border of the clip, for advantages of either sign."""
    import torch
    from dpgbdt import ops

    n = 16
    z, y = _rows(n, k, dtype)
    logp = _logp(z, y)
    x = torch.tensor([-1.0, -0.3, -0.1, 0.0, 0.1, 0.3, 1.0, 2.0], device="cuda").repeat(2)
    sign = torch.where(torch.arange(n, device="cuda") < 8, 1.0, -1.0)
    args = {"old": (logp - x).float(), "advantage": sign, "weight": sign * 0 + 2.0,
            "reference": (logp + 0.2).float()}

    def loss(kl=0.1):
        return ops.policy_loss(ws, z, y, args["old"], args["advantage"], args["weight"],
                               args["reference"], kl=kl, hessian=dtype == "float32")

    clean = loss()
    bad = torch.arange(n, device="cuda") % 2 == 0
    args[what] = torch.where(bad, float("nan"), args[what])
    out = loss()
    held = [out.loss, out.grad] + [out.hess] * (out.hess is not None)
    for got, was in zip(held, [clean.loss, clean.grad, clean.hess]):
        assert got[bad].isnan().all()
        assert torch.equal(got[~bad], was[~bad])
    if what == "reference":  # without the term's weight only its own output has it
        out = loss(kl=0.0)
        assert out.kl[bad].isnan().all() and not out.loss.isnan().any()
        assert not out.grad.isnan().any()


@pytest.mark.parametrize("k", WIDTHS)
def test_hessians_keep_nan(ws, device, k):
    import torch
    from dpgbdt import ops

    z, y = _rows(8, k)
    old = _logp(z, y).float()
    adv = torch.ones(8, device="cuda")
    ptr = torch.tensor([0, 2, 4, 6, 8], device="cuda")
    clean = ops.policy_loss(ws, z, y, old, adv, hessian=True)
    pairs = ops.preference_loss(ws, z, y, ptr, hessian=True)
    z[1, k // 2] = float("nan")
    out = ops.policy_loss(ws, z, y, old, adv, hessian=True)
    for x in out:
        if x is not None:
            assert x[1].isnan().all()
    rest = [i for i in range(8) if i != 1]
    assert torch.equal(out.hess[rest], clean.hess[rest])
    out = ops.preference_loss(ws, z, y, ptr, hessian=True)
    for x in (out.grad, out.hess):
        assert x[:4].isnan().all()  # the pair's
    assert torch.equal(out.grad[4:], pairs.grad[4:]) and torch.equal(out.hess[4:], pairs.hess[4:])


# ---------------------------------------------------------------------------
# Certain preferences
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [3, 400])
@pytest.mark.parametrize("smoothing", [0.0, 1.0, 0.25])
def test_pairs_with_an_illegal_action(ws, device, rows, smoothing):
    """The scores are infinite; a term without weight adds nothing, and no gradient is lost."""
    import torch
    from dpgbdt import ops

    n, beta = 4 * rows, 0.5
    z, y = _rows(n, 10)
    for at in (rows + 1, 2 * rows + 1):  # in the first pair's worse, the second's better sequence
        z[at, y[at]] = -float("inf")
    ptr = torch.arange(0, n + 1, rows, device="cuda")
    out = ops.preference_loss(ws, z, y, ptr, beta=beta, smoothing=smoothing, hessian=True)
    inf = float("inf")
    assert out.score.tolist() == [inf, -inf]
    assert out.loss.tolist() == [inf if smoothing > 0.0 else 0.0, inf if smoothing < 1.0 else 0.0]
    slope = np.array([smoothing, -(1.0 - smoothing)]) * beta  # the limits of the sigmoids
    c = np.repeat(np.stack([slope, -slope], 1).ravel(), rows)
    reference = ref64.Rows(z, y)
    g, off = reference.grad(c, np.zeros(n))
    ref64.close(out.grad, g, off, "grad")
    h, off = reference.hess(c, np.zeros(n))
    ref64.close(out.hess, h, off, "hess")


# ---------------------------------------------------------------------------
# Rows read twice by a workgroup: 256 and more, longer than 128 KB
# ---------------------------------------------------------------------------
LONG = [("float32", 33001), ("bfloat16", 65601), ("float16", 65601)]


def _long(dtype, k, n=257):
    """Margins with an illegal class in ten, rows that are not counted, rows without a class."""
    import torch

    z, y = _rows(n, k, dtype)
    illegal = _normal(n, k, key="illegal") < -1.28
    illegal.scatter_(1, y[:, None], False)
    z.masked_fill_(illegal, -float("inf"))
    y[5::50] = -1
    y[6::50] = k
    z[5::50] = z[6::50] = float("nan")
    z[7::50] = -float("inf")
    y[8], y[9] = k - 1, 0
    z[8, k - 1] = z[9, 0] = 1.0
    return z, y


@pytest.mark.parametrize("dtype,k", LONG)
def test_long_rows_of_many(ws, device, dtype, k):
    import torch
    from dpgbdt import ops

    z, y = _long(dtype, k)
    n = len(y)
    rows = ref64.Rows(z, y)
    logp, h = ops.action_logprobs(ws, z, y, entropy=True)
    ref64.close(logp, rows.keep(rows.logp), rows.logp_bound(), "logp")
    ref64.close(h, rows.keep(rows.h), rows.h_bound(), "entropy")
    dlogp, dent = _normal(n, key="dlogp"), _normal(n, key="dentropy")
    grad = ops.action_logprobs_backward(ws, z, y, dlogp, dent)
    g, off = rows.grad(rows.keep(dlogp.cpu().double().numpy()),
                       rows.keep(-dent.cpu().double().numpy()))
    ref64.close(grad, g, off, "backward")


def _policy_inputs(z, y):
    import torch

    n, k = z.shape
    logp = _logp(torch.nan_to_num(z, 0.0, neginf=-300.0), y.clamp(0, k - 1))
    x = _normal(n, key="x") * 0.4
    x = torch.where((x - 0.2).abs() < 0.05, x - 0.1, x)     # off the borders
    x = torch.where((x + 0.22).abs() < 0.05, x + 0.1, x)
    return ((logp - x).float(), _normal(n, key="adv"), _normal(n, key="w").abs() + 0.5,
            (logp + _normal(n, key="ref") * 0.2).float())


@pytest.mark.parametrize("dtype,k", LONG)
def test_long_rows_of_many_policy(ws, device, dtype, k):
    from dpgbdt import ops

    z, y = _long(dtype, k)
    old, adv, weight, reference = _policy_inputs(z, y)
    weight[3::50] = 0.0
    out = ops.policy_loss(ws, z, y, old, adv, weight, reference, kl=0.05, entropy=0.01,
                          hessian=dtype == "float32")
    _check_policy(out, z, y, old, adv, weight, reference, 0.05, 0.01)
    if out.hess is not None:
        plain = ops.policy_loss(ws, z, y, old, adv, weight, reference, kl=0.05, entropy=0.01)
        assert (plain.grad == out.grad).all()


def _check_policy(out, z, y, old, adv, weight, reference, kl, entropy):
    rows = ref64.Rows(z, y, weight)
    loss, k3, c, n = ref64.policy(rows, old, adv, reference, 0.2, 0.2, kl, entropy)
    off = rows.logp_bound()
    a = np.abs(adv.cpu().double().numpy())
    ratio = np.exp(np.where(rows.counted, rows.logp - old.cpu().double().numpy(), 0.0))
    ed = np.exp(np.where(rows.counted, reference.cpu().double().numpy() - rows.logp, 0.0))
    ref64.close(out.logp, rows.keep(rows.logp), off, "logp")
    ref64.close(out.entropy, rows.keep(rows.h), rows.h_bound(), "entropy")
    k_off = rows.keep(np.abs(ed - 1.0) * off + 1e-12)  # the second order in logp's error
    ref64.close(out.kl, k3, k_off + np.abs(k3) * 2.0 ** -22, "kl")
    slope = rows.keep(rows.w * (a * ratio * (off + 2.0 ** -22) + kl * (ed * off + 2.0 ** -22)))
    loss_off = rows.w * (a * np.maximum(ratio, 1.2) * (off + 2.0 ** -22) + kl * k_off
                         + entropy * rows.h_bound())
    ref64.close(out.loss, loss, rows.keep(loss_off) + np.abs(loss) * 2.0 ** -22, "loss")
    g, g_off = rows.grad(c, n)
    ref64.close(out.grad, g, g_off + slope[:, None], "grad")
    if out.hess is not None:
        h, h_off = rows.hess(c, n)
        ref64.close(out.hess, h, h_off + slope[:, None], "hess")


@pytest.mark.parametrize("dtype,k", LONG)
@pytest.mark.parametrize("average", [False, True])
def test_long_rows_of_many_preference(ws, device, dtype, k, average):
    """Statistics are kept from the scores for the gradient."""
    import torch
    from dpgbdt import ops

    z, y = _long(dtype, k)
    n, beta = len(y), 0.02
    ptr = torch.tensor([0, 30, 50, 50, 120, 200, 250], device="cuda")  # the last rows: of no pair
    reference = _normal(n, key="ref") * 0.1 - 11.0
    out = ops.preference_loss(ws, z, y, ptr, reference, beta=beta, smoothing=0.1, average=average,
                              hessian=dtype == "float32")
    rows = ref64.Rows(z, y)
    score, loss, c = ref64.preference(rows, ptr, reference, beta, 0.1, average)
    off = rows.logp_bound()
    edges = ptr.cpu().numpy()
    count = np.array([rows.counted[b:e].sum() for b, e in zip(edges, edges[1:])])
    share = 1.0 / np.maximum(count, 1) if average else np.ones(6)
    sums = np.array([off[b:e].sum() for b, e in zip(edges, edges[1:])]) * share
    s_off = beta * (sums[0::2] + sums[1::2])
    ref64.close(out.logp, rows.keep(rows.logp), off, "logp")
    ref64.close(out.score, score, s_off, "score")
    ref64.close(out.loss, loss, s_off + 2.0 ** -24, "loss")
    slope = np.zeros(n)
    for i in range(6):
        slope[edges[i]:edges[i + 1]] = beta * s_off[i // 2] * share[i]
    g, g_off = rows.grad(c, np.zeros(n))
    ref64.close(out.grad, g, g_off + rows.keep(slope)[:, None], "grad")
    if out.hess is not None:
        h, h_off = rows.hess(c, np.zeros(n))
        ref64.close(out.hess, h, h_off + rows.keep(slope)[:, None], "hess")


# ---------------------------------------------------------------------------
# The border of the clip
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n,k,dtype", [(300, 9, "bfloat16"), (100, 1500, "float16"),
                                       (64, 2056, "float32"), (64, 5000, "float32"),
                                       (40, 25001, "float32"), (40, 30000, "bfloat16"),
                                       (260, 33001, "float32"), (20, 140001, "float16")])
def test_border_of_the_clip_in_every_kernel(ws, device, n, k, dtype):
    """Old log-probabilities within a rounding of the clip's border: the side is that of 64 bits,
    and rows that were summed again have the gradient of their margins."""
    import torch
    from dpgbdt import ops

    z, y = _rows(n, k, dtype)
    adv = _normal(n, key="adv")
    logp = _logp(z, y)
    border = torch.where(adv > 0, np.log1p(0.2), np.log1p(-0.2))
    old = (logp - border).float()
    out = ops.policy_loss(ws, z, y, old, adv)
    rows = ref64.Rows(z, y)
    up = adv.cpu().numpy() > 0
    gap = (rows.logp - old.cpu().double().numpy()) - np.where(up, np.log1p(0.2), np.log1p(-0.2))
    active = np.where(up, gap < 0, gap > 0)
    clear = np.abs(gap) > 1e-12  # nearer, 64 bits do not tell either
    assert 0.2 < active.mean() < 0.8 and clear.mean() > 0.95 and np.abs(gap).max() < 5e-6
    c = np.where(active, -np.exp(border.cpu().numpy() + gap) * adv.cpu().double().numpy(), 0.0)
    g, off = rows.grad(c, np.zeros(n))
    slope = np.abs(c) * 2.0 ** -20  # logp's error and roundings of the ratio
    some = np.flatnonzero(clear)
    ref64.close(out.grad[some], g[some], (off + slope[:, None])[some], "grad")


# ---------------------------------------------------------------------------
# The same margins in other calls
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,k", [("float32", 7), ("float32", 100), ("bfloat16", 700),
                                     ("float32", 5000), ("float32", 32771), ("float16", 65543)])
def test_log_probabilities_do_not_go_by_the_batch(ws, device, dtype, k):
    """Rows of up to 8192 whole vectors of 16 bytes: the same bits whatever is beside them."""
    import torch
    from dpgbdt import ops

    z, y = _rows(300, k, dtype)
    logp, h = ops.action_logprobs(ws, z, y, entropy=True)
    for first, n in ((0, 1), (3, 24), (17, 255), (40, 256)):
        zz, yy = z[first:first + n], y[first:first + n]
        some, hh = ops.action_logprobs(ws, zz, yy, entropy=True)
        assert torch.equal(some, logp[first:first + n]) and torch.equal(hh, h[first:first + n])
        out = ops.policy_loss(ws, zz, yy, some, some, hessian=dtype == "float32")
        assert torch.equal(out.logp, some) and torch.equal(out.entropy, hh)


@pytest.mark.parametrize("dtype,k", [("float32", 40000), ("bfloat16", 90001)])
@pytest.mark.parametrize("n", [1, 24, 255, 256])
def test_log_probabilities_of_long_rows_go_by_the_row_count_only(ws, device, dtype, k, n):
    import torch
    from dpgbdt import ops

    z, y = _rows(n, k, dtype)
    logp, h = ops.action_logprobs(ws, z, y, entropy=True)
    out = ops.policy_loss(ws, z, y, logp, logp, hessian=dtype == "float32")
    assert torch.equal(out.logp, logp) and torch.equal(out.entropy, h)
    pairs = ops.preference_loss(ws, z, y, torch.tensor([0, n // 2, n], device="cuda"))
    assert torch.equal(pairs.logp, logp)
    rows = ref64.Rows(z, y)
    ref64.close(logp, rows.logp, rows.logp_bound(), "logp")


# ---------------------------------------------------------------------------
# Graphs
# ---------------------------------------------------------------------------
def test_graphs_outlive_a_growth_of_the_workspace(device):
    """Larger calls between the replays take other scratch; memory that is allocated after them is
    not what the graph writes to."""
    import torch
    from dpgbdt import ops

    ws = ops.Workspace()
    z, y = _rows(40, 40000)  # rows in pieces
    few, act = _rows(3000, 10)
    ptr = torch.arange(0, 3001, 100, device="cuda")
    gate = torch.sigmoid(_normal(1, 40000, 64, key="gate") + 3.0)  # in splits
    value = _normal(1, 40000, 64, key="value")

    def calls():
        state, last = ops.linear_recurrence(ws, gate, value)
        back = ops.linear_recurrence_backward(ws, gate, state, value)
        out = [state, last, *back, *ops.action_logprobs(ws, z, y, entropy=True),
               *ops.preference_loss(ws, few, act, ptr),
               *ops.preference_loss(ws, z, y, ptr[:3] // 10)]
        return [x for x in out if x is not None]

    calls()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = calls()
    many, acts = _rows(1 << 21, 4)
    marks = []
    for i in range(4):
        n = len(many) >> (3 - i)  # each larger than any before
        pairs = torch.tensor([0, n // 2, n], device="cuda")
        ops.preference_loss(ws, many[:n], acts[:n], pairs)
        torch.cuda.synchronize()
        marks += [torch.full((1 << 20,), 7.0, device="cuda") for _ in range(64)]
        for x in outs:
            x.zero_()
        value.mul_(-1.0)
        few.add_(0.125)
        graph.replay()
        torch.cuda.synchronize()
        want = calls()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i
    assert all((x == 7.0).all() for x in marks)


# ---------------------------------------------------------------------------
# How exact
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("k", [10, 40, 1000, 5000, 40000])
def test_gradients_by_the_roundings_they_have(ws, device, k):
    """p: z - m and the exponent are rounded once each, |z - m| and |log p| times 2^-24; the
    hardware's 2^x to 2^-23; its products and the slope six times 2^-24.  The sum of exponentials
    has the mean of what its terms are off by."""
    from dpgbdt import ops

    z, y = _rows(64, k, scale=3.0)
    dlogp = _normal(64, key="dlogp")
    grad = ops.action_logprobs_backward(ws, z, y, dlogp)
    rows = ref64.Rows(z, y)
    c = dlogp.cpu().double().numpy()[:, None]
    mean = (rows.p * rows.d).sum(1, keepdims=True)
    rel = (1.25 * rows.d + np.abs(rows.lp) + 1.25 * mean + 2.0 + 2.0 + 6.0) * 2.0 ** -24
    taken = np.zeros_like(rows.p)
    taken[np.arange(64), rows.y] = 1.0
    want = c * (taken - rows.p)
    ref64.close(grad, want, np.abs(c) * rows.p * rel + np.abs(want) * 2.0 ** -24
                + np.abs(c) * taken * 2.0 ** -24, "grad")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("k", [2, 3, 5, 7, 10, 31, 33, 100, 1000, 1500, 3000, 9001, 33001, 70001])
def test_the_logarithm_of_a_sum(ws, device, k, dtype):
    """Equal margins: the sum is k without an error, and a sequence of one row scores -log k less
    a reference of nearly that, of which 2^-39 of the logarithm is left."""
    import torch
    from dpgbdt import ops

    z = torch.full((1, k), 1.5, dtype=getattr(torch, dtype), device="cuda")
    y = torch.zeros(1, dtype=torch.int64, device="cuda")
    reference = torch.tensor([-np.log(k)], dtype=torch.float32, device="cuda")
    out = ops.preference_loss(ws, z, y, torch.tensor([0, 1, 1], device="cuda"), reference,
                              beta=1.0, gradient=False)
    want = -np.log(float(k)) - reference.double().item()
    assert abs(out.score[0].item() - want) <= 2.0 ** -39 * np.log(k) + 2.0 ** -24 * abs(want)


def test_log_probabilities_of_a_sequence_have_no_common_error(ws, device):
    """What all rows are off by in the same way adds up over a sequence.  log2(e) loses 1.3e-8 of
    itself in 32 bits; by 0.8 of probability at e^-10.4 it would be 1.1e-7 a row, against the 2^-25
    that the hardware's exponential may be biased by and the 2^-25 of everything else."""
    import torch
    from dpgbdt import ops

    n, k = 300, 130000
    z = _normal(n, k, key="bias") * 0.25 - float(np.log(k / 4.0))
    y = torch.zeros(n, dtype=torch.int64, device="cuda")
    z[:, 0] = 0.0
    logp = torch.cat([_logp(z[i:i + 50], y[i:i + 50]) for i in range(0, n, 50)])
    reference = logp.float()
    out = ops.preference_loss(ws, z, y, torch.tensor([0, n, n], device="cuda"), reference,
                              beta=1.0, gradient=False)
    want = (logp - reference.double()).sum().item()
    assert abs(out.score[0].item() - want) <= n * 2.0 ** -24
