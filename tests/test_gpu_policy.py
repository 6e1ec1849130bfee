"""The operators over decisions against their definitions in 64 bits: log-probabilities of
actions, the clipped policy loss, the preference loss, gated linear recurrences."""
import zlib

import numpy as np
import policy_reference as ref64
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16", "float16"]
# one class, odd and even small ones, each side of a wavefront and of a workgroup's vectors, rows
# that take a whole workgroup, rows too long for its registers
CLASSES = [1, 2, 3, 7, 10, 16, 31, 64, 65, 100, 257, 515, 1000, 1031, 2056, 4099, 9001, 33001]
LONG = [65537, 140001]


def _rng(*key):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr(key).encode()))  # hash() of a text differs by process
    return g


def _margins(g, n, k, dtype, scale=2.0, illegal=0.0):
    import torch

    z = torch.randn((n, k), generator=g, device="cuda") * scale
    y = torch.randint(k, (n,), generator=g, device="cuda")
    if illegal:
        off = torch.rand((n, k), generator=g, device="cuda") < illegal
        off.scatter_(1, y[:, None], False)
        z.masked_fill_(off, -float("inf"))
    return z.to(getattr(torch, dtype)), y


def _rows(k):
    return 300 if k <= 64 else 37 if k <= 5000 else 5


def _case(k, dtype, n=None, illegal=0.0, scale=2.0):
    import torch

    n = n or _rows(k)
    print(f"case n={n} k={k} {dtype} illegal={illegal}", flush=True)
    g = _rng(k, dtype, n, illegal)
    z, y = _margins(g, n, k, dtype, scale, illegal)
    lp = torch.log_softmax(z.double(), 1).gather(1, y[:, None])[:, 0]
    # on any side of the clip's borders (rows next to one: the border tests)
    old = (lp - torch.randn(n, generator=g, device="cuda") * 0.15).float()
    reference = (lp + torch.randn(n, generator=g, device="cuda") * 0.2).float()
    adv = torch.randn(n, generator=g, device="cuda")
    weight = torch.rand(n, generator=g, device="cuda") + 0.5
    return z, y, old, adv, weight, reference


def _check_policy(out, z, y, old, adv, weight, reference, clip=(0.2, 0.2), kl=0.0, entropy=0.0):
    rows = ref64.Rows(z, y, weight)
    loss, k3, c, n = ref64.policy(rows, old, adv, reference, clip[0], clip[1], kl, entropy)
    off = rows.logp_bound()
    a = np.abs(adv.cpu().double().numpy())
    with np.errstate(over="ignore", invalid="ignore"):
        ratio = np.exp(np.minimum(rows.logp - old.cpu().double().numpy(), 50.0))
    ref64.close(out.logp, rows.keep(rows.logp), off, "logp")
    ref64.close(out.entropy, rows.keep(rows.h), rows.h_bound(), "entropy")
    k_off = np.zeros_like(off)
    if reference is not None:
        with np.errstate(over="ignore", invalid="ignore"):
            d = reference.cpu().double().numpy() - rows.logp
        k_off = rows.keep(np.where(np.isfinite(d), np.abs(np.expm1(np.minimum(d, 50))), 0) * off
                          + np.abs(np.where(np.isfinite(k3), k3, 0)) * 2.0 ** -20 + 1e-12)
        ref64.close(out.kl, k3, k_off, "kl")
    loss_off = rows.w * (a * np.maximum(ratio, 1.3) * (off + 2.0 ** -20) + kl * k_off
                         + entropy * rows.h_bound()) + np.abs(loss) * 2.0 ** -22
    ref64.close(out.loss, loss, rows.keep(loss_off), "loss")
    if out.grad is not None:
        g, g_off = rows.grad(c, n)
        slope_off = rows.w * (a * ratio * off + kl * (off * 2 + 2.0 ** -20))
        ref64.close(out.grad, g, g_off + rows.keep(slope_off)[:, None], "grad")
    if out.hess is not None:
        h, h_off = rows.hess(c, n)
        ref64.close(out.hess, h, h_off + rows.keep(slope_off)[:, None], "hess")


# ---------------------------------------------------------------------------
# Log-probabilities
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", CLASSES + LONG)
def test_action_logprobs(ws, device, k, dtype):
    import torch
    from dpgbdt import ops

    z, y, *_ = _case(k, dtype, illegal=0.2)
    y[1] = -1
    y[3] = k
    z[1] = float("nan")
    logp, none = ops.action_logprobs(ws, z, y)
    both, h = ops.action_logprobs(ws, z, y.int(), entropy=True)
    rows = ref64.Rows(z, y)
    assert none is None and torch.equal(logp, both)
    ref64.close(logp, rows.keep(rows.logp), rows.logp_bound(), "logp")
    ref64.close(h, rows.keep(rows.h), rows.h_bound(), "entropy")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", CLASSES + LONG)
def test_action_logprobs_backward(ws, device, k, dtype):
    import torch
    from dpgbdt import ops

    z, y, dlogp, dent, *_ = _case(k, dtype, illegal=0.2)
    y[2] = -5
    z[2] = float("nan")
    rows = ref64.Rows(z, y)
    for dentropy in (None, dent):
        grad = ops.action_logprobs_backward(ws, z, y, dlogp, dentropy)
        n = np.zeros(rows.n) if dentropy is None else -dentropy.cpu().double().numpy()
        g, off = rows.grad(rows.keep(dlogp.cpu().double().numpy()), rows.keep(n))
        assert grad.dtype == z.dtype and grad.is_contiguous()
        ref64.close(grad, g, off, "grad")


# ---------------------------------------------------------------------------
# Policy loss
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", CLASSES + LONG)
def test_policy_loss(ws, device, k, dtype):
    import torch
    from dpgbdt import ops

    z, y, old, adv, weight, reference = _case(k, dtype, illegal=0.2)
    weight[1], y[2] = 0.0, -1
    z[1] = z[2] = float("nan")
    fp32 = dtype == "float32"
    out = ops.policy_loss(ws, z, y, old, adv, weight, reference, kl=0.05, entropy=0.01,
                          hessian=fp32)
    assert (out.hess is not None) == fp32
    _check_policy(out, z, y, old, adv, weight, reference, kl=0.05, entropy=0.01)
    again = ops.policy_loss(ws, z, y, old, adv, weight, reference, kl=0.05, entropy=0.01,
                            hessian=fp32)
    for a, b in zip(out, again):
        assert a is None and b is None or torch.equal(a, b)


@pytest.mark.parametrize("k", [1, 4, 10, 33, 300, 5000])
def test_policy_loss_without_its_options(ws, device, k):
    from dpgbdt import ops

    z, y, old, adv, weight, reference = _case(k, "float32")
    one = weight * 0 + 1
    out = ops.policy_loss(ws, z, y, old, adv, clip_high=0.28)
    assert out.kl is None and out.hess is None
    _check_policy(out, z, y, old, adv, one, None, clip=(0.2, 0.28))
    out = ops.policy_loss(ws, z, y, old, adv, reference=reference, clip_low=1.0, gradient=False)
    assert out.grad is None
    _check_policy(out, z, y, old, adv, one, reference, clip=(1.0, 0.2))


@pytest.mark.parametrize("n", [1, 2, 63, 255, 256, 257, 1023, 5000])
@pytest.mark.parametrize("k", [1, 5, 10, 12, 48, 130])
def test_row_counts(ws, device, n, k):
    from dpgbdt import ops

    z, y, old, adv, weight, reference = _case(k, "float32", n=n)
    out = ops.policy_loss(ws, z, y, old, adv, weight, reference, kl=0.1, entropy=0.02,
                          hessian=True)
    _check_policy(out, z, y, old, adv, weight, reference, kl=0.1, entropy=0.02)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,wide,first", [(5, 9, 1), (10, 13, 3), (64, 64, 0), (100, 200, 7),
                                          (513, 1001, 5), (3000, 3001, 1), (20000, 20008, 8)])
def test_strided_rows(ws, device, k, wide, first, dtype):
    """Columns of a wider matrix: rows apart, starts at any element of a vector."""
    import torch
    from dpgbdt import ops

    z, y, old, adv, weight, reference = _case(k, dtype)
    whole = torch.full((len(z), wide), float("nan"), dtype=z.dtype, device="cuda")
    whole[:, first:first + k] = z
    view = whole[:, first:first + k]
    out = ops.policy_loss(ws, view, y, old, adv, weight, reference, kl=0.05, entropy=0.01,
                          hessian=dtype == "float32")
    _check_policy(out, z, y, old, adv, weight, reference, kl=0.05, entropy=0.01)
    logp, _ = ops.action_logprobs(ws, view, y)
    assert torch.equal(logp, out.logp)


@pytest.mark.parametrize("k", [10, 900, 40000])
def test_border_of_the_clip_as_in_64_bits(ws, device, k):
    """Old log-probabilities that put the ratio next to its border, nearer than 32 bits tell."""
    import torch
    from dpgbdt import ops

    n = 2000 if k == 10 else 64
    z, y, old, adv, weight, reference = _case(k, "float32", n=n)
    lp = torch.log_softmax(z.double(), 1).gather(1, y[:, None])[:, 0]
    border = torch.where(adv > 0, np.log1p(0.2), np.log1p(-0.2))
    old = (lp - border).float()  # within a rounding of the border, on either side
    out = ops.policy_loss(ws, z, y, old, adv)
    rows = ref64.Rows(z, y)
    up = adv.cpu().numpy() > 0
    gap = (rows.logp - old.cpu().double().numpy()) - np.where(up, np.log1p(0.2), np.log1p(-0.2))
    active = np.where(up, gap < 0, gap > 0)
    clear = np.abs(gap) > 1e-12  # nearer, 64 bits do not tell either
    assert 0.2 < active.mean() < 0.8 and clear.mean() > 0.99
    assert np.array_equal((out.grad.abs().sum(1).cpu().numpy() > 0)[clear], active[clear])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [4, 40, 600, 20000])
def test_rows_with_nothing_and_extreme_margins(ws, device, k, dtype):
    import torch
    from dpgbdt import ops

    z, y, old, adv, weight, reference = _case(k, dtype, n=12)
    low = torch.finfo(z.dtype).min
    z[0] = -float("inf")               # no class at all
    z[1] = low                         # every class at the type's lowest value: uniform
    z[2, :] = low
    z[2, y[2]] = 1.0                   # all but the taken one
    z[3, y[3]] = -float("inf")         # the taken class has probability 0
    z[4, 0] = float("nan")
    z[5] = 60000.0                     # far from 0
    z[5, y[5]] = 59000.0
    z[6, y[6]] = 300.0                 # certain
    old[1] = -np.log(k)
    old[5] = -900.0
    out = ops.policy_loss(ws, z, y, old, adv, weight, reference, kl=0.05, entropy=0.01)
    rows = ref64.Rows(z, y, weight)
    assert out.logp[3] == -float("inf")
    assert not any(x[0].any() for x in out if x is not None)  # not counted
    g, off = rows.grad(*ref64.policy(rows, old, adv, reference, 0.2, 0.2, 0.05, 0.01)[2:])
    assert out.grad[4].isnan().all() and out.loss[4].isnan() and out.logp[4].isnan()
    some = [i for i in range(12) if i not in (3, 4, 5)]
    slope = (weight * (adv.abs() * 1.3 + 1)).cpu().double().numpy()[:, None] * 2.0 ** -18
    ref64.close(out.grad[some], g[some], (off + slope)[some], "grad")
    ref64.close(out.logp[some], rows.keep(rows.logp)[some], rows.logp_bound()[some], "logp")
    plain = ops.action_logprobs_backward(ws, z, y, adv, reference)
    g, off = rows.grad(adv.cpu().double().numpy(), -reference.cpu().double().numpy())
    some = [0, 1, 2, 3, 6]
    ref64.close(plain[some], rows.keep(g)[some], off[some], "backward")
    pairs = ops.preference_loss(ws, z, y, torch.tensor([0, 3, 3], device="cuda"), average=True)
    _check_preference_sums(pairs, rows.logp[1:3].mean())


def _check_preference_sums(out, mean):
    assert abs(out.score[0].item() - 0.1 * mean) <= 0.1 * (2.0 ** -19 + abs(mean) * 2.0 ** -23)
    assert not out.grad[0].any() and out.grad[1].any()


def test_policy_gradient_is_the_slope_of_the_loss(ws, device):
    """Differences of the 64-bit loss against the kernel's gradient."""
    from dpgbdt import ops

    z, y, old, adv, weight, reference = _case(6, "float32", n=40)
    out = ops.policy_loss(ws, z, y, old, adv, weight, reference, kl=0.3, entropy=0.2)

    def losses(m):
        rows = ref64.Rows(m, y, weight)
        return ref64.policy(rows, old, adv, reference, 0.2, 0.2, 0.3, 0.2)[0]

    got, step = out.grad.cpu().double().numpy(), 1e-4
    rows = ref64.Rows(z, y)
    ratio = np.exp(rows.logp - old.cpu().double().numpy())
    clear = (np.abs(ratio - 1.2) > 0.01) & (np.abs(ratio - 0.8) > 0.01)
    assert clear.sum() > 30
    for k in range(6):
        up, down = z.double().cpu(), z.double().cpu()
        up[:, k] += step
        down[:, k] -= step
        slope = (losses(up) - losses(down)) / (2 * step)
        # the third derivative over 6 times step^2, and the kernel's own bound
        assert np.abs(slope - got[:, k])[clear].max() < 1e-6 * (1 + np.abs(got).max()) * 3


# rows of each number of vectors a lane, whole and odd, on both sides of every change of kernel
GROUPS = [17, 24, 32, 33, 48, 63, 66, 95, 127, 129, 191, 193, 255, 256, 258, 300, 384, 385, 511,
          513, 700, 769, 800, 1023, 1024, 1025, 1500, 2047, 2048, 2049, 2200, 2900, 3200, 3600,
          4095, 4096, 4097]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", GROUPS)
def test_rows_of_a_wave(ws, device, k, dtype):
    import torch
    from dpgbdt import ops

    z, y, old, adv, weight, reference = _case(k, dtype, n=301 if k < 300 else 75, illegal=0.1)
    y[::5] = k - 1  # the end of a row, which may be held twice
    weight[7], y[8] = 0.0, -1
    z[7] = z[8] = float("nan")
    z[9] = -float("inf")
    old = torch.log_softmax(z.double(), 1).gather(1, y.clamp(min=0)[:, None])[:, 0]
    old = (old.nan_to_num(0.0, 0.0, -20.0) - 0.05).float()
    out = ops.policy_loss(ws, z, y, old, adv, weight, reference, kl=0.05, entropy=0.01,
                          hessian=dtype == "float32")
    some = [i for i in range(len(z)) if z[i, y[i]] != -float("inf")]
    assert not any(x[7:10].any() for x in out if x is not None)
    pick = type(out)(*(x if x is None else x[some] for x in out))
    _check_policy(pick, z[some], y[some], old[some], adv[some], weight[some], reference[some],
                  kl=0.05, entropy=0.01)
    logp, h = ops.action_logprobs(ws, z, y, entropy=True)
    counted = (weight != 0)
    assert torch.equal(logp[counted], out.logp[counted])
    assert torch.equal(h[counted], out.entropy[counted])


@pytest.mark.parametrize("k", [2, 10, 32, 40, 300, 1000, 5000, 20000, 40000])
def test_log_probabilities_next_to_zero(ws, device, k):
    """A class that has almost everything: what is beside it decides, to its own precision."""
    import torch
    from dpgbdt import ops

    g = _rng(k, "near")
    z = torch.randn((40, k), generator=g, device="cuda") - 14.0 - float(np.log(k))
    y = torch.randint(k, (40,), generator=g, device="cuda")
    z.scatter_(1, y[:, None], 0.0)
    logp, _ = ops.action_logprobs(ws, z, y)
    want = torch.log_softmax(z.double(), 1).gather(1, y[:, None])[:, 0]
    assert want.max() < 0 and want.min() > -1e-4
    # exponentials are off by (|x| + 3) 2^-24 with |x| of up to 40 in powers of two, the sum's
    # logarithm and its rounding by 2^-23
    assert ((logp.double() - want).abs() <= want.abs() * (45 * 2.0 ** -24 + 2.0 ** -22)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [3, 10, 31, 33, 63, 130, 300, 513, 1030, 2050, 9001, 33001, 70001])
def test_nothing_outside_the_rows(dp, ws, device, k, dtype):
    """Margins between NaN and outputs between marks: neither is read nor written."""
    import ctypes

    import torch

    n, edge = 13, 64
    z, y, old, adv, weight, reference = _case(k, dtype, n=n)

    def between(*shape, dtype=torch.float32, mark=float("nan")):
        count = int(np.prod(shape))
        whole = torch.full((count + 2 * edge,), mark, dtype=dtype, device="cuda")
        return whole, whole[edge + 1:edge + 1 + count].view(shape)

    held, zz = between(n, k, dtype=z.dtype)
    zz.copy_(z)
    code = {"float32": 0, "float16": 1, "bfloat16": 2}[dtype]
    d = dp.Decisions(zz.data_ptr(), y.data_ptr(), n, k, k, code, 8)
    param = dp.PolicyParam(0.2, 0.2, 0.05, 0.01)
    outs = [between(n, mark=7.0) for _ in range(4)] + [between(n, k, dtype=z.dtype, mark=7.0)]
    hess = between(n, k, mark=7.0)
    ptr = [o[1].data_ptr() for o in outs]
    dp.check(dp.load().dp_policy_loss(
        ws.handle, ctypes.byref(d), old.data_ptr(), adv.data_ptr(), weight.data_ptr(),
        reference.data_ptr(), ctypes.byref(param), *ptr,
        hess[1].data_ptr() if dtype == "float32" else None,
        torch.cuda.current_stream().cuda_stream))
    for whole, inner in outs + [hess]:
        count = inner.numel()
        assert (whole[:edge + 1] == 7.0).all() and (whole[edge + 1 + count:] == 7.0).all()
    from dpgbdt import ops

    want = ops.policy_loss(ws, z, y, old, adv, weight, reference, kl=0.05, entropy=0.01,
                           hessian=dtype == "float32")
    got = [o[1] for o in outs] + ([hess[1]] if dtype == "float32" else [])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# Preference loss
# ---------------------------------------------------------------------------
def _check_preference(out, z, y, ptr, reference, beta, smoothing, average):
    rows = ref64.Rows(z, y)
    score, loss, c = ref64.preference(rows, ptr, reference, beta, smoothing, average)
    off = rows.logp_bound()
    edges = np.clip(ptr.cpu().numpy(), 0, rows.n)
    share = np.ones(len(edges) - 1)
    if average:
        share = 1.0 / np.maximum([rows.counted[b:e].sum() for b, e in zip(edges, edges[1:])], 1)
    sums = np.array([off[b:e].sum() for b, e in zip(edges, edges[1:])]) * share
    s_off = beta * (sums[0::2] + sums[1::2])
    ref64.close(out.logp, rows.keep(rows.logp), off, "logp")
    ref64.close(out.score, score, s_off, "score")
    ref64.close(out.loss, loss, s_off + 1e-7, "loss")
    if out.grad is not None:
        g, g_off = rows.grad(c, np.zeros(rows.n))
        slope = np.zeros(rows.n)
        for i in range(len(score)):
            for j in (2 * i, 2 * i + 1):
                slope[edges[j]:edges[j + 1]] = beta * s_off[i] * share[j]
        ref64.close(out.grad, g, g_off + rows.keep(slope)[:, None], "grad")
        if out.hess is not None:
            h, h_off = rows.hess(c, np.zeros(rows.n))
            ref64.close(out.hess, h, h_off + rows.keep(slope)[:, None], "hess")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1, 2, 10, 33, 64, 100, 700, 2056, 9001, 33001, 70001])
@pytest.mark.parametrize("average", [False, True])
def test_preference_loss(ws, device, k, dtype, average):
    import torch
    from dpgbdt import ops

    z, y, _, _, _, reference = _case(k, dtype, illegal=0.1)
    n = len(z)
    y[::7] = -1
    z[::7] = float("nan")
    cuts = sorted(np.random.RandomState(k).randint(0, n + 1, 7).tolist())
    ptr = torch.tensor([min(1, n)] + cuts + [n], device="cuda").sort()[0]
    hess = dtype == "float32"
    for smoothing, r in ((0.0, reference), (0.2, None)):
        out = ops.preference_loss(ws, z, y, ptr, r, beta=0.3, smoothing=smoothing,
                                  average=average, hessian=hess)
        _check_preference(out, z, y, ptr, r, 0.3, smoothing, average)


@pytest.mark.parametrize("n,pairs", [(5000, 1), (5000, 700), (3, 40), (20000, 2000)])
def test_preference_sequences(ws, device, n, pairs):
    """One long pair, many short ones, more sequences than rows (most of them empty)."""
    import torch
    from dpgbdt import ops

    z, y, _, _, _, reference = _case(10, "float32", n=n)
    inner = np.sort(np.random.RandomState(n).randint(0, n + 1, 2 * pairs - 1))
    ptr = torch.tensor([0] + inner.tolist() + [n], device="cuda")
    out = ops.preference_loss(ws, z, y, ptr, reference, hessian=True)
    _check_preference(out, z, y, ptr, reference, 0.1, 0.0, False)
    none = ops.preference_loss(ws, z, y, ptr, reference, gradient=False)
    assert none.grad is None and torch.equal(none.loss, out.loss)


def test_preference_offsets_outside_are_cut_and_no_pairs(ws, device):
    import torch
    from dpgbdt import ops

    z, y, _, _, _, reference = _case(10, "float32", n=50)
    ptr = torch.tensor([-4, 20, 80], device="cuda")
    out = ops.preference_loss(ws, z, y, ptr, reference)
    _check_preference(out, z, y, ptr, reference, 0.1, 0.0, False)
    out = ops.preference_loss(ws, z, y, ptr[:1], reference)
    assert len(out.loss) == 0 and not out.grad.any()
    out = ops.preference_loss(ws, z[:0], y[:0], ptr * 0, reference[:0])
    assert abs(out.loss[0].item() - np.log(2)) < 1e-7 and out.grad.shape == (0, 10)


def test_certain_preferences_stay_finite(ws, device):
    import torch
    from dpgbdt import ops

    z = torch.zeros((4, 3), device="cuda")
    z[:2, 0] = 1000.0
    z[2:, 0] = -1000.0
    y = torch.zeros(4, dtype=torch.int64, device="cuda")
    for order, want in (([0, 2, 4], 0.0), ([0, 2, 4], None)):
        zz = z if want is not None else z.flip(0)
        out = ops.preference_loss(ws, zz, y, torch.tensor(order, device="cuda"), beta=1.0)
        _check_preference(out, zz, y, torch.tensor(order), None, 1.0, 0.0, False)
        assert torch.isfinite(out.grad).all()


# ---------------------------------------------------------------------------
# Recurrences
# ---------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (3, 1, 5), (300, 1, 1), (2, 2, 3), (1, 7, 64), (64, 100, 1), (5, 63, 65),
          (2, 257, 130), (1, 1000, 1), (7, 1023, 1), (3, 4097, 2), (2, 5000, 33), (1, 70001, 1),
          (2, 20011, 3), (1, 3001, 520), (600, 33, 8), (4, 1025, 2048), (1, 600000, 1)]


def _scan_case(shape, dtype):
    import torch

    print(f"case {shape} {dtype}", flush=True)
    g = _rng(*shape, dtype)
    b, t, c = shape
    dt = getattr(torch, dtype)
    gate = torch.sigmoid(torch.randn(shape, generator=g, device="cuda") + 3)
    gate[torch.rand(shape, generator=g, device="cuda") < 0.01] = 0.0
    gate[torch.rand(shape, generator=g, device="cuda") < 0.01] = -0.9
    value = torch.randn(shape, generator=g, device="cuda")
    ends = torch.randn((2, b, c), generator=g, device="cuda")
    return gate.to(dt), value.to(dt), ends[0], ends[1]


def _np(x):
    return x.detach().cpu().double().numpy()


def _check_recurrence(ws, gate, value, initial, dlast, reverse):
    import torch
    from dpgbdt import ops

    zero = np.zeros((gate.shape[0], gate.shape[2]))
    start = zero if initial is None else _np(initial)
    state, last = ops.linear_recurrence(ws, gate, value, initial, reverse=reverse)
    want, end, off, off_end = ref64.recurrence(_np(gate), _np(value), start, reverse)
    assert state.dtype == value.dtype and last.dtype == torch.float32
    ref64.close(state, want, off, "state")
    ref64.close(last, end, off_end, "last")
    dstate = value.flip(0)
    outs = ops.linear_recurrence_backward(ws, gate, state, dstate, initial, dlast, reverse)
    want, off = ref64.recurrence_backward(_np(gate), _np(state), _np(dstate), start,
                                          zero if dlast is None else _np(dlast), reverse)
    for got, w, o, name in zip(outs, want, off, ("dgate", "dvalue", "dinitial")):
        ref64.close(got, w, o, name)
    for got, again in zip(outs, ops.linear_recurrence_backward(ws, gate, state, dstate, initial,
                                                               dlast, reverse)):
        assert torch.equal(got, again)
    return state, last


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_recurrence(ws, device, shape, dtype, reverse):
    gate, value, initial, dlast = _scan_case(shape, dtype)
    if shape[0] * shape[1] * shape[2] > 1 << 21 and dtype == "float16":
        gate, value, initial, dlast = (x[..., :8] for x in (gate, value, initial, dlast))
        initial, dlast = initial.contiguous(), dlast.contiguous()
    _check_recurrence(ws, gate, value, initial, dlast, reverse)


@pytest.mark.parametrize("shape", [(3, 1, 5), (64, 100, 1), (2, 5000, 33), (1, 70001, 1)])
def test_recurrence_from_nothing(ws, device, shape):
    gate, value, _, _ = _scan_case(shape, "float32")
    _check_recurrence(ws, gate, value, None, None, False)
    _check_recurrence(ws, gate, value, None, None, True)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("b,t,c", [(50, 1000, 1), (700, 40, 1), (3, 5000, 1), (4, 3000, 6),
                                   (3, 700, 40)])
def test_recurrence_orders_and_strides(ws, device, b, t, c, dtype, reverse):
    """Time-major arrays, gaps between steps, channels off a wider array, an expanded gate."""
    import torch

    gate, value, initial, dlast = _scan_case((b, t, c), dtype)
    want, last = _check_recurrence(ws, gate, value, initial, dlast, reverse)

    def major(x):
        return x.transpose(0, 1).contiguous().transpose(0, 1)

    def apart(x):
        whole = torch.full((b, t, c + 3), float("nan"), dtype=x.dtype, device="cuda")
        whole[..., 1:1 + c] = x
        return whole[..., 1:1 + c]

    for f, g in ((major, major), (apart, apart), (major, apart), (lambda x: x, major)):
        _check_recurrence(ws, f(gate), g(value), initial, dlast, reverse)
    state, _ = _check_recurrence(ws, gate[:1].expand(b, t, c), major(value), initial, dlast,
                                 reverse)
    _check_recurrence(ws, gate[:, :1].expand(b, t, c), value, initial, dlast, reverse)


@pytest.mark.parametrize("shape", [(0, 5, 3), (2, 5, 0), (2, 0, 3)])
def test_recurrence_of_nothing(ws, device, shape):
    import torch
    from dpgbdt import ops

    b, t, c = shape
    x = torch.zeros(shape, device="cuda")
    start = torch.randn((b, c), device="cuda")
    state, last = ops.linear_recurrence(ws, x, x, start)
    assert state.shape == shape and torch.equal(last, start)
    _, last = ops.linear_recurrence(ws, x, x)
    assert not last.any()
    _, _, dinitial = ops.linear_recurrence_backward(ws, x, x, x, start, start)
    assert torch.equal(dinitial, start)


def test_recurrence_steps_join(ws, device):
    """Single steps from the last state, and pieces, are the whole."""
    import torch
    from dpgbdt import ops

    gate, value, initial, _ = _scan_case((40, 33, 70), "float32")
    want, last, off, _ = ref64.recurrence(_np(gate), _np(value), _np(initial), False)
    h = initial
    for t in range(33):
        s, h = ops.linear_recurrence(ws, gate[:, t:t + 1], value[:, t:t + 1], h)
        ref64.close(s[:, 0], want[:, t], off[:, t], f"step {t}")
    ref64.close(h, last, off[:, -1], "last")


@pytest.mark.parametrize("b,t,c", [(6, 3000, 1), (5, 200, 1), (3, 5000, 7), (3, 2000, 64)])
def test_what_is_not_finite_stays_in_its_sequence(ws, device, b, t, c):
    import torch
    from dpgbdt import ops

    gate, value, initial, _ = _scan_case((b, t, c), "float32")
    clean, last = ops.linear_recurrence(ws, gate, value, initial)
    value = value.clone()
    value[1, t // 2, 0] = float("nan")
    value[b - 1, 1, c - 1] = float("inf")
    state, end = ops.linear_recurrence(ws, gate, value, initial)
    assert state[1, t // 2, 0].isnan() and torch.equal(state[0], clean[0])
    assert torch.equal(end[0], last[0])
    assert torch.equal(state[1, :t // 2], clean[1, :t // 2])
    back, end = ops.linear_recurrence(ws, gate, value, initial, reverse=True)
    assert back[0].isfinite().all() and back[1, t // 2 + 1:].isfinite().all()
    assert back[1, t // 2, 0].isnan()
    if c > 1:
        assert torch.equal(state[1, :, 1:], clean[1, :, 1:])


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(5, 8, 13), (4, 3, 70), (7, 5, 9), (6, 2, 4), (3, 9, 5),
                                   (2, 127, 64), (1, 128, 64), (2, 129, 97), (40, 130, 3),
                                   (300, 140, 20), (20, 150, 31), (2, 385, 256), (1, 20000, 64),
                                   (9, 4099, 1), (130, 33, 1), (130, 9, 1), (1, 16385, 1),
                                   (2100, 16, 130), (1100, 11, 256), (1, 16, 70)])
def test_recurrence_layouts(ws, device, shape, dtype, reverse):
    """Every layout of lanes over steps and channels, its last block whole and not, and splits."""
    gate, value, initial, dlast = _scan_case(shape, dtype)
    _check_recurrence(ws, gate, value, initial, dlast, reverse)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,c", [(2, 700, 67), (3, 5, 11), (1, 5000, 1), (70, 40, 3),
                                   (1, 9000, 96)])
def test_recurrence_writes_nothing_outside(dp, ws, device, b, t, c, dtype):
    import ctypes

    import torch

    gate, value, initial, dlast = _scan_case((b, t, c), dtype)
    edge, count = 64, b * t * c

    def between(x=None, mark=float("nan")):
        whole = torch.full((count + 2 * edge,), mark, dtype=gate.dtype, device="cuda")
        inner = whole[edge + 1:edge + 1 + count].view(b, t, c)
        if x is not None:
            inner.copy_(x)
        return whole, inner

    from dpgbdt import ops

    code = {"float32": 0, "float16": 1, "bfloat16": 2}[dtype]
    for reverse in (False, True):
        shape = dp.Recurrence(b, t, c, code, reverse)
        for i in range(5):
            shape.strides[i][0], shape.strides[i][1] = t * c, c
        (_, g), (_, v) = between(gate), between(value)
        out, da, dv = (between(mark=7.0) for _ in range(3))
        stream = torch.cuda.current_stream().cuda_stream
        last, dinitial = torch.empty((2, b, c), device="cuda").unbind()
        dp.check(dp.load().dp_linear_recurrence(
            ws.handle, ctypes.byref(shape), g.data_ptr(), v.data_ptr(), initial.data_ptr(),
            out[1].data_ptr(), last.data_ptr(), stream))
        state, end = ops.linear_recurrence(ws, gate, value, initial, reverse=reverse)
        (_, s) = between(state)
        dp.check(dp.load().dp_linear_recurrence_backward(
            ws.handle, ctypes.byref(shape), g.data_ptr(), s.data_ptr(), v.data_ptr(),
            initial.data_ptr(), dlast.data_ptr(), da[1].data_ptr(), dv[1].data_ptr(),
            dinitial.data_ptr(), stream))
        want = ops.linear_recurrence_backward(ws, gate, state, value, initial, dlast, reverse)
        got = [out[1], last, da[1], dv[1], dinitial]
        for x, w in zip(got, [state, end, *want]):
            assert torch.equal(x, w)
        for whole, _ in (out, da, dv):
            assert (whole[:edge + 1] == 7.0).all() and (whole[edge + 1 + count:] == 7.0).all()


# ---------------------------------------------------------------------------
# Streams, graphs, far offsets
# ---------------------------------------------------------------------------
def _everything(ws, z, y, old, adv, weight, reference, ptr, gate, value, initial):
    from dpgbdt import ops

    a = ops.policy_loss(ws, z, y, old, adv, weight, reference, kl=0.05, entropy=0.01)
    b = ops.preference_loss(ws, z, y, ptr, reference)
    c = ops.action_logprobs(ws, z, y, entropy=True)
    s, last = ops.linear_recurrence(ws, gate, value, initial, reverse=True)
    d = ops.linear_recurrence_backward(ws, gate, s, value, initial, last, reverse=True)
    return [x for x in (*a, *b, *c, s, last, *d) if x is not None]


@pytest.mark.parametrize("k,n,shape", [(10, 3000, (40, 300, 1)), (40000, 20, (2, 5000, 96)),
                                       (700, 200, (1, 200000, 1))])
def test_graph_replays_and_streams(device, k, n, shape):
    import torch
    from dpgbdt import ops

    ws = ops.Workspace()
    z, y, old, adv, weight, reference = _case(k, "float32", n=n)
    ptr = torch.arange(0, n + 1, n // 20, device="cuda")
    ptr = ptr[:len(ptr) - (len(ptr) + 1) % 2].contiguous()
    gate, value, initial, _ = _scan_case(shape, "float32")
    args = [z, y, old, adv, weight, reference, ptr, gate, value, initial]
    want = [x.clone() for x in _everything(ws, *args)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _everything(ws, *args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _everything(ws, *args)
    for i in range(4):
        for x in outs:
            x.zero_()
        adv.mul_(-1.0)
        value.mul_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        eager = [x.clone() for x in _everything(ws, *args)]  # between replays, same workspace
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), i
    assert all(torch.equal(a, b) for a, b in zip(outs, want))  # four changes of sign


def test_offsets_beyond_32_bits(ws, device):
    import torch
    from dpgbdt import ops

    far = (1 << 31) + 24
    whole = torch.empty(2 * far + 40000, dtype=torch.bfloat16, device="cuda")
    for k in (10, 700, 40000):
        z, y, old, adv, weight, reference = _case(k, "bfloat16", n=3)
        view = whole.as_strided((3, k), (far, 1))
        view.copy_(z)
        out = ops.policy_loss(ws, view, y, old, adv, weight, reference, kl=0.05)
        want = ops.policy_loss(ws, z, y, old, adv, weight, reference, kl=0.05)
        assert all(torch.equal(a, b) for a, b in zip(out[:5], want[:5]))
    for c in (1, 5, 512):
        gate, value, initial, _ = _scan_case((2, 3, c), "bfloat16")
        view = whole.as_strided((2, 3, c), (1024, far, 1))
        view.copy_(value)
        state, last = ops.linear_recurrence(ws, gate, view, initial)
        want, end = ops.linear_recurrence(ws, gate, value, initial)
        assert torch.equal(state, want) and torch.equal(last, end)


def test_trees_learn_from_the_losses(dp, device):
    """The example: the operators together with the booster they are for."""
    import os
    import sys

    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(dp.__file__)), "..",
                                    "examples"))
    import train_policy

    first, policy, preferences = train_policy.train(episodes=256, batches=8)
    assert 0.2 < first < 0.3  # four actions
    assert policy > 0.6 and preferences > policy - 0.02  # a sample of 2048 is off by 0.01


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def test_refusals(dp, ws, device):
    import torch
    from dpgbdt import ops

    z, y, old, adv, weight, reference = _case(10, "float32", n=8)
    ptr = torch.tensor([0, 4, 8], device="cuda")
    bad = [
        lambda: ops.action_logprobs(ws, z[0], y),
        lambda: ops.action_logprobs(ws, z.double(), y),
        lambda: ops.action_logprobs(ws, z.t(), y),
        lambda: ops.action_logprobs(ws, z, y[:4]),
        lambda: ops.action_logprobs(ws, z, y.float()),
        lambda: ops.action_logprobs(ws, z, y.cpu()),
        lambda: ops.action_logprobs(ws, z[:, :0], y),
        lambda: ops.action_logprobs_backward(ws, z, y, old.double()),
        lambda: ops.action_logprobs_backward(ws, z, y, old, adv[:3]),
        lambda: ops.policy_loss(ws, z, y, old[::2], adv),
        lambda: ops.policy_loss(ws, z, y, old, adv, clip_low=1.5),
        lambda: ops.policy_loss(ws, z, y, old, adv, clip_high=-0.1),
        lambda: ops.policy_loss(ws, z, y, old, adv, clip_high=float("inf")),
        lambda: ops.policy_loss(ws, z, y, old, adv, kl=0.1),
        lambda: ops.policy_loss(ws, z, y, old, adv, reference=reference, kl=float("nan")),
        lambda: ops.policy_loss(ws, z, y, old, adv, entropy=-1.0),
        lambda: ops.policy_loss(ws, z.half(), y, old, adv, hessian=True),
        lambda: ops.policy_loss(ws, z, y, old, adv, gradient=False, hessian=True),
        lambda: ops.preference_loss(ws, z, y, ptr.int()),
        lambda: ops.preference_loss(ws, z, y, ptr[:2]),
        lambda: ops.preference_loss(ws, z, y, ptr, beta=0.0),
        lambda: ops.preference_loss(ws, z, y, ptr, smoothing=1.5),
        lambda: ops.preference_loss(ws, z, y, ptr, reference=reference[:2]),
        lambda: ops.preference_loss(ws, z.bfloat16(), y, ptr, hessian=True),
        lambda: ops.linear_recurrence(ws, z, z),
        lambda: ops.linear_recurrence(ws, z[None], z[None, :4]),
        lambda: ops.linear_recurrence(ws, z[None], z[None].half()),
        lambda: ops.linear_recurrence(ws, z.t()[None], z.t()[None]),
        lambda: ops.linear_recurrence(ws, z[None], z[None], initial=z[0]),
        lambda: ops.linear_recurrence_backward(ws, z[None], z[None], z[None], dlast=z),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(dp.DPError):
            f()
            print("accepted:", i)
