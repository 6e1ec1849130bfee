"""The operators over decisions by their definitions, in 64 bits on the CPU, with bounds of
what 32-bit statistics and the output's rounding may be off by."""
import numpy as np
import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the distance between the numbers next to 0 (halves flush nothing)."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


class Rows:
    """Distributions of margins [n, K] (any device and dtype) for actions [n]."""

    def __init__(self, margin, action, weight=None):
        z = margin.detach().cpu().double().numpy()
        self.n, self.k = z.shape
        self.y = action.cpu().numpy().astype(np.int64)
        self.counted = (self.y >= 0) & (self.y < self.k)
        self.w = np.ones(self.n) if weight is None else weight.cpu().double().numpy()
        self.counted &= self.w != 0
        self.y = np.where(self.counted, self.y, 0)
        z = np.where(self.counted[:, None], z, 0.0)
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            m = z.max(axis=1, keepdims=True)
            self.counted &= ~(z == -np.inf).all(axis=1)
            d = z - np.where(m == -np.inf, 0.0, m)
            e = np.exp(d)
            s = e.sum(axis=1, keepdims=True)
            self.lp = np.where(s > 0, d - np.log(s), -np.inf)
            self.lp = np.where(np.isnan(s), np.nan, self.lp)
            self.p = np.where(s == 0, 0.0, e / s)
            self.inner = np.where(self.p == 0, 0.0, self.p * self.lp)
            self.h = -self.inner.sum(axis=1)
        self.logp = self.lp[np.arange(self.n), self.y]
        self.d = np.where(np.isfinite(d), np.abs(d), 0.0)

    def keep(self, v):
        return np.where(self.counted.reshape(-1, *[1] * (v.ndim - 1)), v, 0.0)

    def grad(self, c, n):
        """(gradient, its bound in 32 bits) for the slopes c of log p_y and n of -H."""
        taken = np.zeros((self.n, self.k))
        taken[np.arange(self.n), self.y] = 1.0
        c, n = c[:, None], n[:, None]
        with np.errstate(invalid="ignore"):
            tilt = np.where(self.p == 0, 0.0, self.p * (self.lp + self.h[:, None]))
            g = c * (taken - self.p) + n * tilt
            # p: its exponent is off by (|d| + 3) 2^-24 and s by 2^-20; the slopes by 2^-19
            rel = (self.d + 64.0) * 2.0 ** -23
            size = np.abs(np.where(self.p == 0, 0.0, self.inner)) + self.p * np.abs(
                self.h[:, None])
            bound = (np.abs(c) * (taken * 2.0 ** -19 + self.p * (rel + 2.0 ** -19))
                     + np.abs(n) * (size * (rel + 2.0 ** -19) + self.p * 2.0 ** -18))
        return self.keep(g), self.keep(bound)

    def hess(self, c, n):
        v = 2.0 * (np.abs(c) + np.abs(n))[:, None] * self.p * (1.0 - self.p)
        rel = (self.d + 64.0) * 2.0 ** -22 + 2.0 ** -18
        # 1 - p is off by p's own error
        bound = (2.0 * (np.abs(c) + np.abs(n))[:, None] * self.p * rel)
        return self.keep(np.maximum(v, 1e-16)), self.keep(bound)

    def logp_bound(self):
        """s is off by 2^-21 (partial sums of 32 bits), the result rounded once."""
        return self.keep(2.0 ** -20 + np.abs(np.where(np.isfinite(self.logp), self.logp, 0))
                         * 2.0 ** -24)

    def h_bound(self):
        return self.keep(2.0 ** -18 * (1.0 + np.abs(self.inner).sum(axis=1)))


def policy(rows, old, adv, ref, clip_low, clip_high, kl, entropy):
    old, adv = old.cpu().double().numpy(), adv.cpu().double().numpy()
    with np.errstate(over="ignore", invalid="ignore"):
        ratio = np.exp(rows.logp - old)
        plain = ratio * adv
        clipped = np.clip(ratio, 1 - clip_low, 1 + clip_high) * adv
        active = np.where(adv > 0, ratio < 1 + clip_high, ratio > 1 - clip_low)
        loss = -np.minimum(plain, clipped)
        c = np.where(active, -plain, 0.0)
        k3 = np.zeros_like(loss)
        if ref is not None:
            d = ref.cpu().double().numpy() - rows.logp
            k3 = np.expm1(d) - d
            loss = loss + kl * k3
            c = c - kl * np.expm1(d)
    loss = loss - entropy * rows.h
    n = entropy * rows.w
    return (rows.keep(loss * rows.w), rows.keep(k3), rows.keep(c * rows.w),
            rows.keep(n * np.ones(rows.n)))


def preference(rows, sequences, ref, beta, smoothing, average):
    """(score, loss, slopes of the rows)."""
    ptr = np.clip(sequences.cpu().numpy(), 0, rows.n)
    a = rows.keep(rows.logp - (0.0 if ref is None else ref.cpu().double().numpy()))
    total = np.array([a[b:e].sum() for b, e in zip(ptr[:-1], ptr[1:])])
    share = np.ones(len(total))
    if average:
        share = 1.0 / np.maximum([rows.counted[b:e].sum() for b, e in zip(ptr[:-1], ptr[1:])], 1)
    mean = total * share
    score = beta * (mean[0::2] - mean[1::2])
    loss = (1 - smoothing) * np.logaddexp(0, -score) + smoothing * np.logaddexp(0, score)
    with np.errstate(over="ignore"):
        slope = beta * (smoothing / (1 + np.exp(-score)) - (1 - smoothing) / (1 + np.exp(score)))
    c = np.zeros(rows.n)
    for i in range(len(score)):
        for j, sign in ((2 * i, 1), (2 * i + 1, -1)):
            c[ptr[j]:ptr[j + 1]] = sign * slope[i] * share[j]
    return score, loss, rows.keep(c)


def recurrence(gate, value, initial, reverse):
    """(states, last, bound of the states in 32 bits) step by step."""
    a, v = (np.asarray(x, dtype=np.float64) for x in (gate, value))
    if reverse:
        a, v = a[:, ::-1], v[:, ::-1]
    h = np.array(initial, dtype=np.float64)
    size, off = np.abs(h), np.zeros_like(h)
    out, bound = np.zeros_like(v), np.zeros_like(v)
    for t in range(v.shape[1]):
        h = a[:, t] * h + v[:, t]
        size = np.abs(a[:, t]) * size + np.abs(v[:, t])
        # a product and a sum a step, once more where spans are joined
        off = np.abs(a[:, t]) * off + 2.0 ** -21 * size
        out[:, t], bound[:, t] = h, off
    if reverse:
        out, bound = out[:, ::-1], bound[:, ::-1]
    return out, h, bound, off


def recurrence_backward(gate, state, dstate, initial, dlast, reverse):
    """(dgate, dvalue, dinitial) and their bounds."""
    a, s, x = (np.asarray(v, dtype=np.float64) for v in (gate, state, dstate))
    if reverse:
        a, s, x = a[:, ::-1], s[:, ::-1], x[:, ::-1]
    t = a.shape[1]
    if t == 0:
        return (np.zeros_like(a), np.zeros_like(a), dlast), (0.0, 0.0, 0.0)
    after = np.concatenate([a[:, 1:], np.ones_like(a[:, :1])], axis=1)
    before = np.concatenate([initial[:, None], s[:, :-1]], axis=1)
    g, end, off, off_end = recurrence(after, x, dlast, True)
    dgate = g * before
    outs = dgate, g, a[:, 0] * end
    bounds = (off * np.abs(before) + np.abs(dgate) * 2.0 ** -23, off,
              np.abs(a[:, 0]) * off_end + np.abs(outs[2]) * 2.0 ** -23)
    if reverse:
        outs = outs[0][:, ::-1], outs[1][:, ::-1], outs[2]
        bounds = bounds[0][:, ::-1], bounds[1][:, ::-1], bounds[2]
    return outs, bounds


def close(got, want, bound, what):
    """got (a tensor) is want (64 bits) within bound and one rounding to its type."""
    dtype = got.dtype
    x = got.detach().cpu().double().numpy()
    assert x.shape == want.shape, what
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(x), np.isnan(want)), what + ": NaN"
    special = ~fine & ~np.isnan(want)
    assert np.array_equal(x[special], want[special]), what + ": infinities"
    bound = np.broadcast_to(bound, want.shape)
    limit = (bound + np.abs(want) * half_step(dtype)) * 1.0001 + smallest(dtype)
    bad = fine & ~(np.abs(np.where(fine, x - want, 0.0)) <= limit)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off, first at {i}: {x[i]} for "
                             f"{want[i]}, bound {limit[i]}")
