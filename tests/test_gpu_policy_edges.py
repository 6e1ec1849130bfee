"""The operators over decisions where their inputs are special: references that rule the action
out, NaN among the rows' numbers, advantages of zero, certain preferences, rows of every kernel
next to the border of the clip, and how exact the losses are."""
import zlib

import numpy as np
import policy_reference as ref64
import pytest

pytestmark = pytest.mark.gpu


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
