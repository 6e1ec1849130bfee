"""What the operators over decisions refuse, without a GPU: through the Python binding on host
tensors, and through the C entry points on a HIP runtime in host memory."""
import pytest
from test_host_memory import host  # noqa: F401  (fixture)


def test_host_tensors_are_refused(dp):
    import torch
    from dpgbdt import ops

    z, y = torch.zeros((4, 3)), torch.zeros(4, dtype=torch.int64)
    x = torch.zeros((2, 3, 4))
    for call in (lambda: ops.action_logprobs(None, z, y),
                 lambda: ops.action_logprobs_backward(None, z, y, z[:, 0]),
                 lambda: ops.policy_loss(None, z, y, z[:, 0], z[:, 0]),
                 lambda: ops.preference_loss(None, z, y, y),
                 lambda: ops.linear_recurrence(None, x, x),
                 lambda: ops.linear_recurrence_backward(None, x, x, x)):
        with pytest.raises(dp.DPError, match="current device"):
            call()


SETUP = """
    from ctypes import *
    class Decisions(Structure):
        _fields_ = [("margin", c_void_p), ("action", c_void_p), ("n_rows", c_int64),
                    ("row_stride", c_int64), ("n_classes", c_int32), ("dtype", c_int32),
                    ("action_bytes", c_int32), ("pad", c_int32)]
    class Policy(Structure):
        _fields_ = [(n, c_double) for n in ("low", "high", "kl", "entropy")]
    class Preference(Structure):
        _fields_ = [("beta", c_double), ("smoothing", c_double), ("average", c_int32),
                    ("pad", c_int32)]
    class Recurrence(Structure):
        _fields_ = [("batch", c_int64), ("time", c_int64), ("channels", c_int64),
                    ("dtype", c_int32), ("reverse", c_int32), ("strides", (c_int64 * 2) * 5)]
    ws, P = c_void_p(), c_void_p(4096)
    ok(lib.dp_workspace_create(byref(ws)))
    def rows(**kw):
        d = dict(margin=4096, action=4096, n_rows=4, row_stride=3, n_classes=3, dtype=0,
                 action_bytes=8)
        d.update(kw)
        return byref(Decisions(**d))
    def said(status):
        return None if status == 0 else lib.XGBGetLastError().decode()
"""


def test_c_refusals_of_decisions(host):  # noqa: F811
    got = host(SETUP + """
    f = lambda d, w=ws: said(lib.dp_action_logprobs(w, d, P, None, None))
    bad = [rows(dtype=3), rows(action_bytes=2), rows(n_rows=-1), rows(n_classes=0),
           rows(row_stride=-1), rows(row_stride=2**61), rows(n_rows=2**61), rows(margin=None),
           rows(action=None), rows(margin=4097), None]
    out = [f(d) for d in bad] + [f(rows(), None)]
    out.append(said(lib.dp_action_logprobs(ws, rows(), None, None, None)))
    out.append(said(lib.dp_action_logprobs_backward(ws, rows(), None, None, P, None)))
    fake.hipSetDevice(1)
    out.append(f(rows()))
    fake.hipSetDevice(0)
    good = [f(rows()), f(rows(dtype=2, action_bytes=4)), f(rows(n_rows=0, margin=None))]
    print(json.dumps([out, good]))
    """)
    assert all(isinstance(m, str) and m for m in got[0]), got[0]
    assert "device 0" in got[0][-1]
    assert got[1] == [None, None, None]


def test_c_refusals_of_losses(host):  # noqa: F811
    got = host(SETUP + """
    def policy(d=None, low=0.2, high=0.2, kl=0.0, entropy=0.0, old=P, ref=None, k=None, grad=P,
               hess=None):
        return said(lib.dp_policy_loss(ws, d or rows(), old, P, None, ref,
                                       byref(Policy(low, high, kl, entropy)), P, None, k, None,
                                       grad, hess, None))
    def preference(d=None, beta=0.1, smoothing=0.0, pairs=2, seq=P, grad=P, hess=None):
        return said(lib.dp_preference_loss(ws, d or rows(), seq, c_int64(pairs), None,
                                           byref(Preference(beta, smoothing, 0)), P, None, None,
                                           grad, hess, None))
    nan = float("nan")
    bad = [policy(low=-0.1), policy(low=1.1), policy(low=nan), policy(high=-1.0),
           policy(high=float("inf")), policy(kl=0.1), policy(kl=-0.1, ref=P), policy(k=P),
           policy(entropy=nan), policy(hess=P, grad=None), policy(d=rows(dtype=1), hess=P),
           policy(old=None), preference(beta=0.0), preference(beta=nan), preference(smoothing=2.0),
           preference(pairs=-1), preference(pairs=2**31), preference(seq=None),
           preference(hess=P, grad=None), preference(d=rows(dtype=2), hess=P)]
    good = [policy(), policy(kl=0.1, ref=P, k=P, hess=P), preference(), preference(hess=P),
            preference(pairs=0, seq=None)]
    print(json.dumps([bad, good]))
    """)
    assert all(isinstance(m, str) and m for m in got[0]), got[0]
    assert got[1] == [None] * 5


def test_c_refusals_of_recurrences(host):  # noqa: F811
    got = host(SETUP + """
    def scan(batch=2, time=3, channels=4, dtype=0, stride=None, gate=P, back=False, w=ws):
        r = Recurrence(batch, time, channels, dtype, 0)
        for i in range(5):
            r.strides[i][0], r.strides[i][1] = stride or (12, 4)
        if back:
            return said(lib.dp_linear_recurrence_backward(w, byref(r), gate, P, P, None, None, P,
                                                          P, None, None))
        return said(lib.dp_linear_recurrence(w, byref(r), gate, P, None, P, None, None))
    bad = [f for b in (False, True) for f in (
        scan(batch=-1, back=b), scan(time=-1, back=b), scan(channels=-1, back=b),
        scan(channels=2**31, back=b), scan(batch=2**60, back=b), scan(dtype=7, back=b),
        scan(stride=(-1, 1), back=b), scan(stride=(1, -1), back=b), scan(stride=(2**62, 1), back=b),
        scan(gate=None, back=b), scan(w=None, back=b))]
    good = [f for b in (False, True) for f in (
        scan(back=b), scan(batch=0, gate=None, back=b), scan(time=0, gate=None, back=b),
        scan(stride=(0, 0), back=b))]
    print(json.dumps([bad, good]))
    """)
    assert all(isinstance(m, str) and m for m in got[0]), got[0]
    assert got[1] == [None] * 8
