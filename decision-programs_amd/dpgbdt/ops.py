"""Kernel-level operators of libdpgbdt_hip.so on torch device tensors.

Every function launches on torch's current stream of the tensors' device, so
torch.cuda.Event timing and ordering with torch work as usual.  Host arrays
(node segments) are numpy/int sequences.
"""
from __future__ import annotations

import collections
import ctypes
from ctypes import c_int32, c_void_p

import numpy as np

from . import BinLayout, Decisions, DPError, PolicyParam, PreferenceParam, Recurrence
from . import SplitRecord, TrainParam, check, load


class _Torch:
    """Stands for torch until it is first used: the package itself imports without it."""

    def __getattr__(self, name):
        import torch as module

        globals()["torch"] = module
        return getattr(module, name)


torch = _Torch()

SPLIT_DTYPE = np.dtype([("loss_chg", "<f8"), ("gl", "<i8"), ("hl", "<i8"), ("feature", "<i4"),
                        ("bin", "<i4"), ("default_left", "<i4"), ("valid", "<i4"),
                        ("expand", "<i4"), ("pad", "<i4")])
assert SPLIT_DTYPE.itemsize == ctypes.sizeof(SplitRecord)


def _stream():
    # torch.cuda.current_stream().cuda_stream without the objects on the way
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _ptr(t):
    return t.data_ptr() if t is not None else None


class Workspace:
    """Device scratch reused by the operator entry points, by one stream at a time.  A graph that
    calls were captured into uses it at every replay: keep it as long as the graph."""

    def __init__(self):
        self.handle = c_void_p()
        check(load().dp_workspace_create(ctypes.byref(self.handle)))

    def __del__(self):
        # load is None when the interpreter has taken the module down already
        if getattr(self, "handle", None) and load is not None:
            load().dp_workspace_free(self.handle)
            self.handle = None


def layout(n_rows, n_features, tile_width=0, missing_bin=-1):
    out = BinLayout()
    check(load().dp_layout_init(n_rows, n_features, tile_width, missing_bin, ctypes.byref(out)))
    return out


def layout_pair_tiles(lay, cut_ptr):
    """Pairs the layout's tiles whose features all have at most 16 bins (host cut_ptr, as
    sketch_cuts returns it); returns the layout (changed in place)."""
    ptr = np.ascontiguousarray(cut_ptr, dtype=np.int32)
    check(load().dp_layout_pair_tiles(ctypes.byref(lay), ptr.ctypes.data))
    return lay


def join_tiles(bins, lay):
    """Writes the joint tiles of a paired layout into device bins (after its n_tiles tiles)."""
    check(load().dp_join_tiles(_ptr(bins), ctypes.byref(lay), _stream()))
    return bins


def layout_bytes(lay):
    return load().dp_layout_bytes(ctypes.byref(lay))


def to_tiles(bins_rowmajor, lay):
    """Host row-major [n, F] uint8 -> tile-major bytes of `lay` (numpy)."""
    n, f = bins_rowmajor.shape
    tw, nt = lay.tile_width, lay.n_tiles
    pad = np.zeros((n, nt * tw), dtype=np.uint8)
    pad[:, :f] = bins_rowmajor
    return np.ascontiguousarray(pad.reshape(n, nt, tw).transpose(1, 0, 2)).reshape(-1)


def from_tiles(tiles, lay):
    """Tile-major bytes -> row-major [n, F] uint8 (numpy)."""
    n, f, tw, nt = lay.n_rows, lay.n_features, lay.tile_width, lay.n_tiles
    return np.ascontiguousarray(tiles.reshape(nt, n, tw).transpose(1, 0, 2).reshape(n, nt * tw)[:, :f])


def sketch_cuts(ws, values, max_bin):
    """Quantile cuts of a device [n, F] float32 tensor -> (cut_ptr, cut_values, mins, missing)."""
    n, f = values.shape
    cut_ptr = np.zeros(f + 1, dtype=np.int32)
    cuts = np.zeros(f * max_bin, dtype=np.float32)
    mins = np.zeros(f, dtype=np.float32)
    has_missing = c_int32()
    check(load().dp_sketch_cuts(ws.handle, _ptr(values), n, f, max_bin, cut_ptr.ctypes.data,
                                cuts.ctypes.data, mins.ctypes.data, ctypes.byref(has_missing),
                                _stream()))
    return cut_ptr, cuts[: cut_ptr[-1]].copy(), mins, bool(has_missing.value)


def bin_values(values, lay, cut_ptr, cut_values):
    """Device bins (tile-major uint8 tensor) of a device float32 matrix."""
    dev = values.device
    cp = torch.as_tensor(np.asarray(cut_ptr, dtype=np.int32), device=dev)
    cv = torch.as_tensor(np.asarray(cut_values, dtype=np.float32), device=dev)
    bins = torch.empty(layout_bytes(lay), dtype=torch.uint8, device=dev)
    check(load().dp_bin_values(_ptr(values), ctypes.byref(lay), _ptr(cp), _ptr(cv), _ptr(bins),
                               _stream()))
    return bins


def objective_gradients(objective, margin, label, n_classes):
    n = label.shape[0]
    grad = torch.empty((n, n_classes), dtype=torch.float32, device=margin.device)
    hess = torch.empty_like(grad)
    check(load().dp_objective_gradients(objective, _ptr(margin), _ptr(label), n, n_classes,
                                        _ptr(grad), _ptr(hess), _stream()))
    return grad, hess


def quantise(ws, grad, hess):
    """-> (exps [K,2] int32, gpair [K,n,2] int32, sums [K,2] int64) device tensors."""
    if grad.dim() == 1:
        grad, hess = grad.reshape(-1, 1), hess.reshape(-1, 1)
    n, k = grad.shape
    dev = grad.device
    exps = torch.empty((k, 2), dtype=torch.int32, device=dev)
    gpair = torch.empty((k, n, 2), dtype=torch.int32, device=dev)
    sums = torch.empty((k, 2), dtype=torch.int64, device=dev)
    check(load().dp_quantise_gradients(ws.handle, _ptr(grad.contiguous()), _ptr(hess.contiguous()),
                                       n, k, _ptr(exps), _ptr(gpair), _ptr(sums), _stream()))
    return exps, gpair, sums


def hist_build(ws, bins, lay, gpair, segments, bin_stride, ridx=None, out=None):
    """Histograms [len(segments), F, bin_stride, 2] int64 of row segments."""
    seg = np.asarray(segments, dtype=np.int64).reshape(-1, 2)
    begin = np.ascontiguousarray(seg[:, 0])
    end = np.ascontiguousarray(seg[:, 1])
    n_nodes = seg.shape[0]
    if out is None:
        out = torch.empty((n_nodes, lay.n_features, bin_stride, 2), dtype=torch.int64,
                          device=bins.device)
    check(load().dp_hist_build(ws.handle, _ptr(bins), ctypes.byref(lay), _ptr(gpair), _ptr(ridx),
                               begin.ctypes.data, end.ctypes.data, n_nodes, bin_stride, _ptr(out),
                               _stream()))
    return out


def hist_accumulate(ws, bins, lay, gpair, segments, hist, ridx=None):
    """Adds the histograms of row segments into `hist` [n_nodes, F, stride, 2]."""
    seg = np.asarray(segments, dtype=np.int64).reshape(-1, 2)
    begin = np.ascontiguousarray(seg[:, 0])
    end = np.ascontiguousarray(seg[:, 1])
    check(load().dp_hist_accumulate(ws.handle, _ptr(bins), ctypes.byref(lay), _ptr(gpair),
                                    _ptr(ridx), begin.ctypes.data, end.ctypes.data, seg.shape[0],
                                    hist.shape[2], _ptr(hist), _stream()))
    return hist


def hist_tuning(lay, bin_stride):
    """The autotuner's report for contiguous histograms of this layout ({} before tuning)."""
    import json

    n, out = ctypes.c_uint64(), ctypes.c_char_p()
    check(load().dp_hist_tuning(ctypes.byref(lay), bin_stride, ctypes.byref(n),
                                ctypes.byref(out)))
    return json.loads(ctypes.string_at(out, n.value).decode())


def hist_subtract(parent, built):
    out = torch.empty_like(parent)
    check(load().dp_hist_subtract(_ptr(parent), _ptr(built), _ptr(out), parent.numel(), _stream()))
    return out


def train_param(eta=0.3, lam=1.0, alpha=0.0, gamma=0.0, min_child_weight=1.0, max_depth=6):
    return TrainParam(eta, lam, alpha, gamma, min_child_weight, max_depth)


def evaluate_splits(ws, hist, n_bins, node_sums, exp_g, exp_h, param):
    """Best split per node -> device tensor of split records (see splits_to_numpy)."""
    n_nodes, f, stride, _ = hist.shape
    out = torch.empty((n_nodes, ctypes.sizeof(SplitRecord)), dtype=torch.uint8, device=hist.device)
    check(load().dp_evaluate_splits(ws.handle, _ptr(hist), n_nodes, f, stride, _ptr(n_bins),
                                    _ptr(node_sums),
                                    int(exp_g), int(exp_h), ctypes.byref(param), _ptr(out),
                                    _stream()))
    return out


def splits_to_numpy(records):
    return np.frombuffer(records.cpu().numpy().tobytes(), dtype=SPLIT_DTYPE)


def partition(ws, bins, lay, ridx_in, segments, splits):
    """Stable partition -> (ridx_out tensor, left_count tensor)."""
    seg = np.asarray(segments, dtype=np.int64).reshape(-1, 2)
    begin = np.ascontiguousarray(seg[:, 0])
    end = np.ascontiguousarray(seg[:, 1])
    ridx_out = ridx_in.clone()
    left = torch.zeros(seg.shape[0], dtype=torch.int64, device=bins.device)
    check(load().dp_partition(ws.handle, _ptr(bins), ctypes.byref(lay), _ptr(ridx_in),
                              _ptr(ridx_out), begin.ctypes.data, end.ctypes.data, _ptr(splits),
                              seg.shape[0], _ptr(left), _stream()))
    return ridx_out, left


def update_margin(ws, ridx, segments, values, margin, stride=1):
    seg = np.asarray(segments, dtype=np.int64).reshape(-1, 2)
    begin = np.ascontiguousarray(seg[:, 0])
    end = np.ascontiguousarray(seg[:, 1])
    vals = np.ascontiguousarray(np.asarray(values, dtype=np.float32))
    check(load().dp_update_margin(ws.handle, _ptr(ridx), begin.ctypes.data, end.ctypes.data,
                                  vals.ctypes.data, seg.shape[0], _ptr(margin), stride, _stream()))
    return margin


SYNTH_FEATURES = {1: 8, 2: 28, 3: 128, 4: 784, 5: 1000}


def synth(config, n_rows, seed, device="cuda", n_features=None, want_grad=False):
    """Synthetic benchmark inputs -> (values, labels, grad, hess) device tensors."""
    f = n_features or SYNTH_FEATURES[config]
    values = torch.empty((n_rows, f), dtype=torch.float32, device=device)
    labels = torch.empty(n_rows, dtype=torch.float32, device=device)
    grad = hess = None
    if want_grad:
        grad = torch.empty(n_rows, dtype=torch.float32, device=device)
        hess = torch.empty(n_rows, dtype=torch.float32, device=device)
    check(load().dp_synth(config, seed, n_rows, f, _ptr(values), _ptr(labels), _ptr(grad),
                          _ptr(hess), _stream()))
    return values, labels, grad, hess


# ---------------------------------------------------------------------------
# Decisions: policy and preference losses, advantages
# ---------------------------------------------------------------------------
PolicyLoss = collections.namedtuple("PolicyLoss", "loss logp kl entropy grad hess")
PreferenceLoss = collections.namedtuple("PreferenceLoss", "loss score logp grad hess")


def _dtype(t, what):
    dtype = t.dtype
    if dtype is torch.float32:
        return 0
    if dtype is torch.bfloat16:
        return 2
    if dtype is torch.float16:
        return 1
    raise DPError(f"{what} must be float32, float16 or bfloat16, not {dtype}")


def _like(t, first, shape, what):
    """Checks a float32 array that goes with the tensor `first`."""
    if (t.dtype is not torch.float32 or t.shape != shape or not t.is_contiguous()
            or t.get_device() != first.get_device()):
        raise DPError(f"{what} must be a contiguous float32 tensor of shape {tuple(shape)} on "
                      f"{first.device}")


def _on_current_device(t, what):
    if not t.is_cuda or t.get_device() != torch._C._cuda_getDevice():
        raise DPError(f"{what} must be on the current device")


def _decisions(margin, action):
    if margin.dim() != 2:
        raise DPError("margin must have shape [rows, classes]")
    _on_current_device(margin, "margin")
    n, k = margin.shape
    if k < 1:
        raise DPError("margin must have at least one class")
    row, step = margin.stride()
    if step != 1 and k != 1:
        raise DPError("the classes of a row must be adjacent")
    wide = action.dtype is torch.int64
    if (not (wide or action.dtype is torch.int32) or action.shape != (n,)
            or not action.is_contiguous() or action.get_device() != margin.get_device()):
        raise DPError(f"action must be a contiguous int64 or int32 tensor of shape ({n},) on "
                      f"{margin.device}")
    return Decisions(margin.data_ptr(), action.data_ptr(), n, row, k, _dtype(margin, "margin"),
                     8 if wide else 4)


def _floats(x, *shape):
    """An uninitialised float32 tensor beside x."""
    if x.dtype is torch.float32:
        return x.new_empty(shape)
    return torch.empty(shape, dtype=torch.float32, device=x.device)


def _gradient_of(margin):
    """An uninitialised tensor for margin's gradient or hessian."""
    return torch.empty_like(margin, memory_format=torch.contiguous_format)


def action_logprobs(ws, margin, action, entropy=False):
    """Log-probability of the action of every row of margins [n, K] (float32, float16 or
    bfloat16; rows may be strided) -> (logp [n] float32, entropy [n] float32 or None).

    Rows whose action is outside [0, K), or whose margins are all -infinity, are not counted: 0
    for both."""
    d = _decisions(margin, action)
    logp = _floats(margin, d.n_rows)
    h = _floats(margin, d.n_rows) if entropy else None
    check(load().dp_action_logprobs(ws.handle, ctypes.byref(d), _ptr(logp), _ptr(h), _stream()))
    return logp, h


def action_logprobs_backward(ws, margin, action, dlogp, dentropy=None):
    """Gradient of the margins (their dtype, [n, K]) from those of action_logprobs' outputs."""
    d = _decisions(margin, action)
    _like(dlogp, margin, action.shape, "dlogp")
    if dentropy is not None:
        _like(dentropy, margin, action.shape, "dentropy")
    grad = _gradient_of(margin)
    check(load().dp_action_logprobs_backward(ws.handle, ctypes.byref(d), _ptr(dlogp),
                                             _ptr(dentropy), _ptr(grad), _stream()))
    return grad


def policy_loss(ws, margin, action, old_logp, advantage, weight=None, reference=None,
                clip_low=0.2, clip_high=0.2, kl=0.0, entropy=0.0, gradient=True, hessian=False):
    """Clipped policy loss of every row, with a KL term to the policy whose log-probabilities of
    the actions are `reference` and an entropy bonus, and its gradient of the margins
    -> PolicyLoss(loss, logp, kl, entropy, grad, hess).

    old_logp, advantage, weight and reference are float32 [n]; loss [n] holds the weighted rows,
    so its sum is what grad [n, K] is the gradient of.  hess (float32 margins only) is what
    Booster.boost takes beside grad.  kl is None without a reference, grad without gradient."""
    d = _decisions(margin, action)
    _like(old_logp, margin, action.shape, "old_logp")
    _like(advantage, margin, action.shape, "advantage")
    if weight is not None:
        _like(weight, margin, action.shape, "weight")
    if reference is not None:
        _like(reference, margin, action.shape, "reference")
    if hessian and not gradient:
        raise DPError("a hessian needs the gradient")
    rows = _floats(old_logp, 4, d.n_rows)
    at, step = rows.data_ptr(), 4 * d.n_rows
    loss, logp, k, h = rows.unbind()
    k_at = at + 2 * step
    if reference is None:
        k = k_at = None
    grad = _gradient_of(margin) if gradient else None
    hess = _gradient_of(margin) if hessian else None
    param = PolicyParam(clip_low, clip_high, kl, entropy)
    check(load().dp_policy_loss(ws.handle, ctypes.byref(d), old_logp.data_ptr(),
                                advantage.data_ptr(), _ptr(weight), _ptr(reference),
                                ctypes.byref(param), at, at + step, k_at, at + 3 * step,
                                _ptr(grad), _ptr(hess), _stream()))
    return PolicyLoss(loss, logp, k, h, grad, hess)


def preference_loss(ws, margin, action, sequences, reference=None, beta=0.1, smoothing=0.0,
                    average=False, gradient=True, hessian=False):
    """Preference loss of pairs of row sequences and its gradient of the margins
    -> PreferenceLoss(loss [P], score [P], logp [n], grad [n, K], hess).

    sequences (int64 [2 P + 1], on the device) holds the offsets of the sequences' rows; pair i
    prefers sequence 2 i to sequence 2 i + 1.  reference (float32 [n]) holds the reference
    policy's log-probabilities of the actions; loss.sum() is what grad is the gradient of."""
    d = _decisions(margin, action)
    if (sequences.dtype is not torch.int64 or sequences.dim() != 1
            or not sequences.is_contiguous() or len(sequences) % 2 != 1
            or sequences.device != margin.device):
        raise DPError(
            f"sequences must be a contiguous int64 tensor of 2 P + 1 offsets on {margin.device}")
    if reference is not None:
        _like(reference, margin, action.shape, "reference")
    if hessian and not gradient:
        raise DPError("a hessian needs the gradient")
    pairs = len(sequences) // 2
    loss, score = _floats(margin, 2, pairs).unbind()
    logp = _floats(margin, d.n_rows)
    grad = _gradient_of(margin) if gradient else None
    hess = _gradient_of(margin) if hessian else None
    param = PreferenceParam(beta, smoothing, bool(average))
    check(load().dp_preference_loss(ws.handle, ctypes.byref(d), _ptr(sequences), pairs,
                                    _ptr(reference), ctypes.byref(param), _ptr(loss), _ptr(score),
                                    _ptr(logp), _ptr(grad), _ptr(hess), _stream()))
    return PreferenceLoss(loss, score, logp, grad, hess)


def _recurrence(reverse, arrays, ends):
    """The C description of [B, T, C] arrays and checks of the float32 [B, C] ones."""
    first, what = arrays[0]
    if first.dim() != 3:
        raise DPError(f"{what} must have shape [batch, time, channels]")
    _on_current_device(first, what)
    size, dtype, device = first.shape, first.dtype, first.get_device()
    b, t, c = size
    shape = Recurrence(b, t, c, _dtype(first, what), bool(reverse))
    for at, (x, what) in zip(shape.strides, arrays):
        if x.dtype is not dtype or x.shape != size or x.get_device() != device:
            raise DPError(f"{what} must be {dtype} of shape {(b, t, c)} on {first.device}")
        at[0], at[1], step = x.stride()
        if step != 1 and c > 1:
            raise DPError(f"the channels of {what} must be adjacent")
    for x, what in ends:
        if x is not None:
            _like(x, first, (b, c), what)
    return shape


def _dense_like(x):
    """An empty tensor in x's order of dimensions, without its gaps or repeats."""
    out = torch.empty_like(x)  # keeps the strides of dense tensors only
    return out if out.stride(2) == 1 or out.shape[2] <= 1 else out.contiguous()


def linear_recurrence(ws, gate, value, initial=None, reverse=False):
    """state_t = gate_t state_(t-1) + value_t over the time of [B, T, C] tensors (reverse: from
    the state after) -> (state in value's dtype and order, last state [B, C] float32).

    initial (float32 [B, C]) is the state before the first step, zero without.  Batch and time
    may be strided (time-major arrays as a transposed view, a gate expanded over batch or time);
    channels are adjacent.  With a single step (T = 1) and initial = last of the call before, it
    is one step of a running recurrence.  Advantages: value the temporal differences, gate
    gamma * lambda, 0 where an episode ends, reverse=True."""
    shape = _recurrence(reverse, [(gate, "gate"), (value, "value")], [(initial, "initial")])
    state = _dense_like(value)
    at = shape.strides[2]
    at[0], at[1], _ = state.stride()
    last = _floats(gate, shape.batch, shape.channels)
    check(load().dp_linear_recurrence(ws.handle, ctypes.byref(shape), _ptr(gate), _ptr(value),
                                      _ptr(initial), _ptr(state), _ptr(last), _stream()))
    return state, last


def linear_recurrence_backward(ws, gate, state, dstate, initial=None, dlast=None, reverse=False):
    """Gradients of linear_recurrence's inputs from those of its outputs (dlast: float32 [B, C],
    zero without) and the states it returned -> (dgate, dvalue, dinitial [B, C] float32).

    An input that was expanded has the sum of its gradient over the expanded dimension."""
    shape = _recurrence(reverse, [(gate, "gate"), (state, "state"), (dstate, "dstate")],
                        [(initial, "initial"), (dlast, "dlast")])
    dvalue = _dense_like(dstate)
    dgate = _dense_like(dvalue)
    for i, x in ((3, dgate), (4, dvalue)):
        at = shape.strides[i]
        at[0], at[1], _ = x.stride()
    dinitial = _floats(gate, shape.batch, shape.channels)
    check(load().dp_linear_recurrence_backward(ws.handle, ctypes.byref(shape), _ptr(gate),
                                               _ptr(state), _ptr(dstate), _ptr(initial),
                                               _ptr(dlast), _ptr(dgate), _ptr(dvalue),
                                               _ptr(dinitial), _stream()))
    return dgate, dvalue, dinitial
