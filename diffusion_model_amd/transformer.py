"""Operators of a transformer block over tokens (no counterpart in the reference's models): layer norm, rotary positions and
the gated feed-forward block, each with its backward pass, on the HIP kernels of libdm_sampler.so (include/dm_sampler.h).

They work on fp32, bfloat16 and half tensors of one GPU and run on that GPU's current stream; every sum is fp32.  Like
the rest of the package they carry no autograd: a training step calls the backward functions itself.  Inputs may be views:
what the kernels cannot read as it lies (a last dimension with a stride, rows off 16-byte boundaries) is copied first.
Outputs and workspaces come from torch's allocator, so the calls may be captured into a graph.  There is no CPU path."""
import ctypes as C
import math
import struct

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_POSITIONS = (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8)
_KEEP_F32 = 256  # DM_FFN_KEEP_F32
_ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}


def _dtype(t, name):
    if not torch.is_tensor(t):
        raise RuntimeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be on the GPU (it is on {t.device}). There is no CPU path.")
    if t.dtype not in _DTYPES:
        raise RuntimeError(f"{name} must be fp32, bfloat16 or half (got {t.dtype})")
    return _DTYPES[t.dtype]


def _like(t, x, name, dtypes=None):
    if torch.is_tensor(t) and t.is_cuda and t.get_device() == x.get_device() and t.dtype in (dtypes or (x.dtype,)):
        return t
    _dtype(t, name)
    if t.device != x.device:
        raise RuntimeError(f"{name} must be on {x.device} (got {t.device})")
    if t.dtype not in (dtypes or (x.dtype,)):
        raise RuntimeError(f"{name} must be of type {' or '.join(str(d) for d in dtypes or (x.dtype,))} (got {t.dtype})")
    return t


def _vector(t, n, x, name, dtypes=None):
    if t is None:
        return None
    _like(t, x, name, dtypes)
    if t.dim() != 1 or t.shape[0] != n:
        raise RuntimeError(f"{name} must be [{n}] (got {tuple(t.shape)})")
    return t.contiguous()


def _rows(t, pieces=True):
    """[..., C] as rows the kernels can read: (tensor, row stride in elements, number of rows).  ``pieces``: rows of whole 16-byte pieces
    start at multiples of 16 bytes."""
    c = t.shape[-1]
    if t.is_contiguous():
        if not pieces or t.data_ptr() % 16 == 0:
            return t, c, t.numel() // c
        return t.clone(), c, t.numel() // c
    r = t.reshape(-1, c)
    m, whole = r.shape[0], 16 // t.element_size()
    if (c > 1 and r.stride(1) != 1) or (m > 1 and (r.stride(0) < c or r.stride(0) > 1 << 21)) or \
            (pieces and c % whole == 0 and (r.data_ptr() % 16 or (m > 1 and r.stride(0) % whole))):
        r = r.clone(memory_format=torch.contiguous_format)
    return r, (r.stride(0) if m > 1 else c), m


def _matrix(t, rows, cols, x, name):
    _like(t, x, name)
    if t.dim() != 2 or (rows is not None and t.shape[0] != rows) or t.shape[1] != cols:
        raise RuntimeError(f"{name} must be [{rows if rows is not None else 'any'}, {cols}] (got {tuple(t.shape)})")
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(t, fn, *args):
    """fn(*args, stream) on the tensor's device and its current stream; raises what the library reports."""
    index = t.get_device()
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def _empty_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _workspace(t, nbytes):
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=t.device)


# ------------------------------------------------------------------ layer norm

def layer_norm(x, weight=None, bias=None, eps=1e-5, return_stats=False):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.  ``weight`` and ``bias`` ([C], either may be
    missing) are both of x's type or both fp32.  ``return_stats``: (y, mean, rstd), fp32, for the backward pass."""
    dt = _dtype(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"layer_norm needs a last dimension to normalise (got {tuple(x.shape)})")
    c = x.shape[-1]
    w = _vector(weight, c, x, "weight", (x.dtype, torch.float32))
    b = _vector(bias, c, x, "bias", (x.dtype, torch.float32) if w is None else (w.dtype,))
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    p = x if w is None and b is None else b if w is None else w
    r, stride, m = _rows(x, False)
    y = _empty_like(x)
    mean = rstd = None
    if return_stats:
        mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
    _call(x, _lib.lib().dm_layer_norm, r.data_ptr(), stride, _ptr(w), _ptr(b), _DTYPES[p.dtype], y.data_ptr(), _ptr(mean), _ptr(rstd), m, c,
          eps, dt)
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(grad, x, weight, mean, rstd, bias=None):
    """(dx, dweight, dbias) from the output's gradient and what ``layer_norm(..., return_stats=True)`` returned.  The parameters'
    gradients are of their type, summed over all rows in a fixed order: both where there is a ``weight``, dbias alone where only
    the forward call's ``bias`` is given, otherwise None."""
    dt = _dtype(x, "x")
    _like(grad, x, "grad")
    if x.dim() < 1 or x.shape[-1] < 1 or grad.shape != x.shape:
        raise RuntimeError(f"grad must have x's shape {tuple(x.shape)} (got {tuple(grad.shape)})")
    c = x.shape[-1]
    w = _vector(weight, c, x, "weight", (x.dtype, torch.float32))
    b = _vector(bias, c, x, "bias", (x.dtype, torch.float32) if w is None else (w.dtype,))
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        _like(t, x, name, (torch.float32,))
        if t.shape != x.shape[:-1]:
            raise RuntimeError(f"{name} must be {tuple(x.shape[:-1])} (got {tuple(t.shape)})")
    L = _lib.lib()
    r, stride, m = _rows(x, False)
    g, gstride, _ = _rows(grad, False)
    mean, rstd = mean.contiguous(), rstd.contiguous()
    dx = _empty_like(x)
    dw = db = ws = None
    nbytes = 0
    p = b if w is None else w
    if p is not None:
        dw, db = None if w is None else torch.empty_like(w), torch.empty_like(p)
        nbytes = L.dm_layer_norm_backward_workspace_bytes(m, c)
        ws = _workspace(x, nbytes)
    _call(x, L.dm_layer_norm_backward, g.data_ptr(), gstride, r.data_ptr(), stride, _ptr(w), dt if p is None else _DTYPES[p.dtype],
          mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), _ptr(dw), _ptr(db), m, c, dt, _ptr(ws), nbytes)
    return dx, dw, db


# ------------------------------------------------------------------ rotary positions

def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=None, axes=1, device=None):
    """(inv_freq, scale) for ``apply_rotary``: inv_freq[i] = base^(-2i / d), float64, with d = rotary_dim / axes (each axis has
    the whole range).  To stretch positions trained up to ``original_length`` by ``factor``: "linear" divides all frequencies;
    "ntk" raises the base so that the slowest pair is divided by ``factor``; "yarn" divides the pairs that turn less than once over
    the trained length, keeps those that turn more than 32 times, blends between (linearly in the pair, from the last whole pair before the
    one that turns 32 times to the first one behind that which turns once, which may lie behind the slowest pair), and scales by 0.1 ln(factor) + 1."""
    if axes < 1 or rotary_dim < 0 or rotary_dim % (2 * axes):
        raise ValueError(f"rotary_dim {rotary_dim} must be a multiple of {2 * axes} (pairs on {axes} axes)")
    if base <= 0 or factor <= 0:
        raise ValueError("base and factor must be positive")
    pairs = rotary_dim // 2 // axes
    i = torch.arange(pairs, dtype=torch.float64)
    span, scale = max(pairs, 1), 1.0
    if scaling == "ntk" and pairs > 1:
        base = base * factor ** (pairs / (pairs - 1))
    inv = float(base) ** (-i / span)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn":
        if not original_length or original_length <= 0:
            raise ValueError("yarn scaling needs the trained length (original_length)")
        if base <= 1:
            raise ValueError("yarn scaling needs a base above 1")

        def pair_that_turns(n):
            return span * math.log(original_length / (n * 2 * math.pi)) / math.log(base)
        low = max(math.floor(pair_that_turns(32)), 0)
        high = min(math.ceil(pair_that_turns(1)), 2 * span - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"Unknown rotary scaling: {scaling}")
    return inv.repeat(axes).to(device if device is not None else "cpu"), scale


_Strides = C.c_int64 * 3
_TENSOR = struct.Struct("@PP6qi4x")  # dm_rotary_tensor; packed by one call, as a structure built field by field costs more than the launch


def _turned(x, inplace):
    """x as the kernel reads it, where the result goes, and both as dm_rotary_tensor."""
    b, t, heads, d = x.shape
    strides = x.stride()
    if d > 1 and strides[3] != 1:
        if inplace:
            raise RuntimeError("in place needs contiguous head elements")
        x = x.contiguous()
        strides = x.stride()
    if inplace:
        if any(n > 1 and s == 0 for n, s in zip((b, t, heads), strides)):
            raise RuntimeError("in place needs a tensor without expanded dimensions")
        p = x.data_ptr()
        return x, x, _lib.RotaryTensor.from_buffer_copy(_TENSOR.pack(p, p, *strides[:3], *strides[:3], heads))
    out = _empty_like(x)
    return x, out, _lib.RotaryTensor.from_buffer_copy(
        _TENSOR.pack(x.data_ptr(), out.data_ptr(), *strides[:3], t * heads * d, heads * d, d, heads))


def apply_rotary(q, k, inv_freq, positions=None, layout="half", scale=1.0, inverse=False, inplace=False):
    """Turns the pairs of every head of ``q`` [B, T, heads, head_dim] and ``k`` (the same with its own heads, or None) by
    position * inv_freq; returns (q, k).  ``inv_freq`` (float64 [rotary_dim / 2], on the GPU) says how much of the head turns;
    the rest is copied.  ``positions``: integers [T], [B, T], or [axes, B, T] (pair i takes axis i // (pairs / axes)), None for
    0..T-1; angles are formed in 64 bits (off by 2^-51 of themselves).  ``layout``: "half" pairs element i with i + rotary_dim/2, "interleaved" 2i with 2i + 1.
    ``inverse`` turns back: applied to gradients it is the backward pass.  ``inplace`` writes into q and k
    themselves, which must share no elements then."""
    dt = _dtype(q, "q")
    if q.dim() != 4 or q.shape[3] < 1:
        raise RuntimeError(f"q must be [B, T, heads, head_dim] (got {tuple(q.shape)})")
    b, t, _, d = q.shape
    if k is not None:
        _like(k, q, "k")
        if k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != d:
            raise RuntimeError(f"k must be [{b}, {t}, heads, {d}] (got {tuple(k.shape)})")
    if layout not in ("half", "interleaved"):
        raise ValueError(f"Unknown rotary layout: {layout}")
    if not torch.is_tensor(inv_freq) or inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or inv_freq.get_device() != q.get_device():
        raise RuntimeError(f"inv_freq must be a float64 vector on {q.device} (rotary_frequencies makes one)")
    pairs = inv_freq.numel()
    if 2 * pairs > d:
        raise RuntimeError(f"{pairs} pairs do not fit a head of {d} elements")
    axes, strides = 1, None
    if positions is not None:
        if not torch.is_tensor(positions) or positions.dtype not in _POSITIONS or positions.get_device() != q.get_device():
            raise RuntimeError(f"positions must be integers on {q.device}")
        shape = positions.shape
        dims = len(shape)
        axes = shape[0] if dims == 3 else 1
        if dims not in (1, 2, 3) or axes < 1:
            raise RuntimeError(f"positions must be [T], [B, T] or [axes, B, T] (got {tuple(shape)})")
        if shape[-1] not in (1, t) or (dims > 1 and shape[-2] not in (1, b)):
            raise RuntimeError(f"positions must be [T], [B, T] or [axes, B, T] with B = {b}, T = {t} (got {tuple(shape)})")
        if positions.dtype != torch.int64:
            positions = positions.to(torch.int64)
        have = positions.stride()
        strides = _Strides(have[0] if axes > 1 else 0, have[-2] if dims > 1 and shape[-2] > 1 else 0, have[-1] if shape[-1] > 1 else 0)
    if pairs % axes:
        raise RuntimeError(f"{pairs} pairs do not divide into {axes} axes")
    if inplace and k is not None and k.data_ptr() == q.data_ptr() and q.numel() and k.numel():
        raise RuntimeError("in place needs q and k that share no elements")
    q, q_out, q_arg = _turned(q, inplace)
    k_out = k_arg = None
    if k is not None:
        k, k_out, k_arg = _turned(k, inplace)
    inv_freq = inv_freq.contiguous()
    _call(q, _lib.lib().dm_rotary, q_arg, k_arg, _ptr(positions), strides, axes, inv_freq.data_ptr(), b, t, d, 2 * pairs, layout == "interleaved",
          scale, bool(inverse), dt)
    return q_out, k_out


# ------------------------------------------------------------------ gated feed-forward block

def _ffn_check(x, w_gate, w_up, w_down, activation):
    dt = _dtype(x, "x")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"Unknown activation: {activation}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"x must be [..., width] (got {tuple(x.shape)})")
    d = x.shape[-1]
    w_gate = _matrix(w_gate, None, d, x, "w_gate")
    f = w_gate.shape[0]
    w_up = _matrix(w_up, f, d, x, "w_up")
    w_down = _matrix(w_down, None, f, x, "w_down")
    if f < 1 or w_down.shape[0] < 1:
        raise RuntimeError("the weights must not be empty")
    return dt, d, f, w_down.shape[0], w_gate, w_up, w_down


def gated_ffn(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu", save=False):
    """(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down, with weights as nn.Linear holds them: w_gate and w_up
    [hidden, width], w_down [out, hidden].  All tensors are of one type.  ``activation``: silu, gelu (erf), gelu_tanh, relu, sigmoid.
    ``save``: (y, saved), with ``saved`` (opaque) for ``gated_ffn_backward``.  16-bit types round the hidden values (forward, but of one
    or two rows) and their gradients to that type between the matrix products, in half to infinity from 65520 on; what else ``saved`` keeps of them is
    fp32 (10 bytes per hidden value), or with ``save="compact"`` of their type too (6 bytes, gradients less exact by a quarter).  fp32 keeps fp32
    accuracy (an infinite operand may give NaN where fp32 would give an infinity)."""
    if save not in (False, True, "compact"):
        raise ValueError(f"save must be False, True or 'compact' (got {save!r})")
    dt, d, f, n, w_gate, w_up, w_down = _ffn_check(x, w_gate, w_up, w_down, activation)
    b_gate, b_up, b_down = _vector(b_gate, f, x, "b_gate"), _vector(b_up, f, x, "b_up"), _vector(b_down, n, x, "b_down")
    L = _lib.lib()
    r, stride, m = _rows(x)
    y = _empty_like(x) if n == d else torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=x.device)
    keep = _KEEP_F32 if save and save != "compact" else 0
    saved = torch.empty(L.dm_gated_ffn_saved_bytes(m, f, dt | keep), dtype=torch.uint8, device=x.device) if save else None
    nbytes = L.dm_gated_ffn_workspace_bytes(m, d, f, n, dt, bool(save))
    ws = _workspace(x, nbytes)
    _call(x, L.dm_gated_ffn, r.data_ptr(), stride, w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), _ptr(b_gate), _ptr(b_up), _ptr(b_down),
          y.data_ptr(), _ptr(saved), m, d, f, n, _ACTIVATIONS[activation] | keep, dt, ws.data_ptr(), nbytes)
    return (y, saved) if save else y


def gated_ffn_backward(grad, x, w_gate, w_up, w_down, saved, activation="silu", bias=False):
    """(dx, dw_gate, dw_up, dw_down, db_gate, db_up, db_down) from the output's gradient and the ``saved`` of the forward call; the
    biases' gradients are None unless ``bias``.  Sums run in a fixed order: the same inputs give the same bits."""
    dt, d, f, n, w_gate, w_up, w_down = _ffn_check(x, w_gate, w_up, w_down, activation)
    _like(grad, x, "grad")
    if grad.shape != x.shape[:-1] + (n,):
        raise RuntimeError(f"grad must be {tuple(x.shape[:-1]) + (n,)} (got {tuple(grad.shape)})")
    L = _lib.lib()
    r, stride, m = _rows(x)
    g, gstride, _ = _rows(grad)
    keep = _KEEP_F32  # by its size
    if torch.is_tensor(saved) and saved.numel() == L.dm_gated_ffn_saved_bytes(m, f, dt):
        keep = 0
    if not torch.is_tensor(saved) or saved.device != x.device or saved.dtype != torch.uint8 or not saved.is_contiguous() or \
            saved.numel() != L.dm_gated_ffn_saved_bytes(m, f, dt | keep):
        raise RuntimeError("saved must be what gated_ffn(..., save=True) returned for this input")
    dx = _empty_like(x)
    dws = [torch.empty_like(w) for w in (w_gate, w_up, w_down)]
    dbs = [torch.empty(size, dtype=x.dtype, device=x.device) if bias else None for size in (f, f, n)]
    nbytes = L.dm_gated_ffn_backward_workspace_bytes(m, d, f, n, dt)
    ws = _workspace(x, nbytes)
    _call(x, L.dm_gated_ffn_backward, g.data_ptr(), gstride, r.data_ptr(), stride, w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
          saved.data_ptr(), dx.data_ptr(), *(_ptr(t) for t in dws + dbs), m, d, f, n, _ACTIVATIONS[activation] | keep, dt, ws.data_ptr(), nbytes)
    return (dx, *dws, *dbs)
