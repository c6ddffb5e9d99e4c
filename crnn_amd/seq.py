"""Sequence operators on the device: a short causal convolution, the selective state space scan and activation checkpoints in 8 bits.

The scan is the linear member of the ODE family this package integrates: a diagonal linear ODE h' = A h + B(t) u(t) with learned rates,
stepped exactly over steps of their own length (an irregular time grid), thousands of channels and rows, with its discrete adjoint.

    causal_conv / causal_conv_grad / causal_conv_step          p[t, d] = bias[d] + sum_j weight[d, j] x[t - W + 1 + j, d];  y = p, or p sigmoid(p)
    selective_scan / selective_scan_grad / selective_scan_step h = exp(delta A) h + delta u B;  y = sum_n C h + D u, or that times z sigmoid(z);
                                                               delta = softplus(dt + dt_bias), or dt + dt_bias
    pack8 / unpack8                                            a row's channels in 8 bits, a power of two as scale per 32 of them

Arrays are torch tensors on an MI355X; the calls enqueue on that device's current stream and do not wait, so that they may be captured into
a graph.  Rows are time, channels are contiguous: dense [n_seq, rows, D] (lengths=: how many rows of each are its own, the others are
padding), or packed [rows, D] with seq_start [n_seq + 1], int32 on the device: sequence s is rows seq_start[s] .. seq_start[s + 1] - 1.
Lengths and offsets are not read by the host: they are clamped to the arrays.  Rows of a result that belong to no sequence are 0, and stay as
they were where the caller gave the array (out=).  float32, bfloat16, float16 and float64; weights, rates and scan states are float32
(float64 with float64 data).  A checkpoint (Packed8) may stand for x of the convolution, and for u and z of the scan.
"""
from __future__ import annotations

import ctypes as C
from collections import namedtuple

from . import _lib as L
from ._lib import ConvArgs, ScanArgs, View, check, lib

ConvGrads = namedtuple("ConvGrads", "x weight bias state")
ScanGrads = namedtuple("ScanGrads", "u dt A B C D z dt_bias state")

_EMULATED = "SIMT-EMULATION" in lib.crnn_build_info().decode()     # the emulated device's memory is the host's


def _torch():
    import torch
    return torch


def _dtypes():
    t = _torch()
    return {t.float32: L.DT_F32, t.bfloat16: L.DT_BF16, t.float16: L.DT_F16, t.float64: L.DT_F64}


class Packed8:
    """A checkpoint: codes int8 [..., D], scales uint8 [..., ceil(D / 32)] (exponent + 127 of a block of 32 channels), value = code * 2^exponent.
    dtype: the type of the tensor it was made from."""

    __slots__ = ("codes", "scales", "dtype")

    def __init__(self, codes, scales, dtype):
        t = _torch()
        if codes.dtype != t.int8 or scales.dtype != t.uint8:
            raise TypeError("Packed8: codes must be int8 and scales uint8")
        if codes.ndim < 1 or tuple(scales.shape) != (*codes.shape[:-1], -(-codes.shape[-1] // 32)):
            raise ValueError(f"Packed8: scales must be {(*codes.shape[:-1], -(-codes.shape[-1] // 32))}, not {tuple(scales.shape)}")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("Packed8: codes and scales must be contiguous")
        if codes.device != scales.device:
            raise ValueError("Packed8: codes and scales must be on one device")
        if dtype not in (t.float32, t.bfloat16, t.float16):
            raise TypeError("Packed8: float32, bfloat16 or float16 only")
        self.codes, self.scales, self.dtype = codes, scales, dtype

    shape = property(lambda self: self.codes.shape)
    ndim = property(lambda self: self.codes.ndim)
    device = property(lambda self: self.codes.device)


def _on_device(x, what):
    dev = x.device
    if dev.type != "cuda" and not (_EMULATED and dev.type == "cpu"):
        raise ValueError(f"{what} must be on the GPU (there is no CPU path)")
    return dev


def _ordinal(dev):
    return 0 if dev.type == "cpu" else dev.index


def _stream(dev):
    return None if dev.type == "cpu" else _torch().cuda.current_stream(dev).cuda_stream


def _ptr(x):
    return x.data_ptr() if x is not None and x.numel() else None


# a pointer for arrays that may have no elements: "absent" and "empty" differ
_NOTHING = 256


def _view(x):
    """A View of [..., rows, D] or [rows, D] with contiguous channels."""
    v = View()
    if x is None:
        return v
    if isinstance(x, Packed8):
        v.ptr, v.scales, v.dtype = x.codes.data_ptr() or _NOTHING, x.scales.data_ptr() or _NOTHING, L.DT_PACKED8
        v.row_stride, v.scale_row_stride = x.codes.stride(-2), x.scales.stride(-2)
        if x.ndim == 3:
            v.seq_stride, v.scale_seq_stride = x.codes.stride(0), x.scales.stride(0)
        return v
    v.ptr, v.dtype, v.row_stride = x.data_ptr() or _NOTHING, _dtypes()[x.dtype], x.stride(-2)
    if x.ndim == 3:
        v.seq_stride = x.stride(0)
    return v


def _channels(x, name):
    """x with contiguous channels (a view where it has them)."""
    if isinstance(x, Packed8) or x.stride(-1) == 1 or x.shape[-1] <= 1:
        return x
    return x.contiguous()


class _Rows:
    """What the arrays of one call have in common: type, device, sequences and rows."""

    def __init__(self, x, name, seq_start, lengths):
        t = _torch()
        self.packed = seq_start is not None
        if self.packed and lengths is not None:
            raise ValueError("seq_start (packed rows) and lengths (a padded batch) exclude each other")
        if x.ndim != (2 if self.packed else 3):
            raise ValueError(f"{name} must be {'[rows, D] (packed)' if self.packed else '[n_seq, rows, D]'}, not {tuple(x.shape)}")
        if x.dtype not in _dtypes():
            raise TypeError(f"{name}: float32, bfloat16, float16 or float64, not {x.dtype}")
        self.dtype, self.device, self.shape = x.dtype, _on_device(x, name), tuple(x.shape)
        self.D = x.shape[-1]
        self.param = t.float64 if x.dtype == t.float64 else t.float32
        for what, idx, n in (("seq_start", seq_start, None), ("lengths", lengths, x.shape[0])):
            if idx is None:
                continue
            if idx.dtype != t.int32 or idx.ndim != 1 or idx.device != self.device or not idx.is_contiguous():
                raise ValueError(f"{what} must be a contiguous int32 vector on {self.device}")
            if n is not None and idx.shape[0] != n or idx.shape[0] < 1 and what == "seq_start":
                raise ValueError(f"{what} has {idx.shape[0]} entries")
        self.n_seq = seq_start.shape[0] - 1 if self.packed else x.shape[0]
        self.rows = x.shape[0] if self.packed else x.shape[1]
        self.seq_start, self.lengths = seq_start, lengths
        self.ragged = self.packed or lengths is not None

    def like(self, x, name, packed_ok=False):
        if isinstance(x, Packed8) and not packed_ok:
            raise TypeError(f"{name} cannot be an 8-bit checkpoint here")
        if tuple(x.shape) != self.shape or x.dtype != self.dtype or x.device != self.device:
            raise ValueError(f"{name} must be {self.shape} {self.dtype} on {self.device}, not {tuple(x.shape)} {x.dtype} on {x.device}")
        return _channels(x, name)

    def weight(self, x, name, shape):
        """A parameter in the type parameters have here."""
        if x is None:
            return None
        if tuple(x.shape) != shape or x.device != self.device or not x.dtype.is_floating_point:
            raise ValueError(f"{name} must be {shape} on {self.device}, not {tuple(x.shape)} {x.dtype} on {x.device}")
        return x.to(self.param).contiguous()

    def state(self, x, name, shape, dtype):
        if x is None:
            return None
        if tuple(x.shape) != shape or x.dtype != dtype or x.device != self.device:
            raise ValueError(f"{name} must be {shape} {dtype} on {self.device}, not {tuple(x.shape)} {x.dtype} on {x.device}")
        return x.contiguous()

    def out(self, given, name="out"):
        if given is None:
            return _torch().empty(self.shape, dtype=self.dtype, device=self.device)
        if tuple(given.shape) != self.shape or given.dtype != self.dtype or given.device != self.device or given.stride(-1) != 1 and self.D > 1:
            raise ValueError(f"{name} must be {self.shape} {self.dtype} on {self.device} with contiguous channels")
        return given

    def fill(self, a):
        a.struct_size, a.device, a.stream = C.sizeof(a), _ordinal(self.device), _stream(self.device)
        a.n_seq, a.rows, a.D, a.dtype = self.n_seq, self.rows, self.D, _dtypes()[self.dtype]
        a.seq_start = self.seq_start.data_ptr() if self.packed else None
        a.seq_len = self.lengths.data_ptr() if self.lengths is not None and self.n_seq else None

    def workspace(self, a, need):
        """The call's own scratch memory, from torch's allocator on the call's stream (a graph under capture keeps its own)."""
        if need < 0:
            check(-1)
        ws = _torch().empty(max(int(need), 1), dtype=_torch().uint8, device=self.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), int(need)
        return ws


def _slots(rows, slots, n):
    t = _torch()
    if slots is None:
        return None
    if slots.dtype != t.int32 or tuple(slots.shape) != (n,) or slots.device != rows.device or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int32 vector of {n} entries on {rows.device}")
    return slots


# ---------------------------------------------------------------- convolution
def _conv(rows, x, weight, bias, silu, state):
    if weight.ndim != 2 or not 1 <= weight.shape[1] <= L.SEQ_MAX_TAPS:
        raise ValueError(f"weight must be [D, W] with 1 <= W <= {L.SEQ_MAX_TAPS}, not {tuple(weight.shape)}")
    a = ConvArgs()
    rows.fill(a)
    W = a.W = weight.shape[1]
    a.silu = int(bool(silu))
    weight, bias = rows.weight(weight, "weight", (rows.D, W)), rows.weight(bias, "bias", (rows.D,))
    st = rows.state(state, "state", (rows.n_seq, W - 1, rows.D), rows.dtype)
    a.weight, a.bias, a.x, a.state_in = weight.data_ptr(), _ptr(bias), _view(x), _view(st if W > 1 else None)
    return a, W, (weight, bias, st)


def causal_conv(x, weight, bias=None, *, silu=False, seq_start=None, lengths=None, state=None, return_state=False, out=None):
    """The convolution of each sequence with its own past.  weight [D, W]: the last tap meets the row itself.  state [n_seq, W - 1, D]: the rows
    before the first (absent: 0).  Returns y, or (y, the state behind the last rows)."""
    rows = _Rows(x, "x", seq_start, lengths)
    x = rows.like(x, "x", packed_ok=True)
    a, W, keep = _conv(rows, x, weight, bias, silu, state)
    y = rows.out(out)
    a.y, a.zero_outside = _view(y), int(out is None and rows.ragged)
    end = None
    if return_state:
        end = _torch().empty((rows.n_seq, W - 1, rows.D), dtype=rows.dtype, device=rows.device)
        a.state_out = _view(end if W > 1 else None)
    if rows.D:
        check(lib.crnn_conv_forward(C.byref(a)))
    return (y, end) if return_state else y


def causal_conv_grad(dy, x, weight, bias=None, *, silu=False, seq_start=None, lengths=None, state=None, dstate=None):
    """Gradients of causal_conv from dy (and dstate, the gradient of the state it returned): ConvGrads(x, weight, bias, state); bias and state are
    None where the call had none.  x may be a checkpoint: the gradient is taken at the values it holds."""
    t = _torch()
    rows = _Rows(x, "x", seq_start, lengths)
    x, dy = rows.like(x, "x", packed_ok=True), rows.like(dy, "dy")
    a, W, keep = _conv(rows, x, weight, bias, silu, state)
    dstate = rows.state(dstate, "dstate", (rows.n_seq, W - 1, rows.D), rows.dtype)
    dx = rows.out(None)
    dw = t.empty((rows.D, W), dtype=rows.param, device=rows.device)
    db = t.empty((rows.D,), dtype=rows.param, device=rows.device) if bias is not None else None
    ds = t.empty((rows.n_seq, W - 1, rows.D), dtype=rows.dtype, device=rows.device) if state is not None else None
    a.dy, a.dx, a.zero_outside = _view(dy), _view(dx), int(rows.ragged)
    a.dweight, a.dbias = dw.data_ptr(), _ptr(db)
    if W > 1:
        a.dstate_out, a.dstate_in = _view(dstate), _view(ds)
    ws = rows.workspace(a, lib.crnn_conv_workspace(C.byref(a)))  # noqa: F841
    check(lib.crnn_conv_backward(C.byref(a)))
    return ConvGrads(dx, dw, db, ds)


def causal_conv_step(x, weight, bias, state, slots=None, *, silu=False, out=None):
    """One more row for each of many running sequences: x [n, D], state [n_slots, W - 1, D] moved up in place.  slots [n], int32: row r continues
    the state in slots[r] (absent: in r).  A slot outside the state: the row is padding, its result 0.  Rows that name the same slot are
    consecutive rows of its sequence, in their order.  Returns y [n, D]."""
    t = _torch()
    if x.ndim != 2:
        raise ValueError(f"x must be [n, D], not {tuple(x.shape)}")
    rows = _Rows(x[:, None], "x", None, None)
    if isinstance(x, Packed8) or x.dtype not in _dtypes():
        raise TypeError("x cannot be an 8-bit checkpoint here")
    if weight.ndim != 2 or not 1 <= weight.shape[1] <= L.SEQ_MAX_TAPS:
        raise ValueError(f"weight must be [D, W] with 1 <= W <= {L.SEQ_MAX_TAPS}, not {tuple(weight.shape)}")
    a = ConvArgs()
    rows.fill(a)
    n, D = x.shape
    W = a.W = weight.shape[1]
    a.silu, a.rows = int(bool(silu)), 1
    weight, bias = rows.weight(weight, "weight", (D, W)), rows.weight(bias, "bias", (D,))
    if state.ndim != 3 or tuple(state.shape[1:]) != (W - 1, D) or state.dtype != x.dtype or state.device != rows.device or \
            (state.numel() and (state.stride(2) != 1 and D > 1)):
        raise ValueError(f"state must be [n_slots, {W - 1}, {D}] {x.dtype} on {rows.device} with contiguous channels")
    slots = _slots(rows, slots, n)
    if slots is None and n > state.shape[0]:
        raise ValueError(f"{n} rows, but the state has {state.shape[0]} slots")
    x = _channels(x, "x")
    y = t.empty((n, D), dtype=x.dtype, device=x.device) if out is None else out
    if tuple(y.shape) != (n, D) or y.dtype != x.dtype or y.device != rows.device or y.stride(1) != 1 and D > 1:
        raise ValueError(f"out must be [{n}, {D}] {x.dtype} on {rows.device} with contiguous channels")
    a.x, a.y, a.state_in = _view(x), _view(y), _view(state if W > 1 else None)
    a.weight, a.bias, a.slot, a.n_slots = weight.data_ptr(), _ptr(bias), _ptr(slots), state.shape[0]
    check(lib.crnn_conv_step(C.byref(a)))
    return y


# ---------------------------------------------------------------- scan
def _map(rows, m, name, D, lead):
    """B or C as [*lead, G, N]; returns it and (G, N)."""
    if m.ndim == len(lead) + 1:
        m = m.unsqueeze(-2)
    if m.ndim != len(lead) + 2 or tuple(m.shape[:-2]) != lead or m.dtype != rows.dtype or m.device != rows.device:
        raise ValueError(f"{name} must be {(*lead, 'G', 'N')} (or without G) {rows.dtype} on {rows.device}, not {tuple(m.shape)} {m.dtype} on {m.device}")
    return m


def _map_view(m):
    v = View()
    v.ptr, v.dtype, v.row_stride = m.data_ptr() or _NOTHING, _dtypes()[m.dtype], m.stride(-3)
    if m.ndim == 4:
        v.seq_stride = m.stride(0)
    return v, m.stride(-2), m.stride(-1)


def _scan(rows, u, dt, A, B, Cm, D, z, dt_bias, softplus, lead):
    if A.ndim != 2 or A.shape[0] != rows.D or not 1 <= A.shape[1] <= L.SEQ_MAX_STATES:
        raise ValueError(f"A must be [{rows.D}, N] with 1 <= N <= {L.SEQ_MAX_STATES}, not {tuple(A.shape)}")
    a = ScanArgs()
    rows.fill(a)
    N = a.N = A.shape[1]
    B, Cm = _map(rows, B, "B", rows.D, lead), _map(rows, Cm, "C", rows.D, lead)
    if B.shape != Cm.shape or B.shape[-1] != N:
        raise ValueError(f"B and C must both end in [G, {N}], not {tuple(B.shape)} and {tuple(Cm.shape)}")
    a.G = B.shape[-2]
    if a.G < 1 or rows.D % a.G:
        raise ValueError(f"the {rows.D} channels do not fall into {a.G} groups")
    A, D, dt_bias = rows.weight(A, "A", (rows.D, N)), rows.weight(D, "D", (rows.D,)), rows.weight(dt_bias, "dt_bias", (rows.D,))
    a.softplus = int(bool(softplus))
    a.A, a.skip, a.dt_bias = A.data_ptr(), _ptr(D), _ptr(dt_bias)
    a.u, a.dt, a.z = _view(u), _view(dt), _view(z)
    a.B, a.B_group, a.B_state = _map_view(B)
    a.C, a.C_group, a.C_state = _map_view(Cm)
    return a, N, (A, D, dt_bias, B, Cm)


def selective_scan(u, dt, A, B, C_, *, D=None, z=None, dt_bias=None, softplus=True, seq_start=None, lengths=None, state=None, return_state=False, out=None):
    """The scan of each sequence.  u, dt, z as described above; A [D, N]; B, C [.., G, N] or [.., N] (one group) beside u's rows, channel d in group
    d // (D / G); D, dt_bias [D]; state [n_seq, D, N]: h before the first row (absent: 0).  Returns y, or (y, h behind the last rows).
    A sequence's result does not depend on what stands beside it in the batch but for how time is cut into chunks (rounding)."""
    rows = _Rows(dt, "dt", seq_start, lengths)
    u, dt, z = rows.like(u, "u", packed_ok=True), rows.like(dt, "dt"), None if z is None else rows.like(z, "z", packed_ok=True)
    a, N, keep = _scan(rows, u, dt, A, B, C_, D, z, dt_bias, softplus, rows.shape[:-1])
    st = rows.state(state, "state", (rows.n_seq, rows.D, N), rows.param)
    y = rows.out(out)
    end = _torch().empty((rows.n_seq, rows.D, N), dtype=rows.param, device=rows.device) if return_state else None
    a.y, a.zero_outside, a.state_in, a.state_out = _view(y), int(out is None and rows.ragged), _ptr(st), _ptr(end)
    ws = rows.workspace(a, lib.crnn_scan_workspace(C.byref(a), 0))  # noqa: F841
    check(lib.crnn_scan_forward(C.byref(a)))
    return (y, end) if return_state else y


def selective_scan_grad(dy, u, dt, A, B, C_, *, D=None, z=None, dt_bias=None, softplus=True, seq_start=None, lengths=None, state=None, dstate=None):
    """Gradients of selective_scan from dy (and dstate, the gradient of the state it returned): ScanGrads, None where the call had no such input.
    The states are formed again from the inputs; u and z may be checkpoints: the gradients are taken at the values they hold."""
    t = _torch()
    rows = _Rows(dt, "dt", seq_start, lengths)
    u, dt, z = rows.like(u, "u", packed_ok=True), rows.like(dt, "dt"), None if z is None else rows.like(z, "z", packed_ok=True)
    dy = rows.like(dy, "dy")
    a, N, keep = _scan(rows, u, dt, A, B, C_, D, z, dt_bias, softplus, rows.shape[:-1])
    shape = (rows.n_seq, rows.D, N)
    st, dstate = rows.state(state, "state", shape, rows.param), rows.state(dstate, "dstate", shape, rows.param)

    def new(shape, dtype):
        return t.empty(shape, dtype=dtype, device=rows.device)

    du, ddt, dz = rows.out(None), rows.out(None), None if z is None else rows.out(None)
    dB, dC = new(tuple(keep[3].shape), rows.dtype), new(tuple(keep[4].shape), rows.dtype)
    dA, dD = new((rows.D, N), rows.param), None if D is None else new((rows.D,), rows.param)
    db = None if dt_bias is None else new((rows.D,), rows.param)
    ds = None if state is None else new(shape, rows.param)
    if rows.n_seq == 0:
        for x in (du, ddt, dz, dB, dC, dA, dD, db):
            if x is not None:
                x.zero_()
        return ScanGrads(du, ddt, dA, dB.view(B.shape), dC.view(C_.shape), dD, dz, db, ds)
    a.zero_outside = int(rows.ragged)
    a.dy, a.du, a.ddt, a.dz = _view(dy), _view(du), _view(ddt), _view(dz)
    a.dB, a.dC = _map_view(dB)[0], _map_view(dC)[0]
    a.dA, a.dskip, a.ddt_bias = dA.data_ptr(), _ptr(dD), _ptr(db)
    a.state_in, a.dstate_out, a.dstate_in = _ptr(st), _ptr(dstate), _ptr(ds)
    ws = rows.workspace(a, lib.crnn_scan_workspace(C.byref(a), 1))  # noqa: F841
    check(lib.crnn_scan_backward(C.byref(a)))
    return ScanGrads(du, ddt, dA, dB.view(B.shape), dC.view(C_.shape), dD, dz, db, ds)


def selective_scan_step(u, dt, A, B, C_, state, slots=None, *, D=None, z=None, dt_bias=None, softplus=True, out=None):
    """One more row for each of many running sequences: u, dt, z [n, D], B, C [n, G, N] or [n, N], state [n_slots, D, N] updated in place; slots as
    in causal_conv_step.  Returns y [n, D]."""
    t = _torch()
    if dt.ndim != 2:
        raise ValueError(f"dt must be [n, D], not {tuple(dt.shape)}")
    for x, name in ((u, "u"), (z, "z")):
        if isinstance(x, Packed8):
            raise TypeError(f"{name} cannot be an 8-bit checkpoint here")
        if x is not None and (x.shape != dt.shape or x.dtype != dt.dtype or x.device != dt.device):
            raise ValueError(f"{name} must be {tuple(dt.shape)} {dt.dtype} on {dt.device}, not {tuple(x.shape)} {x.dtype} on {x.device}")
    rows = _Rows(dt[:, None], "dt", None, None)
    n = dt.shape[0]
    u, dt, z = _channels(u, "u"), _channels(dt, "dt"), None if z is None else _channels(z, "z")
    a, N, keep = _scan(rows, u, dt, A, B, C_, D, z, dt_bias, softplus, (n,))
    if tuple(state.shape[1:]) != (rows.D, N) or state.ndim != 3 or state.dtype != rows.param or state.device != rows.device or not state.is_contiguous():
        raise ValueError(f"state must be a contiguous [n_slots, {rows.D}, {N}] {rows.param} on {rows.device}")
    slots = _slots(rows, slots, n)
    if slots is None and n > state.shape[0]:
        raise ValueError(f"{n} rows, but the state has {state.shape[0]} slots")
    y = t.empty((n, rows.D), dtype=dt.dtype, device=dt.device) if out is None else out
    if tuple(y.shape) != (n, rows.D) or y.dtype != dt.dtype or y.device != rows.device or y.stride(1) != 1 and rows.D > 1:
        raise ValueError(f"out must be [{n}, {rows.D}] {dt.dtype} on {rows.device} with contiguous channels")
    a.rows, a.y, a.state_out, a.slot, a.n_slots = 1, _view(y), _ptr(state), _ptr(slots), state.shape[0]
    check(lib.crnn_scan_step(C.byref(a)))
    return y


# ---------------------------------------------------------------- checkpoints
def pack8(x):
    """x [..., D] (float32, bfloat16 or float16) in 8 bits: Packed8.  A value comes back within half a code, at most max|x| / 128 of its block of
    32 channels; a block with an infinity or a NaN comes back as NaN."""
    t = _torch()
    if isinstance(x, Packed8) or x.dtype not in (t.float32, t.bfloat16, t.float16):
        raise TypeError(f"pack8: float32, bfloat16 or float16, not {x.dtype}")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError("pack8: x must be [..., D] with D >= 1")
    dev = _on_device(x, "x")
    D = x.shape[-1]
    flat = _channels(x.reshape(-1, D), "x")
    codes = t.empty(x.shape, dtype=t.int8, device=dev)
    scales = t.empty((*x.shape[:-1], -(-D // 32)), dtype=t.uint8, device=dev)
    v = _view(flat)
    check(lib.crnn_pack8(_ordinal(dev), _stream(dev), C.byref(v), flat.shape[0], D, _ptr(codes), _ptr(scales)))
    return Packed8(codes, scales, x.dtype)


def unpack8(p, *, dtype=None, out=None):
    """The values a checkpoint holds, in its own type or in `dtype`, rounded once."""
    t = _torch()
    dev = _on_device(p, "codes")
    dtype = dtype or (p.dtype if out is None else out.dtype)
    if dtype not in (t.float32, t.bfloat16, t.float16):
        raise TypeError(f"unpack8: float32, bfloat16 or float16, not {dtype}")
    y = t.empty(p.shape, dtype=dtype, device=dev) if out is None else out
    if y.shape != p.shape or y.dtype != dtype or y.device != dev or not y.is_contiguous():
        raise ValueError(f"out must be a contiguous {tuple(p.shape)} {dtype} on {dev}")
    D = p.shape[-1]
    v = _view(y.view(-1, D))
    check(lib.crnn_unpack8(_ordinal(dev), _stream(dev), _ptr(p.codes), _ptr(p.scales), y.numel() // D, D, C.byref(v)))
    return y
