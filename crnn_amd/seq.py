"""Sequence operators on the device: a short causal convolution, the selective state space scan and activation checkpoints in 8 bits.

The scan is the linear member of the ODE family this package integrates: a diagonal linear ODE h' = A h + B(t) u(t) with learned rates,
over steps of their own length (an irregular time grid), thousands of channels and rows, with its discrete adjoint.  A step's decay is exact, its
input enters to first order in the step length (delta B u, as in selective state space models; held over the step it would be (exp(delta A) - 1) / A B u).

    causal_conv / causal_conv_grad / causal_conv_step          p[t, d] = bias[d] + sum_j weight[d, j] x[t - W + 1 + j, d];  y = p, or p sigmoid(p)
    selective_scan / selective_scan_grad / selective_scan_step h = exp(delta A) h + delta u B;  y = sum_n C h + D u, or that times z sigmoid(z);
                                                               delta = softplus(dt + dt_bias), or dt + dt_bias
    pack8 / unpack8                                            a row's channels in 8 bits, a power of two as scale per 32 of them

Arrays are torch tensors on an MI355X; the calls enqueue on that device's current stream and do not wait, so that they may be captured into
a graph.  Rows are time, channels are contiguous: dense [n_seq, rows, D] (lengths=: how many rows of each are its own, the others are
padding), or packed [rows, D] with seq_start [n_seq + 1], int32 on the device: sequence s is rows seq_start[s] .. seq_start[s + 1] - 1.
Lengths and offsets are not read by the host: they are clamped to the arrays; offsets may not decrease (entries not in use
repeat the last one), or the results are not defined.  Rows of a result that belong to no sequence are 0, and stay as
they were where the caller gave the array (out=).  Results may not share memory with inputs (refused).  Autograd does not record the calls,
gradients are the *_grad calls: forward calls and steps on tensors that require gradients are refused while it records (call them under
torch.no_grad(), or in the forward of a torch.autograd.Function), and so are forward-mode tangents; the *_grad calls give values that
are not differentiated further.  float32, bfloat16, float16 and float64; weights, rates and scan states are float32
(float64 with float64 data).  A checkpoint (Packed8) may stand for x of the convolution, and for u and z of the scan.
"""
from __future__ import annotations

import ctypes as C
import struct
from collections import namedtuple

from . import _lib as L
from ._lib import ConvArgs, ScanArgs, View, check, lib

ConvGrads = namedtuple("ConvGrads", "x weight bias state")
ScanGrads = namedtuple("ScanGrads", "u dt A B C D z dt_bias state")

_EMULATED = "SIMT-EMULATION" in lib.crnn_build_info().decode()     # the emulated device's memory is the host's


_t = None          # torch, imported by the first call
_DT = {}           # torch's types: ours
_raw_stream = None
_grad_on = None    # torch.is_grad_enabled
_asks = None       # whether one of the arguments is a tensor that requires a gradient
_dual = None       # torch's forward-mode module, if this torch tells whether it is in use
_like = None       # a contiguous tensor of another's shape (and type): half the host time of torch.empty with a shape, a type and a device


def _torch():
    global _t, _raw_stream, _like, _dual, _grad_on, _asks
    if _t is None:
        import torch
        from functools import partial
        _like = partial(torch.empty_like, memory_format=torch.contiguous_format)
        _DT.update({torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16, torch.float64: L.DT_F64})
        _grad_on = torch.is_grad_enabled
        _asks = getattr(torch._C, "_any_requires_grad", None) or (lambda *xs: any(isinstance(x, torch.Tensor) and x.requires_grad for x in xs))
        _dual = torch.autograd.forward_ad if hasattr(torch.autograd.forward_ad, "_current_level") else None
        _t = torch
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
    return _t


def _packer(cls):
    """The struct as one format string: a call fills its arguments with a single pack (the fields one by one take longer than the launch), and
    passes the bytes as they are."""
    codes = {C.c_int32: "i", C.c_int64: "q", C.c_void_p: "P"}

    def fmt(c):
        return "".join(fmt(t) if t is View else codes[t] for _, t in c._fields_)

    f = struct.Struct("@" + fmt(cls))
    if f.size != C.sizeof(cls):
        raise ImportError(f"layout of {cls.__name__}: {f.size} != {C.sizeof(cls)}")
    return f.pack


_pack_conv, _pack_scan, _pack_view = _packer(ConvArgs), _packer(ScanArgs), _packer(View)


def _entry(name, at):
    """An entry point that takes its struct (argument `at`) as bytes."""
    f, known = lib[name], getattr(lib, name)
    f.restype, f.argtypes = known.restype, [C.c_char_p if i == at else t for i, t in enumerate(known.argtypes)]
    return f


_conv_workspace, _conv_forward, _conv_backward, _conv_step = (_entry(f"crnn_conv_{k}", 0) for k in ("workspace", "forward", "backward", "step"))
_scan_workspace, _scan_forward, _scan_backward, _scan_step = (_entry(f"crnn_scan_{k}", 0) for k in ("workspace", "forward", "backward", "step"))
_pack, _unpack = _entry("crnn_pack8", 2), _entry("crnn_unpack8", 6)
_CONV_SIZE, _SCAN_SIZE = C.sizeof(ConvArgs), C.sizeof(ScanArgs)
_ABSENT = (0,) * 8
# a pointer for arrays without elements: "absent" and "empty" differ
_NOTHING = 256


class Packed8:
    """A checkpoint: codes int8 [..., D], scales uint8 [..., ceil(D / 32)] (exponent + 127 of a block of 32 channels), value = code * 2^exponent.
    dtype: the type of the tensor it was made from."""

    __slots__ = ("codes", "scales", "dtype")

    def __init__(self, codes, scales, dtype):
        t = _torch()
        if codes.dtype != t.int8 or scales.dtype != t.uint8:
            raise TypeError("Packed8: codes must be int8 and scales uint8")
        if codes.ndim < 1 or scales.shape != (*codes.shape[:-1], -(-codes.shape[-1] // 32)):
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
    """(device, its ordinal, its current stream)"""
    dev = x.device
    if dev.type != "cuda":
        if _EMULATED and dev.type == "cpu":
            return dev, 0, 0
        raise ValueError(f"{what} must be on the GPU (there is no CPU path)")
    index = dev.index
    return dev, index, _raw_stream(index)


def _ptr(x):
    return 0 if x is None else x.data_ptr()


def _view(x):
    """The fields of a View of [..., rows, D] or [rows, D] with contiguous channels."""
    if x is None:
        return _ABSENT
    if x.__class__ is Packed8:
        c, e = x.codes, x.scales
        s, r = c.stride(), e.stride()
        many = len(s) == 3
        return (c.data_ptr() or _NOTHING, e.data_ptr() or _NOTHING, s[0] if many else 0, s[-2], r[0] if many else 0, r[-2], L.DT_PACKED8, 0)
    s = x.stride()
    return (x.data_ptr() or _NOTHING, 0, s[0] if len(s) == 3 else 0, s[-2], 0, 0, _DT[x.dtype], 0)


def _channels(x):
    """x with contiguous channels (itself where it has them)."""
    if x.__class__ is Packed8 or x.stride(-1) == 1 or x.shape[-1] <= 1:
        return x
    return x.contiguous()


def _recorded(name, *tensors, values=False):
    """Refuses what autograd would lose in silence.  values: a gradient's call, whose results are values even where its inputs require gradients."""
    if not values and _grad_on() and _asks(*tensors):
        raise RuntimeError(f"{name}: autograd does not record this call, an input's gradient would be lost: call it under torch.no_grad() or on detached tensors, and "
                           f"{name.removesuffix('_step')}_grad for the gradient")
    if _dual is not None and _dual._current_level >= 0:
        for x in tensors:
            if x is not None and x.__class__ is not Packed8 and _dual.unpack_dual(x).tangent is not None:
                raise RuntimeError(f"{name}: forward-mode derivatives are not computed, an input's tangent would be lost")


class _Rows:
    """What the arrays of one call have in common: type, device, sequences and rows."""

    __slots__ = ("packed", "dtype", "code", "device", "ordinal", "stream", "shape", "D", "param", "n_seq", "rows", "start", "len", "ragged")

    def __init__(self, x, name, seq_start=None, lengths=None, step=False):
        t = _torch()
        packed = self.packed = seq_start is not None
        if x.__class__ is Packed8 and name != "x":
            raise TypeError(f"{name} cannot be an 8-bit checkpoint here")
        if packed and lengths is not None:
            raise ValueError("seq_start (packed rows) and lengths (a padded batch) exclude each other")
        if x.ndim != (2 if packed or step else 3):
            raise ValueError(f"{name} must be {'[n, D]' if step else '[rows, D] (packed)' if packed else '[n_seq, rows, D]'}, not {tuple(x.shape)}")
        code = _DT.get(x.dtype)
        if code is None:
            raise TypeError(f"{name}: float32, bfloat16, float16 or float64, not {x.dtype}")
        self.dtype, self.code, self.shape = x.dtype, code, x.shape
        self.device, self.ordinal, self.stream = _on_device(x, name)
        self.D = x.shape[-1]
        if self.D < 1:
            raise ValueError(f"{name} has no channels")
        self.param = t.float64 if code == L.DT_F64 else t.float32
        self.start = self.len = 0
        if packed:
            self.start = self._index(seq_start, "seq_start")
            self.n_seq, self.rows = seq_start.shape[0] - 1, x.shape[0]
            if self.n_seq < 0:
                raise ValueError("seq_start is empty")
        else:
            self.n_seq, self.rows = x.shape[0], 1 if step else x.shape[1]
            if lengths is not None:
                self.len = self._index(lengths, "lengths") if self.n_seq else 0
                if lengths.shape[0] != self.n_seq:
                    raise ValueError(f"lengths has {lengths.shape[0]} entries for {self.n_seq} sequences")
        self.ragged = int(packed or lengths is not None)

    def _index(self, idx, what):
        if idx.dtype != _t.int32 or idx.ndim != 1 or idx.device != self.device or not idx.is_contiguous():
            raise ValueError(f"{what} must be a contiguous int32 vector on {self.device}")
        return idx.data_ptr()

    def like(self, x, name, packed_ok=False):
        if x.__class__ is Packed8 and not packed_ok:
            raise TypeError(f"{name} cannot be an 8-bit checkpoint here")
        if x.shape != self.shape or x.dtype != self.dtype or x.device != self.device:
            raise ValueError(f"{name} must be {tuple(self.shape)} {self.dtype} on {self.device}, not {tuple(x.shape)} {x.dtype} on {x.device}")
        return _channels(x)

    def weight(self, x, name, shape):
        """A parameter in the type parameters have here."""
        if x is None:
            return None
        given = x.dtype is self.param
        if x.shape != shape or x.device != self.device or not (given or x.dtype.is_floating_point):
            raise ValueError(f"{name} must be {shape} on {self.device}, not {tuple(x.shape)} {x.dtype} on {x.device}")
        if not given:
            x = x.to(self.param)
        return x if x.is_contiguous() else x.contiguous()

    def state(self, x, name, shape, dtype):
        if x is None:
            return None
        if x.shape != shape or x.dtype != dtype or x.device != self.device:
            raise ValueError(f"{name} must be {shape} {dtype} on {self.device}, not {tuple(x.shape)} {x.dtype} on {x.device}")
        return x if x.is_contiguous() else x.contiguous()

    def new(self, shape, dtype):
        return _t.empty(shape, dtype=dtype, device=self.device)

    def out(self, given, shape, *inputs):
        """The result's array.  inputs: arrays of which other rows, or other lanes of the same row, are read after a row of the result is written."""
        if given is None:
            x = inputs[0]
            return _like(x) if x.__class__ is not Packed8 else _t.empty(shape, dtype=self.dtype, device=self.device)
        if given.shape != shape or given.dtype != self.dtype or given.device != self.device or given.stride(-1) != 1 and self.D > 1:
            raise ValueError(f"out must be {tuple(shape)} {self.dtype} on {self.device} with contiguous channels")
        if given.numel() and any(x is not None and (x.codes if x.__class__ is Packed8 else x).data_ptr() == given.data_ptr() for x in inputs):
            raise ValueError("out may not be an input")
        return given


def _none(y, out, end):
    """The result for no sequences: all rows of y are outside of them."""
    if out is None:
        y.zero_()
    return y if end is None else (y, end)


def _slots(rows, slots, n, n_slots):
    if slots is None:
        if n > n_slots:
            raise ValueError(f"{n} rows, but the state has {n_slots} slots")
        return 0
    if slots.dtype != _t.int32 or slots.shape != (n,) or slots.device != rows.device or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int32 vector of {n} entries on {rows.device}")
    return slots.data_ptr() or _NOTHING


_needs = {}        # bytes of workspace by sizes: a call of sizes seen before need not ask


def _workspace(key, ask):
    """The bytes the call needs.  The memory itself is the call's own, from torch's allocator on the call's stream (a graph under capture keeps its)."""
    need = _needs.get(key)
    if need is None:
        need = ask()
        if need < 0:
            check(-1)
        if len(_needs) >= 4096:
            _needs.clear()
        _needs[key] = need
    return need


# ---------------------------------------------------------------- convolution
def _taps(weight):
    if weight.ndim != 2 or not 1 <= weight.shape[1] <= L.SEQ_MAX_TAPS:
        raise ValueError(f"weight must be [D, W] with 1 <= W <= {L.SEQ_MAX_TAPS}, not {tuple(weight.shape)}")
    return weight.shape[1]


def _conv_args(r, W, silu, rows, zero, weight, bias, x, y, state_in, state_out, dy=_ABSENT, dx=_ABSENT, dstate_out=_ABSENT, dstate_in=_ABSENT, dweight=0, dbias=0, slot=0,
               n_slots=0, ws=0, ws_bytes=0, n_seq=None):
    return _pack_conv(
        _CONV_SIZE, r.ordinal, r.stream, r.n_seq if n_seq is None else n_seq, r.D, W, 1 if silu else 0, rows, r.start, r.len, r.code, zero, _ptr(weight), _ptr(bias), *x, *y,
        *state_in, *state_out, *dy, *dx, *dstate_out, *dstate_in, dweight, dbias, slot, n_slots, ws, ws_bytes)


def causal_conv(x, weight, bias=None, *, silu=False, seq_start=None, lengths=None, state=None, return_state=False, out=None):
    """The convolution of each sequence with its own past.  weight [D, W]: the last tap meets the row itself.  state [n_seq, W - 1, D]: the rows
    before the first (absent: 0).  Returns y, or (y, the state behind the last rows)."""
    r = _Rows(x, "x", seq_start, lengths)
    _recorded("causal_conv", x, weight, bias, state, out)
    x = _channels(x)
    W = _taps(weight)
    D, shape = r.D, (r.n_seq, W - 1, r.D)
    weight, bias, state = r.weight(weight, "weight", (D, W)), r.weight(bias, "bias", (D,)), r.state(state, "state", shape, r.dtype)
    y = r.out(out, r.shape, x)
    end = (r.new(shape, r.dtype) if state is None else _like(state)) if return_state else None
    if r.n_seq == 0:
        return _none(y, out, end)
    a = _conv_args(r, W, silu, r.rows, r.ragged if out is None else 0, weight, bias, _view(x), _view(y), _view(state) if W > 1 else _ABSENT, _view(end) if W > 1 else _ABSENT)
    if _conv_forward(a):
        check(-1)
    return (y, end) if return_state else y


def causal_conv_grad(dy, x, weight, bias=None, *, silu=False, seq_start=None, lengths=None, state=None, dstate=None):
    """Gradients of causal_conv from dy (and dstate, the gradient of the state it returned): ConvGrads(x, weight, bias, state); bias and state are
    None where the call had none.  x may be a checkpoint: the gradient is taken at the values it holds."""
    r = _Rows(x, "x", seq_start, lengths)
    _recorded("causal_conv_grad", dy, x, weight, bias, state, dstate, values=True)
    x, dy = _channels(x), r.like(dy, "dy")
    W = _taps(weight)
    D, shape = r.D, (r.n_seq, W - 1, r.D)
    weight, bias = r.weight(weight, "weight", (D, W)), r.weight(bias, "bias", (D,))
    state, dstate = r.state(state, "state", shape, r.dtype), r.state(dstate, "dstate", shape, r.dtype)
    dx, dw = _like(dy), _like(weight)
    db, ds = None if bias is None else _like(bias), None if state is None else _like(state)
    if r.n_seq == 0:
        return ConvGrads(dx.zero_(), dw.zero_(), None if db is None else db.zero_(), ds)

    def args(ws=0, need=0):
        v = (lambda t: _view(t) if W > 1 else _ABSENT)
        return _conv_args(r, W, silu, r.rows, r.ragged, weight, bias, _view(x), _ABSENT, v(state), _ABSENT, _view(dy), _view(dx), v(dstate), v(ds), dw.data_ptr(), _ptr(db), 0, 0,
                          ws, need)

    need = _workspace(("conv", r.n_seq, r.rows, r.packed, D, W, r.code), lambda: _conv_workspace(args()))
    ws = r.new(max(need, 1), _t.uint8)
    if _conv_backward(args(ws.data_ptr(), need)):
        check(-1)
    return ConvGrads(dx, dw, db, ds)


def causal_conv_step(x, weight, bias, state, slots=None, *, silu=False, out=None):
    """One more row for each of many running sequences: x [n, D], state [n_slots, W - 1, D] moved up in place.  slots [n], int32: row r continues
    the state in slots[r] (absent: in r).  A slot outside the state: the row is padding, its result 0.  Rows that name the same slot are
    consecutive rows of its sequence, in their order.  Returns y [n, D]."""
    if x.__class__ is Packed8:
        raise TypeError("x cannot be an 8-bit checkpoint here")
    r = _Rows(x, "x", step=True)
    _recorded("causal_conv_step", x, weight, bias, state, out)
    n, D = x.shape
    W = _taps(weight)
    weight, bias = r.weight(weight, "weight", (D, W)), r.weight(bias, "bias", (D,))
    if state.ndim != 3 or state.shape[1:] != (W - 1, D) or state.dtype != r.dtype or state.device != r.device or (D > 1 and W > 1 and state.stride(2) != 1):
        raise ValueError(f"state must be [n_slots, {W - 1}, {D}] {r.dtype} on {r.device} with contiguous channels")
    slot = _slots(r, slots, n, state.shape[0])
    x, y = _channels(x), r.out(out, x.shape, x, state)
    a = _conv_args(r, W, silu, 1, 0, weight, bias, _view(x), _view(y), _view(state) if W > 1 else _ABSENT, _ABSENT, slot=slot, n_slots=state.shape[0], n_seq=n)
    if _conv_step(a):
        check(-1)
    return y


# ---------------------------------------------------------------- scan
def _map(r, m, name, lead):
    """The View fields of B or C [*lead, G, N] (or without G), its strides between groups and states, and (G, N)."""
    k = len(lead)
    if m.ndim == k + 1:
        G, sg = 1, 0
    elif m.ndim == k + 2:
        G, sg = m.shape[k], m.stride(k)
    else:
        G = 0
    if G == 0 or m.shape[:k] != lead or m.dtype != r.dtype or m.device != r.device:
        raise ValueError(f"{name} must be {(*lead, 'G', 'N')} (or without G) {r.dtype} on {r.device}, not {tuple(m.shape)} {m.dtype} on {m.device}")
    s = m.stride()
    return (m.data_ptr() or _NOTHING, 0, s[0] if k == 2 else 0, s[k - 1], 0, 0, r.code, 0), sg, s[-1], G, m.shape[-1]


def _scan_params(r, A, B, C_, D, dt_bias, lead):
    if A.ndim != 2 or A.shape[0] != r.D or not 1 <= A.shape[1] <= L.SEQ_MAX_STATES:
        raise ValueError(f"A must be [{r.D}, N] with 1 <= N <= {L.SEQ_MAX_STATES}, not {tuple(A.shape)}")
    N = A.shape[1]
    b, bg, bn, G, nb = _map(r, B, "B", lead)
    c, cg, cn, Gc, nc = _map(r, C_, "C", lead)
    if G != Gc or nb != N or nc != N:
        raise ValueError(f"B and C must both end in [G, {N}], not {tuple(B.shape)} and {tuple(C_.shape)}")
    if r.D % G:
        raise ValueError(f"the {r.D} channels do not fall into {G} groups")
    return N, G, r.weight(A, "A", (r.D, N)), r.weight(D, "D", (r.D,)), r.weight(dt_bias, "dt_bias", (r.D,)), (*b, *c, bg, bn, cg, cn)


def _scan_args(r, N, G, rows, zero, softplus, A, D, dt_bias, u, dt, z, y, maps, state_in, state_out, grads=_ABSENT * 6 + (0,) * 3, dstate_out=0, dstate_in=0, slot=0, n_slots=0,
               ws=0, ws_bytes=0, n_seq=None):
    return _pack_scan(
        _SCAN_SIZE, r.ordinal, r.stream, r.n_seq if n_seq is None else n_seq, r.D, N, G, rows, r.start, r.len, r.code, zero, 1 if softplus else 0, 0, _ptr(A), _ptr(D), _ptr(dt_bias),
        *u, *dt, *z, *y, *maps, state_in, state_out, *grads, dstate_out, dstate_in, slot, n_slots, ws, ws_bytes)


def selective_scan(u, dt, A, B, C_, *, D=None, z=None, dt_bias=None, softplus=True, seq_start=None, lengths=None, state=None, return_state=False, out=None):
    """The scan of each sequence.  u, dt, z as described above; A [D, N]; B, C [.., G, N] or [.., N] (one group) beside u's rows, channel d in group
    d // (D / G); D, dt_bias [D]; state [n_seq, D, N]: h before the first row (absent: 0).  Returns y, or (y, h behind the last rows).
    What stands beside a sequence in its batch changes its result by rounding only (how time is cut into chunks)."""
    r = _Rows(dt, "dt", seq_start, lengths)
    _recorded("selective_scan", u, dt, A, B, C_, D, z, dt_bias, state, out)
    u, dt, z = r.like(u, "u", True), _channels(dt), None if z is None else r.like(z, "z", True)
    N, G, A, D, dt_bias, maps = _scan_params(r, A, B, C_, D, dt_bias, r.shape[:-1])
    shape = (r.n_seq, r.D, N)
    state = r.state(state, "state", shape, r.param)
    y = r.out(out, r.shape, dt, u, z, B, C_)
    end = (r.new(shape, r.param) if state is None else _like(state)) if return_state else None
    if r.n_seq == 0:
        return _none(y, out, end)

    def args(ws=0, need=0):
        return _scan_args(r, N, G, r.rows, r.ragged if out is None else 0, softplus, A, D, dt_bias, _view(u), _view(dt), _view(z), _view(y), maps, _ptr(state), _ptr(end), ws=ws,
                          ws_bytes=need)

    need = _workspace((0, r.n_seq, r.rows, r.packed, r.D, N, G, r.code, u.__class__ is Packed8, z is None or z.__class__ is Packed8, z is None),
                      lambda: _scan_workspace(args(), 0))
    ws = r.new(need, _t.uint8) if need else None
    if _scan_forward(args(_ptr(ws), need)):
        check(-1)
    return (y, end) if return_state else y


def selective_scan_grad(dy, u, dt, A, B, C_, *, D=None, z=None, dt_bias=None, softplus=True, seq_start=None, lengths=None, state=None, dstate=None):
    """Gradients of selective_scan from dy (and dstate, the gradient of the state it returned): ScanGrads, None where the call had no such input.
    The states are formed again from the inputs; u and z may be checkpoints: the gradients are taken at the values they hold."""
    r = _Rows(dt, "dt", seq_start, lengths)
    _recorded("selective_scan_grad", dy, u, dt, A, B, C_, D, z, dt_bias, state, dstate, values=True)
    u, dt, z, dy = r.like(u, "u", True), _channels(dt), None if z is None else r.like(z, "z", True), r.like(dy, "dy")
    N, G, A, D, dt_bias, maps = _scan_params(r, A, B, C_, D, dt_bias, r.shape[:-1])
    shape = (r.n_seq, r.D, N)
    state, dstate = r.state(state, "state", shape, r.param), r.state(dstate, "dstate", shape, r.param)
    du, ddt, dz, dB, dC, dA = _like(dt), _like(dt), None if z is None else _like(dt), _like(B), _like(C_), _like(A)
    dD, db, ds = None if D is None else _like(D), None if dt_bias is None else _like(dt_bias), None if state is None else _like(state)
    if r.n_seq == 0:
        for x in (du, ddt, dz, dB, dC, dA, dD, db):
            if x is not None:
                x.zero_()
        return ScanGrads(du, ddt, dA, dB, dC, dD, dz, db, ds)
    lead = r.shape[:-1]
    grads = (*_view(dy), *_view(du), *_view(ddt), *_view(dz), *_map(r, dB, "dB", lead)[0], *_map(r, dC, "dC", lead)[0], dA.data_ptr(), _ptr(dD), _ptr(db))

    def args(ws=0, need=0):
        return _scan_args(r, N, G, r.rows, r.ragged, softplus, A, D, dt_bias, _view(u), _view(dt), _view(z), _ABSENT, maps, _ptr(state), 0, grads, _ptr(dstate), _ptr(ds), ws=ws,
                          ws_bytes=need)

    need = _workspace((1, r.n_seq, r.rows, r.packed, r.D, N, G, r.code, u.__class__ is Packed8, z is None or z.__class__ is Packed8, z is None),
                      lambda: _scan_workspace(args(), 1))
    ws = r.new(max(need, 1), _t.uint8)
    if _scan_backward(args(ws.data_ptr(), need)):
        check(-1)
    return ScanGrads(du, ddt, dA, dB, dC, dD, dz, db, ds)


def selective_scan_step(u, dt, A, B, C_, state, slots=None, *, D=None, z=None, dt_bias=None, softplus=True, out=None):
    """One more row for each of many running sequences: u, dt, z [n, D], B, C [n, G, N] or [n, N], state [n_slots, D, N] updated in place; slots as
    in causal_conv_step.  Returns y [n, D]."""
    r = _Rows(dt, "dt", step=True)
    _recorded("selective_scan_step", u, dt, A, B, C_, D, z, dt_bias, state, out)
    n = r.n_seq
    u, dt, z = r.like(u, "u"), _channels(dt), None if z is None else r.like(z, "z")
    N, G, A, D, dt_bias, maps = _scan_params(r, A, B, C_, D, dt_bias, (n,))
    if state.ndim != 3 or state.shape[1:] != (r.D, N) or state.dtype != r.param or state.device != r.device or not state.is_contiguous():
        raise ValueError(f"state must be a contiguous [n_slots, {r.D}, {N}] {r.param} on {r.device}")
    slot = _slots(r, slots, n, state.shape[0])
    y = r.out(out, dt.shape, dt, u, z, B, C_, state)
    a = _scan_args(r, N, G, 1, 0, softplus, A, D, dt_bias, _view(u), _view(dt), _view(z), _view(y), maps, 0, state.data_ptr(), slot=slot, n_slots=state.shape[0], n_seq=n)
    if _scan_step(a):
        check(-1)
    return y


# ---------------------------------------------------------------- checkpoints
def pack8(x):
    """x [..., D] (float32, bfloat16 or float16) in 8 bits: Packed8.  A value comes back within half a code, at most max|x| / 127.5 of its block of
    32 channels, or 2^-128 where that is more (within a code, max|x| / 127.5, where max|x| is within 0.4 % of the type's largest); a block with an infinity or a NaN comes back as NaN."""
    t = _torch()
    if x.__class__ is Packed8 or _DT.get(x.dtype) not in (L.DT_F32, L.DT_BF16, L.DT_F16):
        raise TypeError(f"pack8: float32, bfloat16 or float16, not {x.dtype}")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError("pack8: x must be [..., D] with D >= 1")
    dev, ordinal, stream = _on_device(x, "x")
    shape, D = x.shape, x.shape[-1]
    p = Packed8.__new__(Packed8)
    p.codes, p.dtype = _like(x, dtype=t.int8), x.dtype
    p.scales = t.empty((*shape[:-1], -(-D // 32)), dtype=t.uint8, device=dev)
    flat = _channels(x if x.ndim == 2 else x.reshape(p.codes.numel() // D, D))
    if _pack(ordinal, stream, _pack_view(*_view(flat)), flat.shape[0], D, p.codes.data_ptr(), p.scales.data_ptr()):
        check(-1)
    return p


def unpack8(p, *, dtype=None, out=None):
    """The values a checkpoint holds, in its own type or in `dtype`, rounded once."""
    _torch()
    dev, ordinal, stream = _on_device(p, "codes")
    if dtype is None:
        dtype = p.dtype if out is None else out.dtype
    if _DT.get(dtype) not in (L.DT_F32, L.DT_BF16, L.DT_F16):
        raise TypeError(f"unpack8: float32, bfloat16 or float16, not {dtype}")
    y = _like(p.codes, dtype=dtype) if out is None else out
    if y.shape != p.shape or y.dtype != dtype or y.device != dev or not y.is_contiguous():
        raise ValueError(f"out must be a contiguous {tuple(p.shape)} {dtype} on {dev}")
    D = p.shape[-1]
    v = (y.data_ptr() or _NOTHING, 0, 0, D, 0, 0, _DT[dtype], 0)
    if _unpack(ordinal, stream, p.codes.data_ptr(), p.scales.data_ptr(), y.numel() // D, D, _pack_view(*v)):
        check(-1)
    return y
