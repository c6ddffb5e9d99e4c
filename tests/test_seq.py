"""The sequence operators (crnn_amd.seq) against plain implementations in 64 bits: convolution, scan, their gradients and single steps,
8-bit checkpoints, refusals, and a run of them together.

Tolerances.  A result of type T is rounded once: half a unit, finfo(T).eps / 2 relative to it.  The arithmetic before is in float32 (float64): a
sum of n products is off by at most about (n + 2) eps / 2 of the sum of their magnitudes, the exponentials and reciprocals by a few eps of
theirs; a recurrence adds each row's share, weighted by decays below one.  So every result is allowed half a unit of its own type of itself
plus `k` eps of the compute type of the *scale* it was summed at (the same formula with every term's magnitude, computed beside it), with k
the number of roundings a term meets: see `check`.  The device tests also run on the emulated device (tests/test_simt_emulation_seq.py).
"""
import math
import os
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from crnn_amd import seq  # noqa: E402
from crnn_amd import _lib as L  # noqa: E402

DEV = "cpu" if seq._EMULATED else "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "f64": torch.float64}
gpu = pytest.mark.gpu


def rnd(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).to(dtype).to(DEV)


def param_of(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def check(got, want, scale, k, what):
    assert got is not None and tuple(got.shape) == tuple(want.shape), (what, None if got is None else got.shape, want.shape)
    own = torch.finfo(got.dtype)
    eps = torch.finfo(param_of(got.dtype)).eps
    g, w, s = got.detach().cpu().double(), want.detach().cpu().double(), scale.detach().cpu().double()
    # float16 / bfloat16 below the normal range: half the spacing there
    limit = own.eps / 2 * (w.abs() + k * eps * s) + k * eps * s + own.smallest_normal * own.eps
    bad = ~((g - w).abs() <= limit)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((g - w).abs() / limit)[bad].max()):.3g} of the limit"


# ---------------------------------------------------------------- plain implementations, float64 on the CPU, sequence by sequence
def spans(B, Lr, starts=None, lens=None):
    """[(rows of the flat array)] of the sequences."""
    if starts is not None:
        return [(int(a), int(b)) for a, b in zip(starts[:-1], starts[1:])]
    return [(s * Lr, s * Lr + (Lr if lens is None else int(lens[s]))) for s in range(B)]


def sig(x):
    return 1 / (1 + torch.exp(-x))


def plain_conv(x, w, b, silu, spans_, state, dy=None, dstate=None):
    """x [rows, D]; everything float64.  Returns values, and beside each the scale its terms add up to."""
    D, W = w.shape
    bias = torch.zeros(D, dtype=torch.float64) if b is None else b
    y, ys = torch.zeros_like(x), torch.zeros_like(x)
    n = len(spans_)
    st = torch.zeros(n, W - 1, D, dtype=torch.float64) if state is None else state
    out = torch.zeros(n, W - 1, D, dtype=torch.float64)
    dx, dxs = torch.zeros_like(x), torch.zeros_like(x)
    dw, dws, db, dbs = (torch.zeros(D, W, dtype=torch.float64), torch.zeros(D, W, dtype=torch.float64), torch.zeros(D, dtype=torch.float64), torch.zeros(D, dtype=torch.float64))
    dst, dsts = torch.zeros_like(out), torch.zeros_like(out)
    for s, (lo, hi) in enumerate(spans_):
        line = torch.cat([st[s], x[lo:hi]])
        n_ = hi - lo
        p = sum((w[:, j] * line[j:j + n_] for j in range(W)), torch.zeros(n_, D, dtype=torch.float64)) + bias
        ps = sum(((w[:, j] * line[j:j + n_]).abs() for j in range(W)), torch.zeros(n_, D, dtype=torch.float64)) + bias.abs()
        y[lo:hi] = p * sig(p) if silu else p
        ys[lo:hi] = ps * (1 + ps) if silu else ps
        out[s] = line[n_:]
        if dy is None:
            continue
        act = sig(p) * (1 + p * (1 - sig(p))) if silu else torch.ones_like(p)
        dp, dps = dy[lo:hi] * act, dy[lo:hi].abs() * (1 + ps) ** 2 if silu else dy[lo:hi].abs()
        dl, dls = torch.zeros_like(line), torch.zeros_like(line)
        if dstate is not None:
            dl[n_:] += dstate[s]
            dls[n_:] += dstate[s].abs()
        for j in range(W):
            dl[j:j + n_] += dp * w[:, j]
            dls[j:j + n_] += dps * w[:, j].abs()
            dw[:, j] += (dp * line[j:j + n_]).sum(0)
            dws[:, j] += (dps * line[j:j + n_].abs()).sum(0)
        db += dp.sum(0)
        dbs += dps.sum(0)
        dst[s], dsts[s], dx[lo:hi], dxs[lo:hi] = dl[:W - 1], dls[:W - 1], dl[W - 1:], dls[W - 1:]
    return dict(y=(y, ys), state=(out, out.abs()), dx=(dx, dxs), dw=(dw, dws), db=(db, dbs), dstate=(dst, dsts))


def plain_scan(u, dt, A, B, C, D, z, bias, softplus, spans_, state, dy=None, dstate=None, mag=None):
    """u, dt, z [rows, D], B, C [rows, G, N]; everything float64.  mag: the scale `state` was summed at, where that is more than its size."""
    T, Dn = u.shape
    G, N = B.shape[1:]
    of = torch.arange(Dn) // (Dn // G)
    n = len(spans_)
    pre = dt + (0 if bias is None else bias)
    dl = torch.clamp(pre, min=0) + torch.log1p(torch.exp(-pre.abs())) if softplus else pre
    h0 = torch.zeros(n, Dn, N, dtype=torch.float64) if state is None else state
    gate = z * sig(z) if z is not None else None
    skip = torch.zeros(Dn, dtype=torch.float64) if D is None else D
    v, vs = torch.zeros(T, Dn, dtype=torch.float64), torch.zeros(T, Dn, dtype=torch.float64)
    hs, hm = torch.zeros(T, Dn, N, dtype=torch.float64), torch.zeros(T, Dn, N, dtype=torch.float64)
    m0 = h0.abs() if mag is None else mag
    end, ends = h0.clone(), m0.clone()
    for s, (lo, hi) in enumerate(spans_):
        h, m = h0[s], m0[s]
        for t in range(lo, hi):
            e = dl[t][:, None] * A
            a = torch.exp(e)
            x = (dl[t] * u[t])[:, None] * B[t][of]
            # the exponent's rounding weighs |e|
            h, m = a * h + x, a * m * (1 + e.abs()) + x.abs()
            hs[t], hm[t] = h, m
            v[t] = (h * C[t][of]).sum(1) + skip * u[t]
            vs[t] = (m * C[t][of].abs()).sum(1) + (skip * u[t]).abs()
        end[s], ends[s] = h, m
    y, ys = (v * gate, vs * gate.abs() * (1 + z.abs())) if gate is not None else (v, vs)
    r = dict(y=(y, ys), state=(end, ends))
    if dy is None:
        return r
    z64 = lambda *s_: torch.zeros(*s_, dtype=torch.float64)  # noqa: E731
    g = {k: [z64(*sh), z64(*sh)] for k, sh in dict(u=(T, Dn), dt=(T, Dn), A=(Dn, N), B=(T, G, N), C=(T, G, N), D=(Dn,), dt_bias=(Dn,), state=(n, Dn, N)).items()}
    rr = dy * gate if gate is not None else dy
    rs = rr.abs() * (1 + z.abs()) if gate is not None else rr.abs()
    for s, (lo, hi) in enumerate(spans_):
        q = z64(Dn, N) if dstate is None else dstate[s].clone()
        qs = q.abs()
        for t in range(hi - 1, lo - 1, -1):
            e = dl[t][:, None] * A
            a = torch.exp(e)
            hp, hpm = (hs[t - 1], hm[t - 1]) if t > lo else (h0[s], h0[s].abs())
            Bt, Ct = B[t][of], C[t][of]
            q, qs = q + rr[t][:, None] * Ct, qs + rs[t][:, None] * Ct.abs()
            ah, ahm = a * hp, a * hpm * (1 + e.abs())
            x = (dl[t] * u[t])[:, None]
            for key, val, mag in (("C", rr[t][:, None] * hs[t], rs[t][:, None] * hm[t]), ("B", q * x, qs * x.abs())):
                g[key][0][t] = val.view(G, Dn // G, N).sum(1)
                g[key][1][t] = mag.view(G, Dn // G, N).sum(1)
            qb, qbs = (q * Bt).sum(1), (qs * Bt.abs()).sum(1)
            g["u"][0][t], g["u"][1][t] = qb * dl[t] + rr[t] * skip, qbs * dl[t].abs() + rs[t] * skip.abs()
            g["A"][0] += q * ah * dl[t][:, None]
            g["A"][1] += qs * ahm * dl[t].abs()[:, None]
            dd, dds = (q * ah * A).sum(1) + qb * u[t], (qs * ahm * A.abs()).sum(1) + qbs * u[t].abs()
            if softplus:
                dd, dds = dd * sig(pre[t]), dds * sig(pre[t]) * (1 + pre[t].abs())
            g["dt"][0][t], g["dt"][1][t] = dd, dds
            g["D"][0] += rr[t] * u[t]
            g["D"][1] += rs[t] * u[t].abs()
            q, qs = q * a, qs * a * (1 + e.abs())
        g["state"][0][s], g["state"][1][s] = q, qs
    g["dt_bias"] = [g["dt"][0].sum(0), g["dt"][1].sum(0)]
    if z is not None:
        g["z"] = [dy * v * sig(z) * (1 + z * (1 - sig(z))), dy.abs() * vs * (1 + z.abs())]
    r["grad"] = g
    return r


def plain_codes(x, top=2.0 ** 127):
    """One block at a time; (codes, scale bytes).  From `top`, the last binade of the type, on 128 would come back as infinity."""
    T, D = x.shape
    nb = -(-D // 32)
    q, e = np.zeros((T, D), np.int64), np.zeros((T, nb), np.int64)
    for t in range(T):
        for k in range(nb):
            b = x[t, 32 * k:32 * k + 32].double().numpy()
            if not np.isfinite(b).all():
                e[t, k] = 255
                continue
            m = np.abs(b).max()
            p = -127 if m == 0 else max(math.frexp(m)[1] - 7, -127)
            if np.rint(m / 2.0 ** p) > 127 and m < top:
                p += 1
            q[t, 32 * k:32 * k + len(b)], e[t, k] = np.clip(np.rint(b / 2.0 ** p), -127, 127), p + 127
    return torch.from_numpy(q).to(torch.int8), torch.from_numpy(e).to(torch.uint8)


def cpu64(x):
    return None if x is None else x.detach().cpu().double()


# ---------------------------------------------------------------- layouts
#: name -> (sequences, rows, lengths or None, packed lengths or None)
LAYOUTS = {
    "one_row": (1, 1, None, None),
    "dense": (2, 37, None, None),
    "padded": (3, 40, [40, 0, 33], None),
    "packed": (None, None, None, [0, 1, 65, 3, 0, 32]),
    "gap": (None, None, None, [5, 31]),     # rows in front of and behind the sequences
}


def layout(name):
    """(shape of the leading dimensions, seq keyword arguments, spans in the flat rows, rows outside)"""
    B, Lr, lens, packed = LAYOUTS[name]
    if packed is None:
        kw = {} if lens is None else dict(lengths=torch.tensor(lens, dtype=torch.int32, device=DEV))
        sp = spans(B, Lr, None, lens)
        lead = (B, Lr)
    else:
        front, behind = (4, 7) if name == "gap" else (0, 0)
        starts = np.concatenate([[0], np.cumsum(packed)]) + front
        lead = (int(starts[-1]) + behind,)
        kw = dict(seq_start=torch.tensor(starts, dtype=torch.int32, device=DEV))
        sp = spans(None, None, starts)
    inside = torch.zeros(math.prod(lead), dtype=torch.bool)
    for lo, hi in sp:
        inside[lo:hi] = True
    return lead, kw, sp, ~inside


def poison(x, outside, rows_dim):
    """NaN in the rows that belong to no sequence: they may not be looked at."""
    x.view(-1, *x.shape[rows_dim:])[outside.to(x.device)] = float("nan")
    return x


def strided(x, pad):
    """The same values with rows `pad` elements further apart (pad odd: rows whose alignment changes)."""
    wide = torch.full((*x.shape[:-1], x.shape[-1] + pad), 7.0, dtype=x.dtype, device=x.device)
    wide[..., :x.shape[-1]] = x
    return wide[..., :x.shape[-1]]


# ---------------------------------------------------------------- convolution
CONV = [("one_row", "f32", 5, 4, True, True, 0), ("dense", "bf16", 64, 4, True, True, 0), ("dense", "f32", 260, 3, False, False, 3), ("padded", "f16", 72, 4, True, False, 0),
        ("packed", "bf16", 130, 4, True, True, 1), ("packed", "f64", 20, 2, True, True, 0), ("gap", "f32", 12, 8, True, True, 0), ("packed", "f16", 33, 1, True, True, 5),
        ("padded", "f64", 8, 5, False, True, 0), ("packed", "f32", 516, 6, True, True, 4)]


def conv_case(lay, dtype, D, W, silu, bias, pad, seed=0):
    g = torch.Generator().manual_seed(seed + D + W)
    lead, kw, sp, outside = layout(lay)
    dt = DT[dtype]
    x = strided(poison(rnd(g, *lead, D, dtype=dt), outside, len(lead)), pad) if pad else poison(rnd(g, *lead, D, dtype=dt), outside, len(lead))
    c = dict(x=x, w=rnd(g, D, W, dtype=param_of(dt), scale=0.5), b=rnd(g, D, dtype=param_of(dt)) if bias else None, dy=poison(rnd(g, *lead, D, dtype=dt), outside, len(lead)),
             state=rnd(g, len(sp), W - 1, D, dtype=dt), dstate=rnd(g, len(sp), W - 1, D, dtype=dt), silu=silu, kw=kw, spans=sp, outside=outside, D=D)
    return c


def rows_of(x):
    return cpu64(x).reshape(-1, x.shape[-1])


@gpu
@pytest.mark.parametrize("lay,dtype,D,W,silu,bias,pad", CONV)
@pytest.mark.parametrize("with_state", [True, False])
def test_conv_forward(lay, dtype, D, W, silu, bias, pad, with_state):
    c = conv_case(lay, dtype, D, W, silu, bias, pad)
    st = c["state"] if with_state else None
    y, end = seq.causal_conv(c["x"], c["w"], c["b"], silu=silu, state=st, return_state=True, **c["kw"])
    p = plain_conv(torch.nan_to_num(rows_of(c["x"])), cpu64(c["w"]), cpu64(c["b"]), silu, c["spans"], cpu64(st))
    # a product and a sum per tap, the bias, exponential + reciprocal + products of the gate
    check(y.reshape(-1, D), *p["y"], 3 * W + 10, "y")
    assert torch.equal(end.cpu().double(), p["state"][0])
    assert bool((y.reshape(-1, D).cpu()[c["outside"]] == 0).all())
    # an array of the caller's keeps what stands outside the sequences
    own = torch.full_like(y, 3.0)
    assert seq.causal_conv(c["x"], c["w"], c["b"], silu=silu, state=st, out=own, **c["kw"]) is own
    assert bool((own.reshape(-1, D).cpu()[c["outside"]] == 3).all())
    assert torch.equal(own.reshape(-1, D).cpu()[~c["outside"]], y.reshape(-1, D).cpu()[~c["outside"]])


def held(x, packed):
    """(what the call gets, the values that holds)"""
    if not packed:
        return x, x
    p = seq.pack8(torch.nan_to_num(x))
    return p, seq.unpack8(p, dtype=torch.float32)


@gpu
@pytest.mark.parametrize("lay,dtype,D,W,silu,bias,pad", CONV)
@pytest.mark.parametrize("packed,with_state", [(False, True), (True, True), (False, False)])
def test_conv_gradient(lay, dtype, D, W, silu, bias, pad, packed, with_state):
    if packed and dtype == "f64":
        pytest.skip("checkpoints hold float32, bfloat16 and float16")
    c = conv_case(lay, dtype, D, W, silu, bias, pad, seed=1)
    x, values = held(c["x"], packed)
    st, ds = (c["state"], c["dstate"]) if with_state else (None, None)
    g = seq.causal_conv_grad(c["dy"], x, c["w"], c["b"], silu=silu, state=st, dstate=ds, **c["kw"])
    p = plain_conv(torch.nan_to_num(rows_of(values)), cpu64(c["w"]), cpu64(c["b"]), silu, c["spans"], cpu64(st), torch.nan_to_num(rows_of(c["dy"])), cpu64(ds))
    check(g.x.reshape(-1, D), *p["dx"], 4 * W + 20, "dx")
    n = sum(hi - lo for lo, hi in c["spans"])
    k = 3 * W + 20 + min(n, 64)         # a strip's rows are summed in the compute type, the strips in double
    check(g.weight, *p["dw"], k, "dweight")
    if bias:
        check(g.bias, *p["db"], k, "dbias")
    else:
        assert g.bias is None
    if with_state:
        check(g.state, *p["dstate"], 4 * W + 20, "dstate")
    else:
        assert g.state is None
    again = seq.causal_conv_grad(c["dy"], x, c["w"], c["b"], silu=silu, state=st, dstate=ds, **c["kw"])
    assert all(a is None or torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(g, again))


@gpu
def test_conv_gradient_against_differences():
    c = conv_case("packed", "f64", 6, 4, True, True, 0, seed=2)
    f = lambda k: sum(float((a * b).sum()) for a, b in zip(seq.causal_conv(k["x"], k["w"], k["b"], silu=True, state=k["state"], return_state=True, **c["kw"]),  # noqa: E731
                                                           (c["dy"], c["dstate"])))
    g = seq.causal_conv_grad(c["dy"], c["x"], c["w"], c["b"], silu=True, state=c["state"], dstate=c["dstate"], **c["kw"])
    difference_test(f, {k: c[k] for k in ("x", "w", "b", "state")}, dict(x=g.x, w=g.weight, b=g.bias, state=g.state))


def difference_test(f, at, grads, n=4):
    """Central differences in random directions: error h^2 f'''/6 + eps |f| / h, with h = 1e-4 about 1e-8 of the terms' size."""
    g = torch.Generator().manual_seed(5)
    for name in at:
        for _ in range(n):
            d = torch.randn(at[name].shape, generator=g, dtype=torch.float64).to(at[name].device)
            h = 1e-4
            up, down = f({**at, name: at[name] + h * d}), f({**at, name: at[name] - h * d})
            want = float((grads[name].double() * d).sum())
            size = float((grads[name].double() * d).abs().sum()) + 1
            assert abs((up - down) / (2 * h) - want) <= 2e-6 * size, (name, (up - down) / (2 * h), want)


STEP = [("f32", 5, 9, 7, 4), ("bf16", 1, 1, 256, 4), ("bf16", 6, 8, 130, 4), ("f16", 4, 6, 33, 2), ("f64", 3, 3, 12, 5), ("f32", 7, 20, 1030, 1)]


@gpu
@pytest.mark.parametrize("dtype,n,slots,D,W", STEP)
def test_conv_step(dtype, n, slots, D, W):
    g = torch.Generator().manual_seed(n * D)
    dt = DT[dtype]
    w, b, cache = rnd(g, D, W, dtype=param_of(dt), scale=0.5), rnd(g, D, dtype=param_of(dt)), rnd(g, slots, W - 1, D, dtype=dt)
    at = torch.randperm(slots, generator=g)[:n].to(torch.int32)
    if n > 3:
        at[1], at[3] = at[0], -1                # two rows of one sequence, a row that is padding
    x = rnd(g, n, D, dtype=dt)
    mine = cache.clone()
    y = seq.causal_conv_step(x, w, b, mine, at.to(DEV), silu=True)
    ref, st = torch.zeros(n, D, dtype=torch.float64), cpu64(cache).clone()
    scale = torch.zeros(n, D, dtype=torch.float64)
    for r, k in enumerate(at.tolist()):
        if k < 0:
            continue
        p = plain_conv(cpu64(x)[r:r + 1], cpu64(w), cpu64(b), True, [(0, 1)], st[k:k + 1])
        ref[r], scale[r], st[k] = p["y"][0][0], p["y"][1][0], p["state"][0][0]
    check(y, ref, scale, 3 * W + 10, "y")
    assert torch.equal(mine.cpu().double(), st)
    if n <= slots:          # without slots: row r continues state r
        mine = cache.clone()
        y = seq.causal_conv_step(x, w, b, mine, silu=True)
        z = [seq.causal_conv(x[r:r + 1, None], w, b, silu=True, state=cache[r:r + 1], return_state=True) for r in range(n)]
        assert torch.equal(y, torch.cat([a[0][:, 0] for a in z])) and torch.equal(mine[:n], torch.cat([a[1] for a in z])) and torch.equal(mine[n:], cache[n:])


# ---------------------------------------------------------------- scan
#: layout, type, D, N, G, gate, softplus, skip, bias, extra elements between rows
SCAN = [("one_row", "f32", 3, 1, 1, False, True, True, True, 0), ("dense", "bf16", 96, 16, 1, True, True, True, True, 0), ("dense", "f32", 70, 16, 2, False, False, False, False, 0),
        ("padded", "f16", 65, 8, 1, True, True, True, True, 0), ("packed", "f32", 130, 16, 1, True, True, True, True, 0), ("packed", "bf16", 48, 11, 4, True, True, False, True, 3),
        ("gap", "f32", 40, 5, 2, True, False, True, True, 2), ("packed", "f64", 10, 9, 1, True, True, True, True, 0), ("packed", "f32", 24, 37, 3, True, True, True, False, 0),
        ("padded", "f64", 6, 3, 2, False, True, True, True, 1), ("dense", "f16", 12, 64, 1, True, True, True, True, 0)]


def scan_case(lay, dtype, D, N, G, gate, softplus, skip, bias, pad, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * D + N)
    lead, kw, sp, outside = layout(lay)
    dt, pt = DT[dtype], param_of(DT[dtype])

    def act(scale=1.0, *tail):
        x = poison(rnd(g, *lead, *(tail or (D,)), dtype=dt, scale=scale), outside, len(lead))
        return strided(x, pad) if pad else x

    c = dict(u=act(), z=act() if gate else None, dy=act(), A=-torch.exp(rnd(g, D, N, dtype=pt, scale=0.7)),
             B=act(1.0, G, N) if G > 1 else act(1.0, N), C=act(1.0, G, N) if G > 1 else act(1.0, N), D=rnd(g, D, dtype=pt) if skip else None,
             state=rnd(g, len(sp), D, N, dtype=pt), dstate=rnd(g, len(sp), D, N, dtype=pt), kw=kw, spans=sp, outside=outside)
    c["dt"] = act(0.8) if softplus else act(0.2).abs()
    c["bias"] = rnd(g, D, dtype=pt, scale=0.5) - 1.0 if bias and softplus else (rnd(g, D, dtype=pt).abs() * 0.1 if bias else None)
    return c


def scan_ref(c, D, G, N, softplus, state, u=None, z=None, **kw):
    f = lambda x: torch.nan_to_num(rows_of(x))  # noqa: E731
    m = lambda x: torch.nan_to_num(cpu64(x)).reshape(-1, G, N)  # noqa: E731
    zz = c["z"] if z is None else z
    return plain_scan(f(c["u"] if u is None else u), f(c["dt"]), cpu64(c["A"]), m(c["B"]), m(c["C"]), cpu64(c["D"]), None if zz is None else f(zz), cpu64(c["bias"]), softplus,
                      c["spans"], cpu64(state), **{k: f(v) if k == "dy" else cpu64(v) for k, v in kw.items()})


def longest(c):
    return max(hi - lo for lo, hi in c["spans"])


@gpu
@pytest.mark.parametrize("lay,dtype,D,N,G,gate,softplus,skip,bias,pad", SCAN)
@pytest.mark.parametrize("with_state", [True, False])
def test_scan_forward(lay, dtype, D, N, G, gate, softplus, skip, bias, pad, with_state):
    c = scan_case(lay, dtype, D, N, G, gate, softplus, skip, bias, pad)
    st = c["state"] if with_state else None
    kw = dict(D=c["D"], z=c["z"], dt_bias=c["bias"], softplus=softplus, state=st, **c["kw"])
    y, end = seq.selective_scan(c["u"], c["dt"], c["A"], c["B"], c["C"], return_state=True, **kw)
    p = scan_ref(c, D, G, N, softplus, st)
    # a row's input meets: step length (about 12 roundings), decay and product of each later row (the scale carries the decays, so the rows
    # that still weigh are few; 6 a row for the rows of a chunk), the sum over N states, the gate
    k = 30 + N + 4 * min(longest(c), 16)
    check(y.reshape(-1, D), *p["y"], k, "y")
    check(end, *p["state"], k, "state")
    assert bool((y.reshape(-1, D).cpu()[c["outside"]] == 0).all())
    own = torch.full_like(y, 3.0)
    assert seq.selective_scan(c["u"], c["dt"], c["A"], c["B"], c["C"], out=own, **kw) is own
    assert bool((own.reshape(-1, D).cpu()[c["outside"]] == 3).all())
    assert torch.equal(own.reshape(-1, D).cpu()[~c["outside"]], y.reshape(-1, D).cpu()[~c["outside"]])


@gpu
@pytest.mark.parametrize("lay,dtype,D,N,G,gate,softplus,skip,bias,pad", SCAN)
@pytest.mark.parametrize("packed,with_state", [(False, True), (True, True), (False, False)])
def test_scan_gradient(lay, dtype, D, N, G, gate, softplus, skip, bias, pad, packed, with_state):
    if packed and dtype == "f64":
        pytest.skip("checkpoints hold float32, bfloat16 and float16")
    c = scan_case(lay, dtype, D, N, G, gate, softplus, skip, bias, pad, seed=1)
    st, ds = (c["state"], c["dstate"]) if with_state else (None, None)
    u, uv = held(c["u"], packed)
    z, zv = held(c["z"], packed) if gate else (None, None)
    call = lambda: seq.selective_scan_grad(c["dy"], u, c["dt"], c["A"], c["B"], c["C"], D=c["D"], z=z, dt_bias=c["bias"], softplus=softplus, state=st, dstate=ds, **c["kw"])  # noqa: E731
    g = call()
    p = scan_ref(c, D, G, N, softplus, st, u=uv, z=zv, dy=c["dy"], dstate=ds)["grad"]
    n = longest(c)
    k = 60 + N + 8 * min(n, 16)
    for name in ("u", "dt"):
        check(getattr(g, name).reshape(-1, D), *p[name], k, name)
        assert bool((getattr(g, name).reshape(-1, D).cpu()[c["outside"]] == 0).all())
    if gate:
        check(g.z.reshape(-1, D), *p["z"], k, "z")
    else:
        assert g.z is None
    for name in ("B", "C"):
        check(getattr(g, name).reshape(-1, G, N), *p[name], k + D // G, name)
        assert getattr(g, name).shape == c[name].shape
        assert bool((getattr(g, name).reshape(-1, G * N).cpu()[c["outside"]] == 0).all())
    check(g.A, *p["A"], k + 32, "A")
    for name, there in (("D", skip), ("dt_bias", bias)):
        if there:
            check(getattr(g, name), *p[name], k + 32, name)
        else:
            assert getattr(g, name) is None
    if with_state:
        check(g.state, *p["state"], k, "state")
    else:
        assert g.state is None
    assert all(a is None or torch.equal(a, b) for a, b in zip(g, call()))


@gpu
def test_scan_gradient_against_differences():
    D, N, G = 4, 3, 2
    c = scan_case("packed", "f64", D, N, G, True, True, True, True, 0, seed=3)
    names = ("u", "dt", "A", "B", "C", "D", "z", "bias", "state")

    def f(k):
        y, end = seq.selective_scan(k["u"], k["dt"], k["A"], k["B"], k["C"], D=k["D"], z=k["z"], dt_bias=k["bias"], state=k["state"], return_state=True, **c["kw"])
        return float((y * c["dy"]).sum()) + float((end * c["dstate"]).sum())

    g = seq.selective_scan_grad(c["dy"], c["u"], c["dt"], c["A"], c["B"], c["C"], D=c["D"], z=c["z"], dt_bias=c["bias"], state=c["state"], dstate=c["dstate"], **c["kw"])
    difference_test(f, {k: c[k] for k in names}, {**{k: getattr(g, k) for k in names if k != "bias"}, "bias": g.dt_bias})


@gpu
@pytest.mark.parametrize("rows,D,N", [(1000, 64, 16), (517, 200, 8)])
def test_long_scan_is_cut_into_chunks_like_one(rows, D, N):
    """A sequence much longer than a chunk, alone, against the same sequence in pieces that carry their state on."""
    g = torch.Generator().manual_seed(rows)
    u, dt, z = rnd(g, 1, rows, D), rnd(g, 1, rows, D, scale=0.5) - 3, rnd(g, 1, rows, D)
    A, B, C, skip = -torch.exp(rnd(g, D, N)), rnd(g, 1, rows, N), rnd(g, 1, rows, N), rnd(g, D)
    y, end = seq.selective_scan(u, dt, A, B, C, D=skip, z=z, return_state=True)
    st, parts = None, []
    for lo in range(0, rows, 100):
        s = slice(lo, lo + 100)
        yy, st = seq.selective_scan(u[:, s], dt[:, s], A, B[:, s], C[:, s], D=skip, z=z[:, s], state=st, return_state=True)
        parts.append(yy)
    p = plain_scan(*(rows_of(x) for x in (u, dt)), cpu64(A), cpu64(B).view(rows, 1, N), cpu64(C).view(rows, 1, N), cpu64(skip), rows_of(z), None, True, [(0, rows)], None)
    for got, e in ((y, end), (torch.cat(parts, 1), st)):
        check(got.reshape(-1, D), *p["y"], 30 + N + 64, "y")
        check(e, *p["state"], 30 + N + 64, "state")


@gpu
@pytest.mark.parametrize("dtype,n,slots,D,N,G,gate", [("f32", 5, 9, 7, 16, 1, True), ("bf16", 1, 1, 256, 16, 1, True), ("bf16", 6, 8, 130, 16, 2, True), ("f16", 4, 6, 33, 5, 3, False),
                                                       ("f64", 5, 5, 12, 9, 1, True), ("f32", 7, 20, 70, 64, 1, True), ("f32", 2, 2, 3, 1, 1, False), ("f32", 4, 4, 20, 200, 2, True)])
def test_scan_step(dtype, n, slots, D, N, G, gate):
    g = torch.Generator().manual_seed(n * D + N)
    dt, pt = DT[dtype], param_of(DT[dtype])
    u, d, z = rnd(g, n, D, dtype=dt), rnd(g, n, D, dtype=dt, scale=0.5), rnd(g, n, D, dtype=dt) if gate else None
    A, B, C = -torch.exp(rnd(g, D, N, dtype=pt)), rnd(g, n, G, N, dtype=dt), rnd(g, n, G, N, dtype=dt)
    skip, bias, cache = rnd(g, D, dtype=pt), rnd(g, D, dtype=pt), rnd(g, slots, D, N, dtype=pt)
    at = torch.randperm(slots, generator=g)[:n].to(torch.int32)
    if n > 3:
        at[1], at[3] = at[0], slots
    mine = cache.clone()
    y = seq.selective_scan_step(u, d, A, B, C, mine, at.to(DEV), D=skip, z=z, dt_bias=bias)
    st, ref, scale = cpu64(cache).clone(), torch.zeros(n, D, dtype=torch.float64), torch.zeros(n, D, dtype=torch.float64)
    hs = st.abs()
    for r, k in enumerate(at.tolist()):
        if k >= slots:
            continue
        one = lambda x: None if x is None else cpu64(x)[r:r + 1]  # noqa: E731
        # (a second row of one sequence: its state's error is eps of what the first row's terms added up to, whatever of them cancelled)
        p = plain_scan(one(u), one(d), cpu64(A), one(B), one(C), cpu64(skip), one(z), cpu64(bias), True, [(0, 1)], st[k:k + 1], mag=hs[k:k + 1])
        ref[r], scale[r], st[k], hs[k] = p["y"][0][0], p["y"][1][0], p["state"][0][0], p["state"][1][0]
    check(y, ref, scale, 40 + N, "y")
    check(mine, st, hs, 40, "state")
    left = torch.ones(slots, dtype=torch.bool)
    left[at[at < slots].long()] = False
    assert torch.equal(mine.cpu()[left], cache.cpu()[left])


# ---------------------------------------------------------------- what happens at the edges of numbers
@gpu
def test_step_length_keeps_its_relative_accuracy():
    """softplus from -80 (1e-35) to 80: the state after one row from 0 with B = u = 1 is the step length itself."""
    x = torch.cat([torch.linspace(-80, 80, 4001), torch.tensor([0.0, -1e-7, 1e-7, -19.99, 20.01])]).to(DEV)
    D = x.numel()
    one = torch.ones(1, 1, 1, device=DEV)
    _, end = seq.selective_scan(torch.ones(1, 1, D, device=DEV), x.view(1, 1, D), -torch.ones(D, 1, device=DEV), one, one, return_state=True)
    want = torch.nn.functional.softplus(x.double().cpu(), threshold=1e9)
    want = torch.where(x.cpu() < -30, torch.exp(x.double().cpu()), want)
    # the exponent x log2(e) is rounded to 24 bits: |x| eps / 2 of the value each for the product and the constant; then about 8 roundings
    limit = (8 + x.double().cpu().abs()) * 2.0 ** -23
    assert bool(((end.view(-1).cpu().double() / want - 1).abs() <= limit).all())


@gpu
def test_a_step_has_an_exact_decay_and_an_input_of_first_order():
    """h = exp(delta A) h + delta B u, not the integral over a held input (exp(delta A) - 1) / A B u; the two agree to first order in delta A."""
    A = -torch.tensor([[16.0], [1.6], [0.01]], device=DEV)
    one, state = torch.ones(1, 1, 1, device=DEV), torch.full((1, 3, 1), 0.5, device=DEV)
    for delta in (0.1, 1e-3):
        dt = torch.full((1, 1, 3), delta, device=DEV)
        _, end = seq.selective_scan(torch.ones(1, 1, 3, device=DEV), dt, A, one, one, softplus=False, state=state, return_state=True)
        d, a = float(dt[0, 0, 0].double()), cpu64(A)
        want = torch.exp(d * a) * 0.5 + d
        # decay: the exponent's rounding and the exponential's; product and sum
        assert bool(((cpu64(end)[0] - want).abs() <= 8 * 2.0 ** -24 * (1 + (d * a).abs()) * want).all())
        held = torch.exp(d * a) * 0.5 + torch.expm1(d * a) / a
        assert bool(((want - held).abs() <= d * (d * a).abs()).all())


@gpu
def test_infinities_and_nan_stay_in_their_channel_and_after_their_row():
    g = torch.Generator().manual_seed(0)
    u, dt, z = rnd(g, 2, 50, 80), rnd(g, 2, 50, 80), rnd(g, 2, 50, 80)
    A, B, C = -torch.exp(rnd(g, 80, 16)), rnd(g, 2, 50, 16), rnd(g, 2, 50, 16)
    y = seq.selective_scan(u, dt, A, B, C, z=z)
    u[0, 20, 3], dt[1, 10, 70], z[0, 5, 9] = float("inf"), float("nan"), float("nan")
    w = seq.selective_scan(u, dt, A, B, C, z=z)
    touched = torch.zeros(2, 50, 80, dtype=torch.bool, device=DEV)
    touched[0, 20:, 3], touched[1, 10:, 70], touched[0, 5, 9] = True, True, True
    assert torch.equal(y[~touched], w[~touched]) and not bool(torch.isfinite(w[touched]).any())
    c = seq.causal_conv(u, rnd(g, 80, 4))
    assert int((~torch.isfinite(c)).sum()) == 4 and not bool(torch.isfinite(c[0, 20:24, 3]).any())


def not_finite(x):
    return ~torch.isfinite(x.float()).cpu()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f64"])
@pytest.mark.parametrize("D", [5, 40])
@pytest.mark.parametrize("W", range(1, 9))
def test_convolution_takes_nothing_from_rows_its_taps_do_not_reach(W, D, dtype):
    """An infinity and a NaN reach W rows of their own channel, forward, back and in single rows that share a state; all else keeps its bits."""
    g = torch.Generator().manual_seed(W)
    T, dt = 70, DT[dtype]
    x, dy, w, b = rnd(g, 1, T, D, dtype=dt), rnd(g, 1, T, D, dtype=dt), rnd(g, D, W, dtype=param_of(dt)).abs() + 0.1, rnd(g, D, dtype=param_of(dt))
    bx, bdy = x.clone(), dy.clone()
    hit = torch.zeros(1, T, D, dtype=torch.bool)        # rows that see the bad input; back: rows seen by it
    back = hit.clone()
    for t, d, v in ((10, 1, math.inf), (33, D - 1, math.nan), (T - 1, 0, -math.inf)):
        bx[0, t, d] = bdy[0, t, d] = v
        hit[0, t:t + W, d] = True
        back[0, max(t - W + 1, 0):t + 1, d] = True
    y, z = seq.causal_conv(x, w, b), seq.causal_conv(bx, w, b)
    assert torch.equal(not_finite(z), hit) and torch.equal(z.cpu()[~hit], y.cpu()[~hit])
    y, z = seq.causal_conv_grad(dy, x, w, b).x, seq.causal_conv_grad(bdy, x, w, b).x
    assert torch.equal(not_finite(z), back) and torch.equal(z.cpu()[~back], y.cpu()[~back])
    at = torch.zeros(T, dtype=torch.int32, device=DEV)
    states = [torch.zeros(1, W - 1, D, dtype=dt, device=DEV) for _ in range(2)]
    y, z = (seq.causal_conv_step(v[0], w, b, s, at) for v, s in zip((x, bx), states))
    assert torch.equal(not_finite(z), hit[0]) and torch.equal(z.cpu()[~hit[0]], y.cpu()[~hit[0]])
    if dtype != "f64":          # a block that a checkpoint gives back as NaN, met by the gate's derivative
        bx = x.clone()
        bx[0, 33, 2] = math.inf
        y, z = (seq.causal_conv_grad(dy, seq.pack8(v), w, b, silu=True).x for v in (x, bx))
        near = torch.zeros(1, T, D, dtype=torch.bool)
        near[0, 33 - W + 1:33 + W, :32] = True
        assert torch.equal(not_finite(z), near) and torch.equal(z.cpu()[~near], y.cpu()[~near])


@gpu
@pytest.mark.parametrize("D,dtype", [(5, "f32"), (40, "bf16"), (40, "f64")])
@pytest.mark.parametrize("W", range(1, 9))
def test_weight_gradient_takes_each_row_with_its_own_taps_only(W, D, dtype):
    """dweight[d, j] = sum_t dp[t] x[t - W + 1 + j]: the last row meets the last tap alone, the one before it the last two, and so on."""
    g = torch.Generator().manual_seed(W)
    lens, dt = [70, 1, 47], DT[dtype]
    at = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)
    x, dy, w = rnd(g, sum(lens), D, dtype=dt), rnd(g, sum(lens), D, dtype=dt).abs() + 0.1, rnd(g, D, W, dtype=param_of(dt))
    clean = seq.causal_conv_grad(dy, x, w, torch.zeros(D, device=DEV), seq_start=at)
    for s, n in enumerate(lens):
        for back in range(min(n, W + 1)):
            row, bad = int(at[s + 1]) - 1 - back, x.clone()
            bad[row, D - 1] = math.inf
            got = seq.causal_conv_grad(dy, bad, w, torch.zeros(D, device=DEV), seq_start=at)
            want = torch.zeros(D, W, dtype=torch.bool)
            want[D - 1, max(W - 1 - back, 0):] = True
            assert torch.equal(got.weight.cpu() == math.inf, want) and torch.equal(got.weight.cpu()[~want], clean.weight.cpu()[~want]), (row, back)
            assert torch.equal(got.bias, clean.bias) and torch.equal(got.x, clean.x)
    # rows at the ends of the strips that a long sequence is cut into
    for row in (8, 15, 23, 31, 47, 63):
        bad = x.clone()
        bad[row, 1] = math.inf
        got = seq.causal_conv_grad(dy, bad, w, seq_start=at)
        assert torch.equal(got.weight[1].cpu() == math.inf, torch.arange(W) >= W - 1 - (lens[0] - 1 - row)) and torch.equal(got.weight[2:], clean.weight[2:])


def alike(got, want, scale, k, what):
    """Finite where the 64-bit form is, and there like it."""
    g, w = got.detach().cpu(), want.cpu()
    assert torch.equal(torch.isfinite(g), torch.isfinite(w)), (what, torch.isfinite(g) ^ torch.isfinite(w))
    ok = torch.isfinite(w)
    check(g[ok], w[ok], torch.nan_to_num(scale.cpu()[ok], nan=math.inf, posinf=math.inf), k, what)


def scan_with(T, D, N, bad, dtype=torch.float32, skip=True, seed=0):
    """Positive inputs (no sum of two infinities is NaN), `bad` = {(array, row, channel): value} put into them."""
    g = torch.Generator().manual_seed(seed + N)
    c = {k: rnd(g, T, n, dtype=dtype).abs() + 0.1 for k, n in (("u", D), ("dt", D), ("z", D), ("dy", D), ("B", N), ("C", N))}
    c.update(A=-(rnd(g, D, N).abs() + 0.1), D=rnd(g, D).abs() + 0.1 if skip else None, bias=None, state=rnd(g, 1, D, N).abs(), dstate=rnd(g, 1, D, N).abs(), spans=[(0, T)],
             kw=dict(seq_start=torch.tensor([0, T], dtype=torch.int32, device=DEV)))
    for (name, row, col), v in bad.items():
        c[name][row, col] = v
    return c


def scan_all(c):
    """{name: (result, how it is called in the 64-bit form)} of the forward call and the gradient."""
    kw = dict(D=c["D"], z=c["z"], state=c["state"], softplus=False, **c["kw"])
    y, end = seq.selective_scan(c["u"], c["dt"], c["A"], c["B"], c["C"], return_state=True, **kw)
    g = seq.selective_scan_grad(c["dy"], c["u"], c["dt"], c["A"], c["B"], c["C"], dstate=c["dstate"], **kw)
    return {"y": y, "end": end, **{k: v for k, v in g._asdict().items() if v is not None}}


def scan_all_plain(c):
    N = c["A"].shape[1]
    m = lambda x: cpu64(x).view(-1, 1, N)  # noqa: E731
    p = plain_scan(cpu64(c["u"]), cpu64(c["dt"]), cpu64(c["A"]), m(c["B"]), m(c["C"]), cpu64(c["D"]), cpu64(c["z"]), None, False, c["spans"], cpu64(c["state"]), dy=cpu64(c["dy"]),
                   dstate=cpu64(c["dstate"]))
    g = {k: tuple(v) for k, v in p["grad"].items()}
    g["B"], g["C"] = (tuple(v.view(-1, N) for v in g[k]) for k in ("B", "C"))
    return {"y": p["y"], "end": p["state"], **g}


@gpu
@pytest.mark.parametrize("T", [50, 150])
@pytest.mark.parametrize("N", [1, 5, 8, 11, 16, 20, 32, 37])
@pytest.mark.parametrize("name,row", [("u", 5), ("u", 44), ("dt", 23), ("dy", 30), ("dt", 49)])
def test_states_that_are_not_there_take_no_part(name, row, N, T):
    """Any number of states, an infinity in the data: infinite where the formula is, finite where it is finite."""
    c = scan_with(T, 7, N, {(name, row, 3): math.inf})
    got, want = scan_all(c), scan_all_plain(c)
    for k, v in got.items():
        alike(v, *want[k], 60 + N + 8 * 16, k)
    # the single step: the row with the infinity, its state and the row behind it
    st = c["state"].clone()
    at = torch.zeros(2, dtype=torch.int32, device=DEV)
    s = lambda k: c[k][row - 1:row + 1]  # noqa: E731
    y = seq.selective_scan_step(s("u"), s("dt"), c["A"], s("B"), s("C"), st, at, D=c["D"], z=s("z"), softplus=False)
    m = lambda k: cpu64(s(k)).view(2, 1, N)  # noqa: E731
    p = plain_scan(cpu64(s("u")), cpu64(s("dt")), cpu64(c["A"]), m("B"), m("C"), cpu64(c["D"]), cpu64(s("z")), None, False, [(0, 2)], cpu64(c["state"]))
    alike(y, *p["y"], 60 + N, "step")
    alike(st, *p["state"], 60, "state")


@gpu
@pytest.mark.parametrize("T", [50, 150])
@pytest.mark.parametrize("N", [8, 16, 32])
@pytest.mark.parametrize("name,row", [("u", 5), ("u", 44), ("dy", 30)])
def test_absent_skip_is_not_a_skip_of_zero(name, row, N, T):
    """Without D there is no D u: an infinite u comes through the states as an infinity, not as NaN, and so does an infinite gradient back to u."""
    c = scan_with(T, 7, N, {(name, row, 3): math.inf}, skip=False)
    got, want = scan_all(c), scan_all_plain(c)
    for k in ("y", "u", "z"):
        v, (w, s) = got[k].cpu(), want[k]
        reach = {"u": {"y": slice(row, T), "u": None, "z": slice(row, T)}, "dy": {"y": None, "u": slice(0, row + 1), "z": slice(row, row + 1)}}[name][k]
        bad = torch.zeros(T, 7, dtype=torch.bool)
        if reach is not None:
            bad[reach, 3] = True
        assert torch.equal(v == math.inf, bad) and not bool(torch.isnan(v).any()), k
        check(v[~bad], w[~bad], torch.nan_to_num(s[~bad], nan=math.inf, posinf=math.inf), 60 + N + 8 * 16, k)
    st = c["state"].clone()
    s = lambda k: c[k][row:row + 1]  # noqa: E731
    y = seq.selective_scan_step(s("u"), s("dt"), c["A"], s("B"), s("C"), st, z=s("z"), softplus=False).cpu()[0]
    assert bool((y == math.inf)[3]) == (name == "u") and int(torch.isfinite(y).sum()) == (6 if name == "u" else 7)


@gpu
@pytest.mark.parametrize("T", [40, 70, 200])
@pytest.mark.parametrize("N", [3, 16, 32])
@pytest.mark.parametrize("sign", ["rate", "step"])
@pytest.mark.parametrize("dtype", ["f32", "f64"])
def test_modes_that_grow_stay_in_range_where_the_formula_does(sign, N, T, dtype):
    """A positive rate, or a negative step length: exp(A sum delta) over a chunk is out of range (e^120 in 20 rows; double: e^1500), but nothing has come in yet,
    or nothing is asked of it any more: the states and gradients are 0 there, not 0 times infinity."""
    c = scan_with(T, 7, N, {}, dtype=DT[dtype])
    for k in ("A", "D", "state", "dstate"):
        c[k] = c[k].to(param_of(DT[dtype]))
    c["A"][:, :] = c["A"] - 2 if sign == "step" else -c["A"] + 2
    c["dt"] = c["dt"] * 0 + (3.0 if dtype == "f32" else 40.0) * (-1 if sign == "step" else 1)
    c["u"][:T - 1], c["dy"][1:], c["state"][:], c["dstate"][:] = 0, 0, 0, 0
    got, want = scan_all(c), scan_all_plain(c)
    for k, v in got.items():
        assert bool(torch.isfinite(want[k][0]).all()) and float(want[k][0].abs().max()) < (1e30 if dtype == "f32" else 1e300), k
        alike(v, *want[k], 60 + N + 8 * 16, k)
    # a state of 1e-30 that grows by e^96 in 16 rows comes out at 1e11
    if dtype == "f32" and T > 64:
        c["A"][:] = 2.0 if sign == "rate" else -2.0
        c["dt"][:16], c["dt"][16:] = (3.0, 0.0) if sign == "rate" else (-3.0, 0.0)
        c["u"][:], c["state"][:] = 0, 1e-30
        y, end = seq.selective_scan(c["u"], c["dt"], c["A"], c["B"], c["C"], state=c["state"], softplus=False, return_state=True, **c["kw"])
        want = math.exp(96 + math.log(float(c["state"][0, 0, 0])))
        # 16 rows (or a chunk's one product) with an exponent's relative error of 2^-24 times its size each: 96 + 16 times 3 eps
        assert bool(((end.double() / want - 1).abs() <= (96 + 48) * 2.0 ** -23).all())


@gpu
@pytest.mark.parametrize("T", [50, 200])
@pytest.mark.parametrize("N", [16, 20])
@pytest.mark.parametrize("what", ["growth", "nan"])
def test_a_channel_out_of_range_leaves_the_others_their_bits(what, N, T):
    c = scan_with(T, 70, N, {})
    clean = scan_all(c)
    if what == "growth":
        c["A"][3, :] = 2.0
        c["dt"][:, 3] = 3.0
    else:
        c["dt"][T // 2, 3] = math.nan
    got = scan_all(c)
    others = torch.arange(70, device=DEV) != 3
    for k, v in got.items():
        if k in ("B", "C"):
            continue            # (sums over the channels)
        at = {"A": 0, "D": 0, "end": 1, "state": 1}.get(k, 1)
        assert torch.equal(v.movedim(at, 0)[others], clean[k].movedim(at, 0)[others]), k


@gpu
@pytest.mark.parametrize("T", [1, 11, 64, 70, 151])
@pytest.mark.parametrize("N", [5, 16, 32])
@pytest.mark.parametrize("dtype", ["f32", "f64"])
def test_rows_behind_the_last_one_change_nothing(N, T, dtype):
    """Batches of rows that a sequence does not fill: an infinite rate (a decay of 0), an infinity in the last row's maps."""
    def run(c):
        y, end = seq.selective_scan(c["u"], c["dt"], c["A"], c["B"], c["C"], D=c["D"], z=c["z"], state=c["state"], softplus=False, return_state=True, **c["kw"])
        p = scan_all_plain(c)
        alike(y, *p["y"], 60 + N + 64, "y")
        alike(end, *p["end"], 60 + N + 64, "end")
        assert torch.equal(end.cpu() == math.inf, p["end"][0] == math.inf) and torch.equal(torch.isnan(y.cpu()), torch.isnan(p["y"][0]))

    def case():
        c = scan_with(T, 7, N, {}, dtype=DT[dtype])
        return {k: v.to(param_of(DT[dtype])) if k in ("A", "D", "state", "dstate") else v for k, v in c.items()}

    c = case()
    c["A"][2, :], c["A"][4, 1] = -math.inf, -math.inf
    run(c)
    c = case()
    c["B"][T - 1, 0] = math.inf
    run(c)


@gpu
@pytest.mark.parametrize("starts", [[0, 90, 40, 60], [-5, 20, 300], [50, 10], [0]])
def test_offsets_that_make_no_sense_stay_inside_the_arrays(starts):
    g = torch.Generator().manual_seed(1)
    at = torch.tensor(starts, dtype=torch.int32, device=DEV)
    u, dt, dy, B, C = (rnd(g, 60, n) for n in (20, 20, 20, 16, 16))
    A = -torch.exp(rnd(g, 20, 16))
    assert seq.causal_conv(u, rnd(g, 20, 4), seq_start=at, return_state=True)[1].shape == (len(starts) - 1, 3, 20)
    seq.causal_conv_grad(dy, u, rnd(g, 20, 4), seq_start=at)
    assert seq.selective_scan(u, dt, A, B, C, seq_start=at, return_state=True)[1].shape == (len(starts) - 1, 20, 16)
    seq.selective_scan_grad(dy, u, dt, A, B, C, seq_start=at)


@gpu
def test_offsets_not_in_use_repeat_the_last_one():
    g = torch.Generator().manual_seed(6)
    x, dt, dy, m = (rnd(g, 90, n) for n in (20, 20, 20, 16))
    A, w = -torch.exp(rnd(g, 20, 16)), rnd(g, 20, 4)
    few, more = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([0, 25, 70], [0, 25, 70] + [70] * 70))
    assert torch.equal(seq.causal_conv(x, w, seq_start=few), seq.causal_conv(x, w, seq_start=more))
    ga, gb = (seq.causal_conv_grad(dy, x, w, seq_start=at) for at in (few, more))
    assert torch.equal(ga.x, gb.x) and torch.allclose(ga.weight, gb.weight, rtol=1e-5, atol=1e-4)
    (ya, ea), (yb, eb) = (seq.selective_scan(x, dt, A, m, m, seq_start=at, return_state=True) for at in (few, more))
    # (the number of sequences is part of the rule how time is cut: another order of the same sums)
    assert bool(((ya - yb).abs() <= 1e-5 * (1 + ya.abs())).all()) and torch.allclose(ea, eb[:2], rtol=1e-5, atol=1e-5) and not bool(eb[2:].any())


# ---------------------------------------------------------------- checkpoints
@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,pad", [((3, 64), 0), ((2, 5, 33), 0), ((7, 1), 0), ((4, 100), 3), ((1, 31), 0), ((0, 40), 0), ((9, 48), 16), ((5, 160), 8)])
def test_checkpoint_codes_and_values(dtype, shape, pad):
    g = torch.Generator().manual_seed(shape[-1])
    x = rnd(g, *shape, dtype=torch.float32) * torch.exp(3 * rnd(g, *shape[:-1], 1))
    x = x.to(DT[dtype])
    if x.numel() > 50:
        x.view(-1)[:5] = torch.tensor([0.0, 127.5, -127.5, 1.0, 255.0], dtype=torch.float32).to(DT[dtype]).to(DEV)
    p = seq.pack8(strided(x, pad) if pad else x)
    codes, scales = plain_codes(x.reshape(math.prod(shape[:-1]), shape[-1]).cpu().float())
    assert torch.equal(p.codes.cpu().view(codes.shape), codes) and torch.equal(p.scales.cpu().view(scales.shape), scales)
    back = seq.unpack8(p)
    want = (codes.double() * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)[:, :shape[-1]])
    assert back.dtype == x.dtype and torch.equal(back.cpu().double().view(want.shape), want.to(DT[dtype]).double())
    wide = seq.unpack8(p, dtype=torch.float32)
    assert torch.equal(wide.cpu().double().view(want.shape), want)
    # within half a code, and a code is at most max|x| / 64 of its block
    if x.numel():
        big = torch.nn.functional.pad(x.cpu().double().view(-1, shape[-1]).abs(), (0, -shape[-1] % 32)).view(len(codes), -1, 32).amax(-1)
        assert bool(((wide.cpu().double().view(-1, shape[-1]) - x.cpu().double().view(-1, shape[-1])).abs() <= big.repeat_interleave(32, 1)[:, :shape[-1]] / 128 + 2.0 ** -128).all())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_checkpoint_error_reaches_its_bound(dtype):
    """max|x| / 127.5 is the bound: reached where the largest value would round to 128 codes and the code is doubled (64 of them, half a code off is max / 127.5); 2^-128
    where the smallest scale is in use; a code where the type's last binade leaves no room for the doubled one."""
    dt = DT[dtype]
    small = -10 if dtype == "f16" else -120
    x = torch.zeros(4, 32, dtype=torch.float64)
    for r, e in enumerate((0, 5, small)):
        x[r, 0] = 255 / 128
        x[r, 1:] = (2 * torch.arange(31) + 1) / 64           # half a code of 2^-5 each
        x[r] *= 2.0 ** e
    x[3, :3] = torch.tensor([2.0 ** -124, 2.0 ** -130, -(2.0 ** -128)], dtype=torch.float64) if dtype != "f16" else 0
    got = seq.unpack8(seq.pack8(x.to(dt).to(DEV)), dtype=torch.float32).cpu().double()
    assert torch.equal(x.to(dt).double(), x)
    big = x.abs().amax(1, keepdim=True)
    off = (got - x).abs()
    assert bool((off <= torch.clamp(big / 127.5, min=2.0 ** -128)).all())
    assert bool((off.amax(1)[:3] == big[:3, 0] / 127.5).all()) and (dtype == "f16" or float(off[3].max()) == 2.0 ** -128)
    top = torch.full((1, 32), torch.finfo(dt).max, dtype=dt, device=DEV)
    assert bool(((seq.unpack8(seq.pack8(top)).double() - top.double()).abs() <= top.double() / 127.5).all())


@gpu
def test_checkpoint_of_extreme_values():
    x = torch.zeros(8, 64, device=DEV)
    x[0, 3], x[1, 40], x[2, 0] = float("nan"), float("inf"), float("-inf")
    x[3, 5], x[4, 7], x[5, 33] = torch.finfo(torch.float32).max, 2.0 ** -149, -(2.0 ** -126)
    x[6, :32] = 2.0 ** -121 * 1.9999
    v = seq.unpack8(seq.pack8(x))
    codes, scales = plain_codes(x.cpu())
    want = codes.double() * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    for r, block in ((0, 0), (1, 1), (2, 0)):
        assert bool(torch.isnan(v[r, 32 * block:32 * block + 32]).all()) and bool((v[r, 32 - 32 * block:64 - 32 * block] == 0).all())
    assert torch.equal(v[3:].cpu().double(), want[3:]) and bool((v[7] == 0).all()) and bool(torch.isfinite(v[3:]).all())
    for dt, top in ((torch.float16, 2.0 ** 15), (torch.bfloat16, 2.0 ** 127)):
        x = torch.tensor([[torch.finfo(dt).max, 1.0] + [0.0] * 30, [-torch.finfo(dt).max] * 32], dtype=dt, device=DEV)
        codes, scales = plain_codes(x.cpu().float(), top)
        v = seq.unpack8(seq.pack8(x))
        assert torch.equal(v.cpu().double(), codes.double() * torch.exp2(scales.double() - 127)) and bool(torch.isfinite(v).all())


# ---------------------------------------------------------------- together
@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompts_then_single_rows_give_what_one_pass_gives(dtype):
    """Convolution and scan over packed prompts of unequal length, their states put into a cache, then row by row through the cache, against
    one pass over the whole series."""
    g = torch.Generator().manual_seed(11)
    D, N, W, dt = 72, 16, 4, DT[dtype]
    lens, more, slots = [3, 0, 41, 1], 4, 6
    total = [n + more for n in lens]
    w, b, A, skip, bias = rnd(g, D, W, scale=0.5), rnd(g, D), -torch.exp(rnd(g, D, N)), rnd(g, D), rnd(g, D) - 2
    x, z = [rnd(g, n, D, dtype=dt) for n in total], [rnd(g, n, D, dtype=dt) for n in total]
    d, Bm, Cm = [rnd(g, n, D, dtype=dt) for n in total], [rnd(g, n, N, dtype=dt) for n in total], [rnd(g, n, N, dtype=dt) for n in total]
    at = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)
    head = lambda v: torch.cat([a[:n] for a, n in zip(v, lens)])  # noqa: E731
    c, cst = seq.causal_conv(head(x), w, b, silu=True, seq_start=at, return_state=True)
    y, hst = seq.selective_scan(c, head(d), A, head(Bm), head(Cm), D=skip, z=head(z), dt_bias=bias, seq_start=at, return_state=True)
    where = torch.tensor([4, 0, 5, 2], device=DEV)
    ccache, hcache = torch.zeros(slots, W - 1, D, dtype=dt, device=DEV), torch.zeros(slots, D, N, device=DEV)
    ccache[where], hcache[where] = cst, hst
    got = [[y[lo:hi]] for lo, hi in zip(at[:-1].tolist(), at[1:].tolist())]
    for k in range(more):
        row = lambda v: torch.stack([a[n + k] for a, n in zip(v, lens)])  # noqa: E731
        c1 = seq.causal_conv_step(row(x), w, b, ccache, where.to(torch.int32), silu=True)
        y1 = seq.selective_scan_step(c1, row(d), A, row(Bm), row(Cm), hcache, where.to(torch.int32), D=skip, z=row(z), dt_bias=bias)
        for s in range(4):
            got[s].append(y1[s:s + 1])
    for s in range(4):
        c1, cend = seq.causal_conv(x[s][None], w, b, silu=True, return_state=True)
        y1, hend = seq.selective_scan(c1, d[s][None], A, Bm[s][None], Cm[s][None], D=skip, z=z[s][None], dt_bias=bias, return_state=True)
        a, e = torch.cat(got[s]).double(), y1[0].double()
        # both are roundings of the same sums, formed in another order: a unit of the type, and 1e-5 for the order
        assert bool(((a - e).abs() <= torch.finfo(dt).eps * e.abs() + 1e-5 * (1 + e.abs())).all())
        assert torch.equal(ccache[where[s]], cend[0]) and bool(((hcache[where[s]] - hend[0]).abs() <= 1e-5 * (1 + hend[0].abs())).all())


@gpu
@pytest.mark.parametrize("packed", [False, True])
def test_training_step_through_both_operators(packed):
    """conv -> scan and back, the inputs kept as they are or in 8 bits: the gradients against differences of the whole (kept as they are), and
    against the same chain at the restored values (8 bits)."""
    g = torch.Generator().manual_seed(4)
    D, N, W, B, T = 40, 4, 4, 2, 45
    dt = torch.float32 if packed else torch.float64
    pt = param_of(dt)
    x, z, d = (rnd(g, B, T, D, dtype=dt) for _ in range(3))
    w, b, A, skip, bias = rnd(g, D, W, dtype=pt, scale=0.5), rnd(g, D, dtype=pt), -torch.exp(rnd(g, D, N, dtype=pt)), rnd(g, D, dtype=pt), rnd(g, D, dtype=pt) - 1
    Bm, Cm, dy = rnd(g, B, T, N, dtype=dt), rnd(g, B, T, N, dtype=dt), rnd(g, B, T, D, dtype=dt)

    def forward(k):
        return seq.selective_scan(seq.causal_conv(k["x"], k["w"], k["b"], silu=True), d, k["A"], Bm, Cm, D=skip, z=k["z"], dt_bias=bias)

    def backward(x_, z_):
        u = seq.causal_conv(x_, w, b, silu=True)
        s = seq.selective_scan_grad(dy, u, d, A, Bm, Cm, D=skip, z=z_, dt_bias=bias)
        c = seq.causal_conv_grad(s.u, x_, w, b, silu=True)
        return dict(x=c.x, w=c.weight, b=c.bias, A=s.A, z=s.z)

    if not packed:
        difference_test(lambda k: float((forward(k) * dy).sum()), dict(x=x, w=w, b=b, A=A, z=z), backward(x, z))
        return
    px, pz = seq.pack8(x), seq.pack8(z)
    got, want = backward(px, pz), backward(seq.unpack8(px), seq.unpack8(pz))
    for k in got:
        assert torch.equal(got[k], want[k]), k


# ---------------------------------------------------------------- how the arrays lie
@gpu
def test_arrays_of_other_strides():
    """Maps whose states are not neighbours, an input shared by the batch (stride 0), channels that are not contiguous, parameters in the data's type:
    the same values as contiguous copies."""
    g = torch.Generator().manual_seed(8)
    B, T, D, N, G, dt = 2, 33, 24, 16, 3, torch.bfloat16
    u, d, z = rnd(g, 1, T, D, dtype=dt).expand(B, T, D), rnd(g, B, D, T, dtype=dt).transpose(1, 2), rnd(g, B, T, 2 * D, dtype=dt)[..., D:]
    A, skip, bias = (-torch.exp(rnd(g, D, N))).to(dt), rnd(g, D, dtype=dt), rnd(g, D, dtype=dt) - 1
    Bm, Cm, dy = rnd(g, B, T, N, G, dtype=dt).transpose(2, 3), rnd(g, B, T, G, 2 * N, dtype=dt)[..., ::2], rnd(g, B, T, D, dtype=dt)
    given = dict(u=u, dt=d, A=A, B=Bm, C_=Cm, D=skip, z=z, dt_bias=bias)
    plain = {k: v.contiguous() if k not in ("A", "D", "dt_bias") else v.float() for k, v in given.items()}
    assert not any(given[k].is_contiguous() for k in ("u", "dt", "z", "B", "C_"))
    assert torch.equal(seq.selective_scan(**given), seq.selective_scan(**plain))
    for a, b in zip(seq.selective_scan_grad(dy, **given), seq.selective_scan_grad(dy, **plain)):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))
    w = rnd(g, 4, D, dtype=dt).t()
    assert torch.equal(seq.causal_conv(z, w, skip), seq.causal_conv(z.contiguous(), w.float().contiguous(), skip.float()))
    row = lambda k: given[k][:, 5]  # noqa: E731
    s1, s2 = (torch.zeros(B, D, N, device=DEV) for _ in range(2))
    y1 = seq.selective_scan_step(row("u"), row("dt"), A, row("B"), row("C_"), s1, D=skip, z=row("z"), dt_bias=bias)
    y2 = seq.selective_scan_step(*(row(k).contiguous() for k in ("u", "dt")), A.float(), row("B").contiguous(), row("C_").contiguous(), s2, D=skip.float(), z=row("z").contiguous(),
                                 dt_bias=bias.float())
    assert torch.equal(y1, y2) and torch.equal(s1, s2)
    assert torch.equal(seq.unpack8(seq.pack8(d)), seq.unpack8(seq.pack8(d.contiguous())))


@gpu
def test_single_rows_of_any_stride():
    """One row a sequence, cut out of arrays with time as the fastest index: the stride between rows means nothing, for results and for states of one row either."""
    g = torch.Generator().manual_seed(9)
    n, D, N = 3, 12, 4
    late = lambda k: torch.full((n, D, k), 7.0, device=DEV).transpose(1, 2)  # noqa: E731
    x, m, w, A = rnd(g, n, D, 1).transpose(1, 2), rnd(g, n, 1, N), rnd(g, D, 2), -torch.exp(rnd(g, D, N))
    state = rnd(g, n, D, 1).transpose(1, 2)
    assert x.stride() == (D, 1, 1) and late(1).stride() == (D, 1, 1)
    y, end = seq.causal_conv(x, w, state=state, return_state=True)
    assert torch.equal(seq.causal_conv(x, w, state=state, out=late(1)), y)
    assert torch.equal(seq.selective_scan(x, x, A, m, m, out=late(1)), seq.selective_scan(x.contiguous(), x.contiguous(), A, m, m))
    st = late(1)
    st.copy_(state)
    assert st.stride() == (D, 1, 1) and torch.equal(seq.causal_conv_step(x[:, 0], w, None, st), y[:, 0]) and torch.equal(st, end)
    one = rnd(g, 1, D).as_strided((1, D), (1, 1))
    assert torch.equal(seq.causal_conv_step(one, w, None, rnd(g, 1, 1, D) * 0, out=torch.empty(D, device=DEV).as_strided((1, D), (1, 1))), seq.causal_conv(one[None], w)[0])


def shifted(x):
    """x one element behind a 16-byte boundary, contiguous as before."""
    if x is None or x.numel() == 0:
        return x
    y = torch.empty(x.numel() + 32, dtype=x.dtype, device=x.device)
    at = next(i for i in range(32) if y[i:].data_ptr() % 16 == x.element_size() % 16)
    y = y[at:at + x.numel()].view(x.shape)
    y.copy_(x)
    assert y.is_contiguous() and y.data_ptr() % 16 != 0
    return y


@gpu
@pytest.mark.parametrize("dtype,W,N", [("f32", 4, 16), ("f32", 3, 8), ("bf16", 4, 16), ("bf16", 7, 12), ("f16", 1, 4), ("f16", 8, 20), ("f64", 4, 8), ("f64", 6, 5)])
@pytest.mark.parametrize("which", ["parameters", "all"])
def test_arrays_off_their_alignment(dtype, W, N, which):
    """Parameters, or all arrays, one element behind a 16-byte boundary: the narrow loads give the bits of the wide ones."""
    g = torch.Generator().manual_seed(W)
    B, T, D, dt = 2, 90, 64, DT[dtype]
    pt = param_of(dt)
    x, d, z, dy = (rnd(g, B, T, D, dtype=dt) for _ in range(4))
    Bm, Cm = (rnd(g, B, T, N, dtype=dt) for _ in range(2))
    w, b, A, skip, bias = (v.to(pt) for v in (rnd(g, D, W), rnd(g, D), -torch.exp(rnd(g, D, N)), rnd(g, D), rnd(g, D)))
    cst, hst, dhs = rnd(g, B, W - 1, D, dtype=dt), rnd(g, B, D, N).to(pt), rnd(g, B, D, N).to(pt)

    def run(par, arr):
        kw = dict(D=par(skip), dt_bias=par(bias), z=arr(z))
        y, end = seq.causal_conv(arr(x), par(w), par(b), silu=True, state=arr(cst), return_state=True)
        cg = seq.causal_conv_grad(arr(dy), arr(x), par(w), par(b), silu=True, state=arr(cst), dstate=arr(cst))
        s, h = seq.selective_scan(arr(x), arr(d), par(A), arr(Bm), arr(Cm), state=par(hst), return_state=True, **kw)
        sg = seq.selective_scan_grad(arr(dy), arr(x), arr(d), par(A), arr(Bm), arr(Cm), state=par(hst), dstate=par(dhs), **kw)
        c1, h1 = arr(cst.clone()), par(hst.clone())
        row = lambda v: arr(v[:, 3].contiguous())  # noqa: E731
        y1 = seq.causal_conv_step(row(x), par(w), par(b), c1)
        y2 = seq.selective_scan_step(row(x), row(d), par(A), row(Bm), row(Cm), h1, D=par(skip), z=row(z))
        back = [] if dtype == "f64" else [seq.unpack8(seq.pack8(arr(x)))]
        return [y, end, *cg, s, h, *sg, c1, h1, y1, y2, *back]

    keep = lambda v: v  # noqa: E731
    for k, (p, q) in enumerate(zip(run(keep, keep), run(shifted, shifted if which == "all" else keep))):
        assert torch.equal(p, q), k


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_nothing_to_do(dtype):
    """No sequences, no rows, only empty sequences: states pass through, gradients of parameters are 0."""
    g = torch.Generator().manual_seed(2)
    D, N, W, dt = 12, 16, 4, DT[dtype]
    w, A = rnd(g, D, W), -torch.exp(rnd(g, D, N))
    for shape, n, kw in (((0, 5, D), 0, {}), ((6, D), 0, dict(seq_start=torch.zeros(1, dtype=torch.int32, device=DEV))), ((3, 0, D), 3, {}), ((0, D), 2, dict(seq_start=torch.zeros(3, dtype=torch.int32, device=DEV))),
                         ((4, D), 2, dict(seq_start=torch.tensor([1, 1, 1], dtype=torch.int32, device=DEV)))):
        x = rnd(g, *shape, dtype=dt)
        m = rnd(g, *shape[:-1], N, dtype=dt)
        cst, hst = rnd(g, n, W - 1, D, dtype=dt), rnd(g, n, D, N)
        y, end = seq.causal_conv(x, w, state=cst, return_state=True, **kw)
        assert y.shape == x.shape and torch.equal(end, cst) and not bool(y.any())
        y, end = seq.selective_scan(x, x, A, m, m, state=hst, return_state=True, **kw)
        assert y.shape == x.shape and torch.equal(end, hst) and not bool(y.any())
        gc = seq.causal_conv_grad(x, x, w, state=cst, dstate=cst, **kw)
        assert not bool(gc.x.any()) and not bool(gc.weight.any()) and torch.equal(gc.state, cst)
        gs = seq.selective_scan_grad(x, x, x, A, m, m, D=A[:, 0], state=hst, dstate=hst, **kw)
        assert not any(bool(v.any()) for v in (gs.u, gs.dt, gs.A, gs.B, gs.C, gs.D)) and torch.equal(gs.state, hst)
    y = seq.selective_scan_step(*(torch.zeros(0, D, dtype=dt, device=DEV),) * 2, A, *(torch.zeros(0, N, dtype=dt, device=DEV),) * 2, torch.zeros(2, D, N, device=DEV))
    assert y.shape == (0, D)
    assert seq.causal_conv_step(torch.zeros(0, D, dtype=dt, device=DEV), w, None, torch.zeros(2, W - 1, D, dtype=dt, device=DEV)).shape == (0, D)


# ---------------------------------------------------------------- streams, graphs, sizes: the device only
def everything(D=96, N=16, rows=200, dtype=torch.bfloat16, seed=0):
    """Inputs, and a function that runs every operator on them and returns all results."""
    g = torch.Generator().manual_seed(seed)
    at = torch.tensor([0, 70, 70, rows], dtype=torch.int32, device=DEV)
    x, d, z, dy = (rnd(g, rows, D, dtype=dtype) for _ in range(4))
    Bm, Cm, w, b = rnd(g, rows, N, dtype=dtype), rnd(g, rows, N, dtype=dtype), rnd(g, D, 4, scale=0.5), rnd(g, D)
    A, skip, bias, st = -torch.exp(rnd(g, D, N)), rnd(g, D), rnd(g, D) - 2, rnd(g, 3, D, N)

    def run():
        kw = dict(D=skip, dt_bias=bias, seq_start=at, state=st)
        px, pz = seq.pack8(x), seq.pack8(z)
        c = seq.causal_conv(x, w, b, silu=True, seq_start=at)
        y, end = seq.selective_scan(c, d, A, Bm, Cm, z=z, return_state=True, **kw)
        s = seq.selective_scan_grad(dy, c, d, A, Bm, Cm, z=pz, **kw)
        cg = seq.causal_conv_grad(s.u, px, w, b, silu=True, seq_start=at)
        h, cs = end.clone(), x[:9].view(3, 3, D).clone()
        c1 = seq.causal_conv_step(x[:3], w, b, cs, silu=True)
        y1 = seq.selective_scan_step(c1, d[:3], A, Bm[:3], Cm[:3], h, D=skip, z=z[:3], dt_bias=bias)
        return [seq.unpack8(px), c, y, end, *s, *cg[:3], cs, h, c1, y1]

    return dict(x=x, d=d, z=z, dy=dy, B=Bm, C=Cm), run


def same(a, b):
    return all(p is None and q is None or torch.equal(p, q) for p, q in zip(a, b))


@gpu
def test_on_a_stream_of_its_own_and_two_at_once():
    if DEV == "cpu":
        pytest.skip("the emulated device has no streams")
    calls = [everything(seed=k)[1] for k in range(2)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = []
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(c())
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(got, want))


@gpu
def test_captured_into_two_graphs_and_replayed():
    """Two captured graphs, replayed in turn with other inputs, eager calls and waits between them, give what eager calls give."""
    if DEV == "cpu":
        pytest.skip("the emulated device has no graphs")
    sets = [everything(seed=10 + k) for k in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _, run in sets:
            run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _, run in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for turn in range(4):
        for k in (0, 1, 1, 0):
            inputs, run = sets[k]
            for v in inputs.values():
                v.copy_(torch.randn(v.shape, generator=torch.Generator().manual_seed(turn * 7 + k), dtype=torch.float32))
            graphs[k][0].replay()
            torch.cuda.synchronize()
            got = [None if v is None else v.clone() for v in graphs[k][1]]
            want = run()
            torch.cuda.synchronize()
            assert same(got, want), (turn, k)


@gpu
def test_arrays_over_two_to_the_31_elements():
    """Rows far behind 2^31 elements: the last of them against a call on them alone that starts from the state in front."""
    if DEV == "cpu":
        pytest.skip("sizes for the device")
    D, T, tail, N = 8192, 266_000, 40, 8
    assert D * T > 2 ** 31 + D * tail
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(1, T, D, generator=g, device=DEV, dtype=torch.bfloat16)
    w = torch.randn(D, 4, generator=g, device=DEV)
    y = seq.causal_conv(x, w, silu=True)
    assert torch.equal(y[:, -tail:], seq.causal_conv(x[:, -tail:], w, silu=True, state=x[:, -tail - 3:-tail].contiguous()))
    gx = seq.causal_conv_grad(y, x, w, silu=True).x
    assert torch.equal(gx[:, -tail:], seq.causal_conv_grad(y[:, -tail:], x[:, -tail:], w, silu=True, state=x[:, -tail - 3:-tail].contiguous()).x)
    del gx
    p = seq.pack8(x)
    q = seq.pack8(x[:, -tail:].contiguous())
    assert torch.equal(p.codes[:, -tail:], q.codes) and torch.equal(p.scales[:, -tail:], q.scales)
    assert torch.equal(seq.unpack8(p)[:, -tail:], seq.unpack8(q))
    del p, q
    A, m = -torch.rand(D, N, generator=g, device=DEV) - 0.5, torch.randn(1, T, N, generator=g, device=DEV, dtype=torch.bfloat16)
    _, st = seq.selective_scan(x[:, :-tail], x[:, :-tail], A, m[:, :-tail], m[:, :-tail], return_state=True, out=y[:, :-tail])
    yy, end = seq.selective_scan(x[:, -tail:], x[:, -tail:], A, m[:, -tail:], m[:, -tail:], state=st, return_state=True)
    y, e = seq.selective_scan(x, x, A, m, m, return_state=True, out=y)
    # chunks elsewhere: a unit of bfloat16, and 1e-5 of the sums' size for the order
    a, b = y[:, -tail:].double(), yy.double()
    assert bool(((a - b).abs() <= 2.0 ** -7 * b.abs() + 1e-4).all()) and bool(((e - end).abs() <= 1e-4 * (1 + end.abs())).all())


# ---------------------------------------------------------------- refusals: before any launch
def args(**over):
    g = torch.Generator().manual_seed(0)
    a = dict(u=rnd(g, 2, 6, 8), dt=rnd(g, 2, 6, 8), A=-torch.ones(8, 4, device=DEV), B=rnd(g, 2, 6, 4), C_=rnd(g, 2, 6, 4))
    a.update(over)
    return a


def bad_scans():
    z = lambda *s, **k: torch.zeros(*s, device=DEV, **k)  # noqa: E731
    return {"u shape": (ValueError, args(u=z(2, 6, 9))), "u type": (ValueError, args(u=z(2, 6, 8, dtype=torch.float16))), "integer": (TypeError, args(dt=z(2, 6, 8, dtype=torch.int32))),
            "A rows": (ValueError, args(A=z(9, 4))), "no states": (ValueError, args(A=z(8, 0))), "states": (ValueError, args(A=z(8, 257), B=z(2, 6, 257), C_=z(2, 6, 257))),
            "B rows": (ValueError, args(B=z(2, 5, 4))), "B states": (ValueError, args(B=z(2, 6, 5))), "groups": (ValueError, args(B=z(2, 6, 3, 4), C_=z(2, 6, 3, 4))),
            "B and C": (ValueError, args(B=z(2, 6, 2, 4))), "D": (ValueError, args(D=z(7))), "bias": (ValueError, args(dt_bias=z(8, 1))), "state": (ValueError, args(state=z(2, 8, 5))),
            "state type": (ValueError, args(state=z(2, 8, 4, dtype=torch.float16))), "starts type": (ValueError, args(seq_start=z(3, dtype=torch.int64))),
            "dense rows with offsets": (ValueError, args(seq_start=z(3, dtype=torch.int32))), "both": (ValueError, args(seq_start=z(3, dtype=torch.int32), lengths=z(2, dtype=torch.int32))),
            "lengths": (ValueError, args(lengths=z(3, dtype=torch.int32))), "out": (ValueError, args(out=z(2, 6, 8, dtype=torch.float16)))}


@gpu
@pytest.mark.parametrize("what", ["u shape", "u type", "integer", "A rows", "no states", "states", "B rows", "B states", "groups", "B and C", "D", "bias", "state", "state type", "starts type",
                                  "dense rows with offsets", "both", "lengths", "out"])
def test_scan_refuses(what):
    err, a = bad_scans()[what]
    with pytest.raises(err):
        seq.selective_scan(**a)


@gpu
def test_other_refusals():
    z = lambda *s, **k: torch.zeros(*s, device=DEV, **k)  # noqa: E731
    p = seq.pack8(z(2, 6, 8))
    for err, call in [
            (ValueError, lambda: seq.causal_conv(z(2, 6, 8), z(8, 9))), (ValueError, lambda: seq.causal_conv(z(2, 6, 8), z(7, 4))), (ValueError, lambda: seq.causal_conv(z(6, 8), z(8, 4))),
            (ValueError, lambda: seq.causal_conv(z(2, 6, 8), z(8, 4), state=z(2, 4, 8))), (ValueError, lambda: (lambda x: seq.causal_conv(x, z(8, 4), out=x))(z(2, 6, 8))),
            (ValueError, lambda: (lambda x: seq.causal_conv_step(x, z(8, 4), None, z(2, 3, 8), out=x))(z(2, 8))), (RuntimeError, lambda: seq.causal_conv(z(2, 6, 8), z(8, 4), out=z(1, 6, 8).expand(2, 6, 8))),
            (ValueError, lambda: (lambda x: seq.selective_scan(z(2, 6, 8), x, z(8, 4), z(2, 6, 4), z(2, 6, 4), out=x))(z(2, 6, 8))),
            (ValueError, lambda: (lambda x: seq.selective_scan_step(x, z(2, 8), z(8, 4), z(2, 4), z(2, 4), z(2, 8, 4), out=x))(z(2, 8))), (ValueError, lambda: seq.causal_conv_grad(z(2, 6, 7), z(2, 6, 8), z(8, 4))),
            (TypeError, lambda: seq.causal_conv_grad(p, z(2, 6, 8), z(8, 4))), (TypeError, lambda: seq.selective_scan(**args(dt=p))),
            (ValueError, lambda: seq.causal_conv_step(z(3, 8), z(8, 4), None, z(2, 3, 8))), (ValueError, lambda: seq.causal_conv_step(z(3, 8), z(8, 4), None, z(4, 3, 8), z(2, dtype=torch.int32))),
            (ValueError, lambda: seq.selective_scan_step(z(3, 8), z(3, 8), z(8, 4), z(3, 4), z(3, 4), z(2, 8, 4))),
            (TypeError, lambda: seq.selective_scan_step(p, z(3, 8), z(8, 4), z(3, 4), z(3, 4), z(4, 8, 4))), (TypeError, lambda: seq.pack8(z(4, 8, dtype=torch.float64))),
            (ValueError, lambda: seq.Packed8(z(4, 33, dtype=torch.int8), z(4, 1, dtype=torch.uint8), torch.float32)),
            (TypeError, lambda: seq.Packed8(z(4, 32), z(4, 1, dtype=torch.uint8), torch.float32)), (TypeError, lambda: seq.unpack8(p, dtype=torch.float64))]:
        with pytest.raises(err):
            call()


def test_there_is_no_cpu_path():
    if seq._EMULATED:
        pytest.skip("the emulated device's memory is the host's")
    with pytest.raises(ValueError):
        seq.causal_conv(torch.zeros(1, 2, 3), torch.zeros(3, 4))
    with pytest.raises(ValueError):
        seq.pack8(torch.zeros(2, 32))


def test_c_entry_points_refuse_before_any_launch():
    """The C ABI by itself: sizes, missing arrays, types, workspace -- refused with a message, on a host without a device too.  The pointers are
    made up, so the calls name a device that does not exist: one that got past every check would be refused for that."""
    import ctypes as C
    lib = L.lib
    said = lambda: lib.crnn_last_error(None).decode()  # noqa: E731

    def view(dt=L.DT_F32, rs=8, ptr=4096, ss=8192):
        return L.View(ptr=ptr, row_stride=rs, seq_stride=ss, dtype=dt)

    def scan(**over):
        a = L.ScanArgs(struct_size=C.sizeof(L.ScanArgs), device=99, n_seq=2, D=8, N=4, G=1, rows=6, A=4096, u=view(), dt=view(), y=view(ptr=64), B=view(rs=4), C=view(rs=4))
        for k, v in over.items():
            setattr(a, k, v)
        return a

    for over, word in [(dict(struct_size=8), "struct_size"), (dict(N=0), "N must"), (dict(N=257), "N must"), (dict(G=3), "divide"), (dict(rows=-1), "negative"), (dict(rows=1 << 31), "rows"),
                       (dict(D=0), "D must"), (dict(A=None), "A is missing"), (dict(u=view(ptr=None)), "u is missing"), (dict(u=view(L.DT_BF16)), "element type"),
                       (dict(u=view(L.DT_PACKED8)), "scales"), (dict(dt=view(L.DT_PACKED8)), "checkpoint"), (dict(y=view(rs=7)), "overlap"), (dict(y=view(ptr=64, ss=47)), "sequences of an output overlap"),
                       (dict(y=view(ptr=64, rs=15, ss=8)), "sequences of an output overlap"), (dict(y=view(ptr=64, rs=16, ss=8)), "device"), (dict(y=view()), "also an input"), (dict(dtype=9), "element type"),
                       (dict(seq_start=64, seq_len=64), "exclude"), (dict(rows=600), "workspace"), ({}, "device")]:
        assert lib.crnn_scan_forward(C.byref(scan(**over))) == -1 and word in said(), (over, said())
    assert lib.crnn_scan_forward(None) == -1 and "null" in said()
    assert lib.crnn_scan_workspace(C.byref(scan()), 2) == -1 and lib.crnn_scan_workspace(C.byref(scan()), 0) == 0 and lib.crnn_scan_workspace(C.byref(scan(rows=600)), 0) > 0
    assert lib.crnn_scan_backward(C.byref(scan())) == -1 and "dA" in said()
    assert lib.crnn_scan_step(C.byref(scan(n_slots=1))) == -1 and "n_slots" in said()

    def conv(**over):
        a = L.ConvArgs(struct_size=C.sizeof(L.ConvArgs), device=99, n_seq=2, D=8, W=4, rows=6, weight=4096, x=view(), y=view(ptr=64))
        for k, v in over.items():
            setattr(a, k, v)
        return a

    for over, word in [(dict(struct_size=0), "struct_size"), (dict(W=0), "W must"), (dict(W=9), "W must"), (dict(weight=None), "weight"), (dict(x=view(ptr=None)), "x is missing"),
                       (dict(y=view(rs=4)), "overlap"), (dict(state_in=view(), state_out=view()), "state_out"), (dict(y=view()), "also an input"), (dict(y=view(ptr=64, ss=0)), "sequences"),
                       (dict(state_out=view(ptr=64, ss=23)), "sequences"), ({}, "device")]:
        assert lib.crnn_conv_forward(C.byref(conv(**over))) == -1 and word in said(), (over, said())
    assert lib.crnn_conv_backward(C.byref(conv(dx=view(ptr=64), dy=view(), dweight=64))) == -1 and "workspace" in said()
    assert lib.crnn_conv_backward(C.byref(conv(dx=view(), dy=view(), dweight=64))) == -1 and "also an input" in said()
    assert lib.crnn_scan_backward(C.byref(scan(dA=64, dy=view(), du=view(ptr=64), ddt=view(), dB=view(rs=4, ptr=64), dC=view(rs=4, ptr=64)))) == -1 and "also an input" in said()
    assert lib.crnn_conv_step(C.byref(conv(n_slots=1))) == -1 and "n_slots" in said()
    v = view(L.DT_F64)
    assert lib.crnn_pack8(99, None, C.byref(v), 2, 8, 4096, 4096) == -1 and "half" in said()
    v = view()
    assert lib.crnn_unpack8(99, None, 4096, None, 2, 8, C.byref(v)) == -1 and "missing" in said()


def test_launches_the_card_would_cut_off_are_refused():
    """A grid counts its threads in 32 bits: 2^24 blocks of 256 and more would be cut off without an error.  Sizes alone decide, on a host without a device too (a call that
    gets past the checks is refused for a device that does not exist)."""
    import ctypes as C
    lib = L.lib

    def view(ptr, D, n):
        return L.View(ptr=ptr, row_stride=D, seq_stride=D, dtype=L.DT_BF16)

    def scan(n, D, N, **over):
        v = {k: view((1 + i) << 44, D if k in ("u", "dt", "y", "dy", "du", "ddt") else N, n) for i, k in enumerate(("u", "dt", "y", "B", "C", "dy", "du", "ddt", "dB", "dC"))}
        a = L.ScanArgs(struct_size=C.sizeof(L.ScanArgs), device=99, n_seq=n, D=D, N=N, G=1, rows=1, dtype=L.DT_BF16, A=1 << 40, dA=1 << 41, workspace=1 << 42, workspace_bytes=1 << 62, **v)
        for k, w in over.items():
            setattr(a, k, w)
        return a

    def conv(n, D, **over):
        v = {k: view((1 + i) << 44, D, n) for i, k in enumerate(("x", "y", "dy", "dx"))}
        a = L.ConvArgs(struct_size=C.sizeof(L.ConvArgs), device=99, n_seq=n, D=D, W=1, rows=1, dtype=L.DT_BF16, weight=1 << 40, dweight=1 << 41, workspace=1 << 42, workspace_bytes=1 << 62, **v)
        for k, w in over.items():
            setattr(a, k, w)
        return a

    top = (1 << 24) - 1
    for call, args, word in [
            (lib.crnn_scan_forward, scan(top // 32, 2048, 8), "device"), (lib.crnn_scan_forward, scan(top // 32 + 1, 2048, 8), "too many"),
            (lib.crnn_scan_forward, scan((1 << 19) + 8, 2048, 8), "too many"), (lib.crnn_scan_workspace, scan(1 << 28, 2048, 8), "too many"),
            # the gradient: four tiles a block, and a thread for each sequence, state and channel of the carry
            (lib.crnn_scan_backward, scan(top // 64, 2048, 8), "device"), (lib.crnn_scan_backward, scan(top // 64 + 1, 2048, 8), "too many"),
            # four wavefronts a block, four channels a lane (one where a row does not allow that)
            (lib.crnn_conv_forward, conv(top // 8 * 4, 2048), "device"), (lib.crnn_conv_forward, conv(top // 8 * 4 + 4, 2048), "too many"),
            (lib.crnn_conv_forward, conv(top // 33 * 4 + 4, 2049), "too many"), (lib.crnn_conv_backward, conv(top // 8 * 4, 2048), "device"),
            (lib.crnn_conv_backward, conv(top // 8 * 4 + 4, 2048), "too many"),
            # single rows: a block has 256 threads of four channels
            (lib.crnn_conv_step, conv(top // 2, 2048, n_slots=1 << 30), "device"), (lib.crnn_conv_step, conv(top // 2 + 1, 2048, n_slots=1 << 30), "too many"),
            (lib.crnn_scan_step, scan(top // 2, 2048, 1, n_slots=1 << 30, state_out=1 << 43), "device"), (lib.crnn_scan_step, scan(top // 2 + 1, 2048, 1, n_slots=1 << 30, state_out=1 << 43), "too many")]:
        got = call(C.byref(args), 0) if call is lib.crnn_scan_workspace else call(C.byref(args))
        assert got == -1 and word in lib.crnn_last_error(None).decode(), (word, lib.crnn_last_error(None).decode())
    v = L.View(ptr=1 << 44, row_stride=4096, dtype=L.DT_BF16)
    for rows, word in ((top, "device"), (top + 1, "too many")):
        assert lib.crnn_pack8(99, None, C.byref(v), rows, 4096, 1 << 45, 1 << 46) == -1 and word in lib.crnn_last_error(None).decode()


@gpu
def test_the_largest_launch_reaches_its_last_rows():
    if DEV == "cpu":
        pytest.skip("sizes for the device")
    n, D, N = ((1 << 24) - 1) // 32, 2048, 8
    g = torch.Generator(device=DEV).manual_seed(0)
    u = torch.randn(n, 1, D, generator=g, device=DEV, dtype=torch.bfloat16)
    A, m, w = -torch.rand(D, N, generator=g, device=DEV), torch.randn(n, 1, N, generator=g, device=DEV, dtype=torch.bfloat16), torch.randn(D, 2, generator=g, device=DEV)
    y = seq.selective_scan(u, u, A, m, m, out=torch.full_like(u, 7.0))
    for rows in (slice(0, 9), slice(n // 2, n // 2 + 9), slice(n - 9, n)):
        assert torch.equal(y[rows], seq.selective_scan(u[rows], u[rows], A, m[rows], m[rows]))
    assert not bool((y == 7).all(-1).any())
    with pytest.raises(L.CrnnError, match="too many"):
        seq.selective_scan(torch.empty(n + 1, 1, D, dtype=torch.bfloat16, device=DEV), torch.empty(n + 1, 1, D, dtype=torch.bfloat16, device=DEV), A,
                           *(torch.empty(n + 1, 1, N, dtype=torch.bfloat16, device=DEV),) * 2)


@gpu
@pytest.mark.parametrize("zero", [0, 1])
@pytest.mark.parametrize("packed", [False, True])
def test_rows_of_gradients_outside_the_sequences_are_kept_or_cleared(packed, zero):
    """The C ABI's zero_outside, all five row gradients of the scan and the convolution's."""
    import ctypes as C
    g = torch.Generator().manual_seed(5)
    n, T, D, N, G = (1, 50, 12, 4, 2) if packed else (2, 25, 12, 4, 2)
    at = torch.tensor([7, 31], dtype=torch.int32, device=DEV) if packed else torch.tensor([25, 9], dtype=torch.int32, device=DEV)
    outside = torch.ones(50, dtype=torch.bool)
    for lo, hi in ([(7, 31)] if packed else [(0, 25), (25, 34)]):
        outside[lo:hi] = False
    rows = [rnd(g, 50, D) for _ in range(4)]
    maps = [rnd(g, 50, G * N) for _ in range(2)]
    A, dA, w, dw = -torch.exp(rnd(g, D, N)), torch.zeros(D, N, device=DEV), rnd(g, D, 3), torch.zeros(D, 3, device=DEV)
    out = [torch.full((50, D), 7.0, device=DEV) for _ in range(4)] + [torch.full((50, G * N), 7.0, device=DEV) for _ in range(2)]
    view = lambda x: L.View(ptr=x.data_ptr(), row_stride=x.shape[1], seq_stride=0 if packed else T * x.shape[1], dtype=L.DT_F32)  # noqa: E731
    stream = 0 if DEV == "cpu" else torch.cuda.current_stream().cuda_stream
    kw = dict(n_seq=n, D=D, rows=T, dtype=L.DT_F32, zero_outside=zero, stream=stream, **{"seq_start" if packed else "seq_len": at.data_ptr()})
    a = L.ScanArgs(struct_size=C.sizeof(L.ScanArgs), N=N, G=G, softplus=1, A=A.data_ptr(), dA=dA.data_ptr(), B_group=N, B_state=1, C_group=N, C_state=1,
                   **{k: view(x) for k, x in zip(("u", "dt", "z", "dy", "B", "C", "du", "ddt", "dz", "dB", "dC"), rows + maps + out[:3] + out[4:])}, **kw)
    c = L.ConvArgs(struct_size=C.sizeof(L.ConvArgs), W=3, weight=w.data_ptr(), dweight=dw.data_ptr(), x=view(rows[0]), dy=view(rows[1]), dx=view(out[3]), **kw)
    for args, need, call in ((a, L.lib.crnn_scan_workspace(C.byref(a), 1), L.lib.crnn_scan_backward), (c, L.lib.crnn_conv_workspace(C.byref(c)), L.lib.crnn_conv_backward)):
        ws = torch.empty(need, dtype=torch.uint8, device=DEV)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
        assert call(C.byref(args)) == 0, L.lib.crnn_last_error(None)
        if DEV != "cpu":
            torch.cuda.synchronize()
    for k, x in enumerate(out):
        assert bool((x.cpu()[outside] == (0 if zero else 7)).all()), k
        assert bool((x.cpu()[~outside] != 7).any(-1).all()) and bool((x.cpu()[~outside] != 0).any(-1).all()), k


@gpu
def test_autograd_is_not_cut_in_silence():
    """A tensor that requires a gradient, or carries a tangent, where the result could not have one: refused; values alone are fine."""
    import torch.autograd.forward_ad as fwd
    g = torch.Generator().manual_seed(1)
    n, T, D, N, W = 2, 5, 8, 4, 4
    c = dict(x=rnd(g, n, T, D), w=rnd(g, D, W), b=rnd(g, D), cst=rnd(g, n, W - 1, D), u=rnd(g, n, T, D), dt=rnd(g, n, T, D), A=-torch.exp(rnd(g, D, N)), B=rnd(g, n, T, N), C=rnd(g, n, T, N),
             D=rnd(g, D), z=rnd(g, n, T, D), bias=rnd(g, D), hst=rnd(g, n, D, N), dy=rnd(g, n, T, D), out=rnd(g, n, T, D), out1=rnd(g, n, D))
    calls = {
        "conv": (("x", "w", "b", "cst", "out"), lambda k: seq.causal_conv(k["x"], k["w"], k["b"], state=k["cst"], out=k["out"])),
        "conv_step": (("x", "w", "b", "cst", "out1"), lambda k: seq.causal_conv_step(k["x"][:, 0], k["w"], k["b"], k["cst"], out=k["out1"])),
        "scan": (("u", "dt", "A", "B", "C", "D", "z", "bias", "hst", "out"),
                 lambda k: seq.selective_scan(k["u"], k["dt"], k["A"], k["B"], k["C"], D=k["D"], z=k["z"], dt_bias=k["bias"], state=k["hst"], out=k["out"])),
        "scan_step": (("u", "dt", "A", "B", "C", "D", "z", "bias", "hst", "out1"),
                      lambda k: seq.selective_scan_step(k["u"][:, 0], k["dt"][:, 0], k["A"], k["B"][:, 0], k["C"][:, 0], k["hst"], D=k["D"], z=k["z"][:, 0], dt_bias=k["bias"], out=k["out1"]))}
    grads = {"conv_grad": (("dy", "x", "w", "b", "cst"), lambda k: seq.causal_conv_grad(k["dy"], k["x"], k["w"], k["b"], state=k["cst"])),
             "scan_grad": (("dy", "u", "dt", "A", "B", "C", "D", "z", "bias", "hst"),
                           lambda k: seq.selective_scan_grad(k["dy"], k["u"], k["dt"], k["A"], k["B"], k["C"], D=k["D"], z=k["z"], dt_bias=k["bias"], state=k["hst"]))}
    for names, call in calls.values():
        call(c)
        for name in names:
            asks = {**c, name: c[name].clone().requires_grad_()}
            with pytest.raises(RuntimeError, match="autograd"):
                call(asks)
            with torch.no_grad():
                call(asks)
            with torch.inference_mode():
                call({k: v.clone() for k, v in c.items()})
    for names, call in grads.values():
        want = call(c)
        for name in names:
            assert same(call({**c, name: c[name].clone().requires_grad_()}), want)
    for names, call in (*calls.values(), *grads.values()):
        with fwd.dual_level():
            call(c)
            for name in names:
                with pytest.raises(RuntimeError, match="tangent"):
                    call({**c, name: fwd.make_dual(c[name].clone(), torch.ones_like(c[name]))})
    assert not any(v.requires_grad for v in c.values())
    p = seq.pack8(c["x"].clone().requires_grad_())       # codes are whole numbers: nothing to lose
    assert torch.equal(seq.unpack8(p), seq.unpack8(seq.pack8(c["x"])))


@gpu
def test_results_over_parts_of_inputs_are_refused():
    """Memory that an input and a result share is found wherever it lies, not at equal pointers only; columns and blocks of one array beside each other are fine."""
    g = torch.Generator().manual_seed(3)
    n, T, D, N, W = 3, 9, 32, 4, 4
    w, A = rnd(g, D, W), -torch.exp(rnd(g, D, N))
    buf, m, st = rnd(g, n, T + 1, D), rnd(g, n, T, N), rnd(g, n, W - 1, D)
    conv = lambda x, out, **kw: seq.causal_conv(x, w, out=out, **kw)  # noqa: E731
    scan = lambda u, dt, out, B=m, C=m, **kw: seq.selective_scan(u, dt, A, B, C, out=out, **kw)  # noqa: E731
    x = rnd(g, n, T, D)
    one = rnd(g, 1, 40, D + 8)
    h, rows = rnd(g, 8, D, N), rnd(g, 5, D)
    big = rnd(g, 8 * D * N)
    wide = rnd(g, n, T, D * D)
    flat = rnd(g, n * T * D + n * T * N)
    for call in (lambda: conv(buf[:, :-1], buf[:, 1:]), lambda: conv(buf[:, 1:], buf[:, :-1]), lambda: conv(one[..., 1:D + 1], one[..., :D]), lambda: scan(x, buf[:, :-1], buf[:, 1:]),
                 lambda: scan(buf[:, :-1], x, buf[:, 1:]), lambda: scan(x, x, buf[:, 1:], z=buf[:, :-1]), lambda: scan(one[:, 1:, :D], one[:, 1:, 8:], one[:, :-1, :D], rnd(g, 1, 39, N), rnd(g, 1, 39, N)),
                 # a result inside the maps, a state, the weights, and the states of the single steps
                 lambda: scan(x, x, flat[n * T * N - 4:][:n * T * D].view(n, T, D), flat[:n * T * N].view(n, T, N)),
                 lambda: conv(x[:, :3], st, state=st), lambda: seq.causal_conv(rnd(g, 1, 4, D), wide[0, 0, :D * W].view(D, W), out=wide[0, 0, :D * W].view(1, W, D)),
                 lambda: seq.causal_conv_step(rows, w, None, buf.view(-1, 3, D)[:8], out=buf.view(-1, 3, D)[1:6, 0]),
                 lambda: seq.selective_scan_step(rows, rows, A, m[0, :5], m[0, :5], big.view(8, D, N), out=big[7:7 + 5 * D].view(5, D)),
                 lambda: seq.unpack8(seq.Packed8(one.view(torch.int8).view(-1)[4:4 + 40 * D].view(40, D), torch.zeros(40, 1, dtype=torch.uint8, device=DEV), torch.float32),
                                     out=one.view(-1)[:40 * D].view(40, D))):
        with pytest.raises(L.CrnnError, match="share"):
            call()
    with pytest.raises(ValueError):
        seq.causal_conv(x, w, out=x)
    was = buf.clone()       # (a state that is not contiguous is copied before the call)
    assert torch.equal(conv(buf[:, 4:7], buf[:, :3], state=buf[:, 1:4]), seq.causal_conv(was[:, 4:7], w, state=was[:, 1:4]))
    # beside each other: halves of a row, a sequence's first and last rows, time and batch swapped, another part of the states' array
    both = rnd(g, n, T, 2 * D)
    swap = rnd(g, T, n, 2 * D).transpose(0, 1)
    rest = rnd(g, n, 2 * T, D)
    for a, b in ((both[..., :D], both[..., D:]), (both[..., D:], both[..., :D]), (swap[..., :D], swap[..., D:]), (rest[:, :T], rest[:, T:]), (rest[:, T:], rest[:, :T]), (rest[:1, :T], rest[2:, :T])):
        k = a.shape[0]
        want, src = seq.causal_conv(a.clone(), w), a.clone()
        assert torch.equal(conv(a, b), want) and torch.equal(a, src)
        want = seq.selective_scan(a.clone(), a.clone(), A, m[:k], m[:k])
        assert torch.equal(scan(a, a, b, m[:k], m[:k]), want) and torch.equal(a, src)
    y = seq.selective_scan_step(rows, rows, A, m[0, :5], m[0, :5], h.clone())
    room = torch.zeros(8 * D * N + 5 * D, device=DEV)
    room[:8 * D * N] = h.view(-1)
    assert torch.equal(seq.selective_scan_step(rows, rows, A, m[0, :5], m[0, :5], room[:8 * D * N].view(8, D, N), out=room[8 * D * N:].view(5, D)), y)


def test_c_entry_points_refuse_arrays_that_share_memory():
    """Pointers of the C ABI that meet: outputs with inputs and with one another; a state that is updated in place is allowed where every element is read by the thread that writes it."""
    import ctypes as C
    lib = L.lib
    KB = 1 << 10

    def view(at, rs=8, ss=48, dt=L.DT_F32, scales=None):
        return L.View(ptr=at * KB, row_stride=rs, seq_stride=ss, dtype=dt, scales=scales, scale_row_stride=1, scale_seq_stride=6)

    def scan(**over):       # each array in a KB of its own: 2 sequences of 6 rows, 8 channels, 4 states
        a = L.ScanArgs(struct_size=C.sizeof(L.ScanArgs), device=99, n_seq=2, D=8, N=4, G=1, rows=6, A=KB, u=view(2), dt=view(3), y=view(4), B=view(5, 4, 24), C=view(6, 4, 24), z=view(7), skip=8 * KB,
                       dt_bias=9 * KB, state_in=10 * KB, state_out=11 * KB, dy=view(12), du=view(13), ddt=view(14), dz=view(15), dB=view(16, 4, 24), dC=view(17, 4, 24), dA=18 * KB,
                       dskip=19 * KB, ddt_bias=20 * KB, dstate_out=21 * KB, dstate_in=22 * KB, seq_len=23 * KB, workspace=1 << 30, workspace_bytes=1 << 40)
        for k, v in over.items():
            setattr(a, k, v)
        return a

    def conv(**over):
        a = L.ConvArgs(struct_size=C.sizeof(L.ConvArgs), device=99, n_seq=2, D=8, W=4, rows=6, weight=KB, bias=2 * KB, x=view(3), y=view(4), state_in=view(5, 8, 24), state_out=view(6, 8, 24), dy=view(7),
                       dx=view(8), dstate_out=view(9, 8, 24), dstate_in=view(10, 8, 24), dweight=11 * KB, dbias=12 * KB, seq_len=13 * KB, workspace=1 << 30, workspace_bytes=1 << 40)
        for k, v in over.items():
            setattr(a, k, v)
        return a

    def at(k, off, **kw):
        v = view(k, **kw)
        v.ptr = k * KB + off
        return v

    IN, OUT = "shares memory with an input", "two outputs"
    packed = view(2, dt=L.DT_PACKED8, scales=30 * KB)
    for call, make, over, word in [
            (lib.crnn_scan_forward, scan, {}, "device"), (lib.crnn_scan_backward, scan, {}, "device"), (lib.crnn_conv_forward, conv, {}, "device"), (lib.crnn_conv_backward, conv, {}, "device"),
            (lib.crnn_scan_forward, scan, dict(y=at(2, 4)), IN), (lib.crnn_scan_forward, scan, dict(y=at(2, -4)), IN), (lib.crnn_scan_forward, scan, dict(y=at(1, 32)), IN),
            (lib.crnn_scan_forward, scan, dict(y=at(10, 252)), IN), (lib.crnn_scan_forward, scan, dict(y=at(10, 256)), "device"), (lib.crnn_scan_forward, scan, dict(y=at(23, 4)), IN),
            (lib.crnn_scan_forward, scan, dict(state_out=10 * KB), "device"), (lib.crnn_scan_forward, scan, dict(state_out=10 * KB + 4), IN), (lib.crnn_scan_forward, scan, dict(state_out=4 * KB + 4), OUT),
            (lib.crnn_scan_forward, scan, dict(u=packed, y=at(30, -4)), IN), (lib.crnn_scan_forward, scan, dict(u=packed, y=at(30, -384)), "device"),
            (lib.crnn_scan_backward, scan, dict(du=at(12, 8)), IN), (lib.crnn_scan_backward, scan, dict(ddt=at(13, 8)), OUT), (lib.crnn_scan_backward, scan, dict(dA=KB), IN),
            (lib.crnn_scan_backward, scan, dict(dstate_in=21 * KB), "device"), (lib.crnn_scan_backward, scan, dict(dstate_in=21 * KB + 8), IN), (lib.crnn_scan_backward, scan, dict(dskip=19 * KB, ddt_bias=19 * KB), OUT),
            (lib.crnn_conv_forward, conv, dict(y=at(5, 64)), IN), (lib.crnn_conv_forward, conv, dict(y=at(2, 16)), IN), (lib.crnn_conv_forward, conv, dict(state_out=at(5, 32, ss=24)), IN),
            (lib.crnn_conv_backward, conv, dict(dstate_in=view(9, 8, 24)), IN), (lib.crnn_conv_backward, conv, dict(dweight=KB), IN), (lib.crnn_conv_backward, conv, dict(dx=at(3, 4)), IN)]:
        assert call(C.byref(make(**over))) == -1 and word in lib.crnn_last_error(None).decode(), (over, lib.crnn_last_error(None).decode())
    v = view(2)
    for codes, scales, word in ((2 * KB + 8, 8 * KB, IN), (8 * KB, 2 * KB + 380, IN), (8 * KB, 8 * KB + 95, OUT), (8 * KB, 8 * KB + 96, "device")):
        assert lib.crnn_pack8(99, None, C.byref(v), 12, 8, codes, scales) == -1 and word in lib.crnn_last_error(None).decode(), (codes, scales)
