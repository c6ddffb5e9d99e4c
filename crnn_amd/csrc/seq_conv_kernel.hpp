// crnn_amd/csrc/seq_conv_kernel.hpp -- gfx950: the short causal convolution over time, its gradient and its single step.
//
//     p[t, d] = bias[d] + sum_j w[d, j] x[t - W + 1 + j, d],   y = p or p sigmoid(p)
//
// x before a sequence's first row is its state (the last W - 1 rows before it), or 0.  Depthwise: a few multiply-adds per element read,
// bound by memory.  A thread owns V neighbouring channels (four, two in double; one where rows are not so aligned) and walks down a strip of rows,
// kConvTB at a time: the next ones are on their way while these are worked on, the last W rows stay in registers, so that each row is read
// once but for the W - 1 rows in front of a strip.  Rows behind the last one are read as the last, threads behind the last channels do the
// last channels once more: loads and stores stand without branches between them, and no wait reaches over a store.
#pragma once
#include "seq_common.hpp"

namespace crnn {

constexpr int kConvTB = 4;       // rows on their way together

struct ConvP {
    SeqMap m;
    SeqV x, y, dy, dx;
    SeqV st_in, st_out, dst_out, dst_in;     // [n_seq][W - 1][D]; bs: between sequences, rs: between rows
    const void *w, *bias;                    // [D][W], [D] in the compute type
    void *part;                              // gradient: [block][W + 1][D]
    int32_t D, W, silu, zero_outside;
};

template <int DT> struct SeqT { using C = float; };
template <> struct SeqT<CRNN_DT_F64> { using C = double; };

// V channels of a row as they stand in memory
template <int DT, int V>
struct ConvRaw {
    using C = typename SeqT<DT>::C;
    static constexpr int ES = DT == CRNN_DT_F64 ? 8 : DT == CRNN_DT_F32 ? 4 : DT == CRNN_DT_PACKED8 ? 1 : 2;
    static constexpr int NW = V * ES >= 4 ? V * ES / 4 : 1;
    uint32_t w[NW];
    uint32_t e;              // checkpoint: the scale byte (V divides 32)
    // row: the row's first channel (uniform), sc: its first scale
    __device__ __forceinline__ void load(const void *row, const uint8_t *sc, uint32_t d) {
        const char *q = (const char *)row + d * ES;
        if (V * ES == 16) {
            typedef uint32_t U4 __attribute__((ext_vector_type(4)));
            const U4 b = *(const U4 *)q;
#pragma unroll
            for (int i = 0; i < NW; ++i) w[i] = b[i & 3];
        } else if (V * ES == 8) {
            typedef uint32_t U2 __attribute__((ext_vector_type(2)));
            const U2 b = *(const U2 *)q;
#pragma unroll
            for (int i = 0; i < NW; ++i) w[i] = b[i & 1];
        } else if (V * ES == 4) w[0] = *(const uint32_t *)q;
        else if (V * ES == 2) w[0] = *(const uint16_t *)q;
        else w[0] = *(const uint8_t *)q;
        if (DT == CRNN_DT_PACKED8) e = sc[d >> 5];
    }
    __device__ __forceinline__ C get(int i) const {
        if (DT == CRNN_DT_F64) {
            const uint64_t b = (uint64_t)w[(2 * i) % NW] | (uint64_t)w[(2 * i + 1) % NW] << 32;
            return (C)__builtin_bit_cast(double, b);
        }
        if (DT == CRNN_DT_F32) return (C)seq_as_float(w[i % NW]);
        if (DT == CRNN_DT_BF16) return (C)seq_as_float(i & 1 ? w[(i / 2) % NW] & 0xffff0000u : w[(i / 2) % NW] << 16);
        if (DT == CRNN_DT_F16) return (C)seq_from_f16(w[(i / 2) % NW] >> (16 * (i & 1)) & 0xffffu);
        return (C)seq_unpack((int8_t)(w[(i / 4) % NW] >> (8 * (i & 3))), e << 23);
    }
};
template <int DT, int V>
__device__ __forceinline__ void conv_put(void *row, uint32_t d, const typename SeqT<DT>::C (&x)[V]) {
    using R = ConvRaw<DT, V>;
    R r;
#pragma unroll
    for (int i = 0; i < R::NW; ++i) r.w[i] = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (DT == CRNN_DT_F64) {
            const uint64_t b = __builtin_bit_cast(uint64_t, (double)x[i]);
            r.w[(2 * i) % R::NW] = (uint32_t)b;
            r.w[(2 * i + 1) % R::NW] = (uint32_t)(b >> 32);
        } else if (DT == CRNN_DT_F32) r.w[i % R::NW] = seq_as_bits((float)x[i]);
        else r.w[(i / 2) % R::NW] |= (uint32_t)(DT == CRNN_DT_BF16 ? seq_to_bf16((float)x[i]) : seq_to_f16((float)x[i])) << (16 * (i & 1));
    }
    char *q = (char *)row + d * R::ES;
    if (V * R::ES == 16) {
        typedef uint32_t U4 __attribute__((ext_vector_type(4)));
        U4 b;
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = r.w[i % R::NW];
        *(U4 *)q = b;
    } else if (V * R::ES == 8) {
        typedef uint32_t U2 __attribute__((ext_vector_type(2)));
        U2 b;
#pragma unroll
        for (int i = 0; i < 2; ++i) b[i] = r.w[i % R::NW];
        *(U2 *)q = b;
    } else if (V * R::ES == 4) *(uint32_t *)q = r.w[0];
    else *(uint16_t *)q = (uint16_t)r.w[0];
}

// Weights of a thread's channels (tap W - 1 is the row itself).  The V W weights of a thread stand together: read V at a time (one at a time,
// 4 W bytes between the lanes, they took as long as 32 rows).  The kernels are built for each W: a tap that a call does not have is not there, for as
// a weight of 0 it would carry an infinity or a NaN to rows that the call's taps do not reach.
template <class CT, int W, int V>
__device__ __forceinline__ void conv_weights(const void *pw, const void *pb, int d, CT (&w)[W][V], CT (&bias)[V]) {
    typedef CT VV __attribute__((ext_vector_type(V)));
    const CT *q = (const CT *)pw + (int64_t)d * W;
    const VV b = pb ? *(const VV *)((const CT *)pb + d) : VV(CT(0));
    VV f[W];
#pragma unroll
    for (int k = 0; k < W; ++k) f[k] = ((const VV *)q)[k];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = b[i];
#pragma unroll
        for (int j = 0; j < W; ++j) w[j][i] = f[(i * W + j) / V][(i * W + j) % V];
    }
}

template <int DT>
__device__ __forceinline__ char *conv_row(const SeqMap &m, const SeqV &v, const SeqChunk &k, int64_t t) {
    return (char *)v.p + seq_off(m, v, k, t) * ConvRaw<DT, 1>::ES;
}
template <int DT>
__device__ __forceinline__ const uint8_t *conv_scales(const SeqMap &m, const SeqV &v, const SeqChunk &k, int64_t t) {
    return DT == CRNN_DT_PACKED8 ? v.sc + seq_soff(m, v, k, t) : nullptr;
}
// x of any row of a sequence (negative: the state's, or 0)
template <int XT, int YT, int W, int V>
__device__ __forceinline__ void conv_x(const ConvP &p, const SeqChunk &k, int64_t t, int d, typename SeqT<YT>::C (&o)[V]) {
    using CT = typename SeqT<YT>::C;
    if (t >= 0) {
        ConvRaw<XT, V> r;
        r.load(conv_row<XT>(p.m, p.x, k, t), conv_scales<XT>(p.m, p.x, k, t), d);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = (CT)r.get(i);
    } else if (p.st_in.p && t >= -(W - 1)) {
        ConvRaw<YT, V> r;
        r.load((const char *)p.st_in.p + ((int64_t)k.s * p.st_in.bs + (t + W - 1) * p.st_in.rs) * ConvRaw<YT, 1>::ES, nullptr, d);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = (CT)r.get(i);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = CT(0);
    }
}

// the place of a thread: 64 threads along the channels, a strip for each of the block's four wavefronts
struct ConvAt { SeqChunk k; int64_t b; int d; bool on; };
template <int V>
__device__ __forceinline__ ConvAt conv_at(const ConvP &p) {
    ConvAt a;
    const uint32_t gx = (uint32_t)(p.D + 64 * V - 1) / (64 * V), by = blockIdx.x / gx;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    a.b = (int64_t)by * 4 + wave;
    const int d = (int)(blockIdx.x - by * gx) * 64 * V + (int)(threadIdx.x & 63) * V;
    a.d = d + V <= p.D ? d : p.D - V;
    a.on = a.b < p.m.nblk;
    a.k = seq_locate(p.m, a.on ? a.b : p.m.nblk - 1);
    return a;
}

// 12001 rows of 4096 channels, bf16, 4 taps: 197 MB in 46 us where nothing is in a cache (4.2 TB/s; a copy reaches 4.7), 38 us again and again on the
// same arrays; 60000 rows 193 us (5.1 TB/s).  130 rows of 768: 6.5 us, a thread's chain of dependent loads.
template <int XT, int YT, int W, int V>
__global__ __launch_bounds__(256) void seq_conv_fwd_kernel(const ConvP p) {
    using CT = typename SeqT<YT>::C;
    constexpr int TB = kConvTB;
    const ConvAt a = conv_at<V>(p);
    if (!a.on) return;
    if (p.zero_outside)
        for (int i = 0; i < V; ++i) seq_zero_outside(p.m, p.y, a.b, a.d + i, true);
    if (!a.k.live) return;
    if (a.k.n > 0) {
        CT w[W][V], bias[V], x[W - 1 + TB][V];
        conv_weights<CT, W, V>(p.w, p.bias, a.d, w, bias);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) conv_x<XT, YT, W, V>(p, a.k, a.k.t0 - (W - 1) + j, a.d, x[j]);
        const char *xrow = conv_row<XT>(p.m, p.x, a.k, a.k.t0);
        const uint8_t *srow = conv_scales<XT>(p.m, p.x, a.k, a.k.t0);
        char *yrow = conv_row<YT>(p.m, p.y, a.k, a.k.t0);
        const int64_t xs = (int64_t)p.x.rs * ConvRaw<XT, V>::ES, ss = p.x.srs, ys = (int64_t)p.y.rs * ConvRaw<YT, V>::ES;
        ConvRaw<XT, V> raw[TB];
#pragma unroll
        for (int i = 0; i < TB; ++i) {
            const int64_t r = i < a.k.n ? i : a.k.n - 1;
            raw[i].load(xrow + r * xs, srow + r * ss, a.d);
        }
#pragma unroll 1
        for (int t = 0; t < a.k.n; t += TB) {
#pragma unroll
            for (int i = 0; i < TB; ++i)
#pragma unroll
                for (int c = 0; c < V; ++c) x[W - 1 + i][c] = (CT)raw[i].get(c);
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const int64_t r = t + TB + i < a.k.n ? t + TB + i : a.k.n - 1;
                raw[i].load(xrow + r * xs, srow + r * ss, a.d);
            }
            __builtin_amdgcn_sched_barrier(0);       // (the loads are issued here, not where the compiler would like them)
            CT y[TB][V];
#pragma unroll
            for (int i = 0; i < TB; ++i)
#pragma unroll
                for (int c = 0; c < V; ++c) {
                    CT s = bias[c];
#pragma unroll
                    for (int j = 0; j < W; ++j) s = seq_fma(w[j][c], x[i + j][c], s);
                    y[i][c] = s;
                }
            if (p.silu) {
#pragma unroll
                for (int i = 0; i < TB; ++i)
#pragma unroll
                    for (int c = 0; c < V; ++c) y[i][c] *= seq_sigmoid(y[i][c]);
            }
            if (t + TB > a.k.n) {
#pragma unroll
                for (int i = 1; i < TB; ++i)
#pragma unroll
                    for (int c = 0; c < V; ++c) y[i][c] = t + i < a.k.n ? y[i][c] : y[i - 1][c];
            }
#pragma unroll
            for (int i = 0; i < TB; ++i) conv_put<YT, V>(yrow + (int64_t)(t + i < a.k.n ? t + i : a.k.n - 1) * ys, a.d, y[i]);
#pragma unroll
            for (int j = 0; j < W - 1; ++j)
#pragma unroll
                for (int c = 0; c < V; ++c) x[j][c] = x[j + TB][c];
        }
    }
    if (a.k.last && p.st_out.p)        // rows len - (W - 1) .. len - 1 of (state, x)
        for (int j = 0; j < W - 1; ++j) {
            CT v[V];
            conv_x<XT, YT, W, V>(p, a.k, a.k.len - (W - 1) + j, a.d, v);
            conv_put<YT, V>((char *)p.st_out.p + ((int64_t)a.k.s * p.st_out.bs + j * (int64_t)p.st_out.rs) * ConvRaw<YT, V>::ES, a.d, v);
        }
}

// Gradient.  dp = dy act'(p) needs p once more; dx[t] = sum_j w[j] dp[t + W - 1 - j] needs the W - 1 rows behind t: the strip is walked W - 1
// rows past its end.  A sequence's first strip starts W - 1 rows early: those are the state's.  dw, db: a strip's part, summed in order.
// 8192 rows of 2048 channels, x in 8 bits, bf16, 4 taps: 33 us (84 MB, 2.5 TB/s) and 6.3 us for the sums.  Neither memory nor the vector unit (half
// busy) binds it: at 128 registers four wavefronts a SIMD wait for loads one batch of rows ahead; longer strips leave SIMDs without a wavefront.
template <int XT, int YT, int W, int V>
__global__ __launch_bounds__(256, W <= 4 && (YT == CRNN_DT_BF16 || YT == CRNN_DT_F16) ? 4 : 1) void seq_conv_bwd_kernel(const ConvP p) {
    using CT = typename SeqT<YT>::C;
    constexpr int TB = kConvTB;
    const ConvAt a = conv_at<V>(p);
    if (!a.on) return;
    if (p.zero_outside)
        for (int i = 0; i < V; ++i) seq_zero_outside(p.m, p.dx, a.b, a.d + i, true);
    CT dw[W][V], db[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
        db[c] = CT(0);
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][c] = CT(0);
    }
    if (a.k.live) {
        // x[W - 1 + i], dp[W - 1 + i]: the batch's row i
        CT w[W][V], bias[V], x[W - 1 + TB][V], dp[W - 1 + TB][V];
        conv_weights<CT, W, V>(p.w, p.bias, a.d, w, bias);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            conv_x<XT, YT, W, V>(p, a.k, a.k.t0 - (W - 1) + j, a.d, x[j]);
#pragma unroll
            for (int c = 0; c < V; ++c) dp[j][c] = CT(0);
        }
        constexpr int back = W - 1;
        // (fewer than 2^31 rows: uniform comparisons of 32 bits stay out of the vector unit)
        const int t0 = (int)a.k.t0, len = (int)a.k.len, lo = t0 == 0 ? -back : t0, hi = t0 + a.k.n;     // rows whose dx this strip writes
        const int lastrow = len - 1;
        const char *xrow = conv_row<XT>(p.m, p.x, a.k, 0), *grow = conv_row<YT>(p.m, p.dy, a.k, 0);
        const uint8_t *srow = conv_scales<XT>(p.m, p.x, a.k, 0);
        char *orow = conv_row<YT>(p.m, p.dx, a.k, 0);
        const int64_t xs = (int64_t)p.x.rs * ConvRaw<XT, V>::ES, ss = p.x.srs, gs = (int64_t)p.dy.rs * ConvRaw<YT, V>::ES, os = (int64_t)p.dx.rs * ConvRaw<YT, V>::ES;
        ConvRaw<XT, V> rx[TB];
        ConvRaw<YT, V> rg[TB];
        auto fetch = [&](int t) {
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const int64_t r = t + i < lastrow ? t + i : lastrow;
                rx[i].load(xrow + r * xs, srow + r * ss, a.d);
                rg[i].load(grow + r * gs, nullptr, a.d);
            }
        };
        if (a.k.n > 0) fetch(t0);
#pragma unroll 1
        for (int t = t0; t < hi + W - 1; t += TB) {
            if (a.k.n > 0) {
#pragma unroll
                for (int i = 0; i < TB; ++i)
#pragma unroll
                    for (int c = 0; c < V; ++c) {
                        x[W - 1 + i][c] = (CT)rx[i].get(c);
                        dp[W - 1 + i][c] = (CT)rg[i].get(c);
                    }
                fetch(t + TB);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < TB; ++i) {
                    const bool in = t + i <= lastrow;
#pragma unroll
                    for (int c = 0; c < V; ++c) {
                        CT s = bias[c];
#pragma unroll
                        for (int j = 0; j < W; ++j) s = seq_fma(w[j][c], x[i + j][c], s);
                        const CT sg = seq_sigmoid(s);
                        CT g = dp[W - 1 + i][c];
                        const CT ga = g * (sg * seq_fma(s, CT(1) - sg, CT(1)));
                        g = p.silu ? ga : g;
                        dp[W - 1 + i][c] = in ? g : CT(0);
                    }
                    if (t + i < hi) {       // the strip's own rows only: one behind them would add 0 times its x, which an infinity makes NaN
#pragma unroll
                        for (int c = 0; c < V; ++c) {
                            db[c] += dp[W - 1 + i][c];
#pragma unroll
                            for (int j = 0; j < W; ++j) dw[j][c] = seq_fma(dp[W - 1 + i][c], x[i + j][c], dw[j][c]);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < TB; ++i)
#pragma unroll
                    for (int c = 0; c < V; ++c) dp[W - 1 + i][c] = CT(0);
            }
            // row t - (W - 1) + i has all its uses now: tap W - 1 - j met it in output row t - (W - 1) + i + j
            CT o[TB][V];
#pragma unroll
            for (int i = 0; i < TB; ++i)
#pragma unroll
                for (int c = 0; c < V; ++c) {
                    CT s = CT(0);
#pragma unroll
                    for (int j = 0; j < W; ++j) s = seq_fma(w[W - 1 - j][c], dp[i + j][c], s);
                    o[i][c] = s;
                }
            const int r0 = t - (W - 1);
            if (r0 >= (lo > 0 ? lo : 0) && r0 + TB <= hi && !(p.dst_out.p && r0 + TB > len - back)) {
#pragma unroll
                for (int i = 0; i < TB; ++i) conv_put<YT, V>(orow + (int64_t)(r0 + i) * os, a.d, o[i]);
            } else {
#pragma unroll
                for (int i = 0; i < TB; ++i) {
                    const int r = r0 + i;
                    if (r < lo || r >= hi) continue;
                    if (p.dst_out.p && r >= len - back) {
                        ConvRaw<YT, V> d;
                        d.load((const char *)p.dst_out.p + ((int64_t)a.k.s * p.dst_out.bs + (int64_t)(r - (len - back)) * p.dst_out.rs) * ConvRaw<YT, V>::ES, nullptr, a.d);
#pragma unroll
                        for (int c = 0; c < V; ++c) o[i][c] += (CT)d.get(c);
                    }
                    if (r >= 0) conv_put<YT, V>(orow + (int64_t)r * os, a.d, o[i]);
                    else if (p.dst_in.p) conv_put<YT, V>((char *)p.dst_in.p + ((int64_t)a.k.s * p.dst_in.bs + (int64_t)(r + back) * p.dst_in.rs) * ConvRaw<YT, V>::ES, a.d, o[i]);
                }
            }
#pragma unroll
            for (int j = 0; j < W - 1; ++j)
#pragma unroll
                for (int c = 0; c < V; ++c) {
                    x[j][c] = x[j + TB][c];
                    dp[j][c] = dp[j + TB][c];
                }
        }
    }
    CT *part = (CT *)p.part + a.b * (W + 1) * p.D + a.d;
#pragma unroll
    for (int c = 0; c < V; ++c) {
#pragma unroll
        for (int j = 0; j < W; ++j) part[(int64_t)j * p.D + c] = dw[j][c];
        part[(int64_t)W * p.D + c] = db[c];
    }
}

// one row for each of many running sequences; the states (the last W - 1 rows) move up in place.  Rows that name one slot: seq_same_slot.
// 192 rows of 4096 channels, bf16, 4 taps: 5.6 us (12.7 MB: 2.7 us of a copy's rate), a chain of slot, state and weights, then the stores.
struct ConvStepP {
    SeqV x, y, st;                   // st.bs: between slots
    const void *w, *bias;
    const int32_t *slot;
    int64_t rows, n_slots;
    int32_t D, W, silu;
};
template <int YT, int W, int V>
__global__ __launch_bounds__(256) void seq_conv_step_kernel(const ConvStepP p) {
    using CT = typename SeqT<YT>::C;
    constexpr int ES = ConvRaw<YT, V>::ES;
    __shared__ int before, next;
    const uint32_t gx = (uint32_t)(p.D + 256 * V - 1) / (256 * V), r0 = blockIdx.x / gx;
    int64_t r = r0;
    const int d0 = (int)(blockIdx.x - r0 * gx) * 256 * V + (int)threadIdx.x * V;
    const bool on = d0 < p.D;        // (D is a multiple of V)
    const int d = on ? d0 : 0;
    const int64_t slot = p.slot ? p.slot[r] : r;
    const bool there = slot >= 0 && slot < p.n_slots;
    char *yp = (char *)p.y.p;
    if (!there) {
        CT y[V];
#pragma unroll
        for (int c = 0; c < V; ++c) y[c] = CT(0);
        if (on) conv_put<YT, V>(yp + r * (int64_t)p.y.rs * ES, d, y);
        return;
    }
    // all that the row reads is on its way before other rows' slots are looked at
    CT w[W][V], bias[V], x[W][V];
    char *st = (char *)p.st.p + slot * p.st.bs * ES;
    ConvRaw<YT, V> q, qs[W > 1 ? W - 1 : 1];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) qs[j].load(st + j * (int64_t)p.st.rs * ES, nullptr, d);
    q.load((const char *)p.x.p + r * (int64_t)p.x.rs * ES, nullptr, d);
    conv_weights<CT, W, V>(p.w, p.bias, d, w, bias);
    int64_t nx = -1;
    if (p.slot && p.rows > 1) {
        if (threadIdx.x == 0) { before = 0; next = 0x7fffffff; }
        __syncthreads();
        seq_same_slot(p.slot, p.rows, r, &before, &next);
        __syncthreads();
        if (before) return;
        nx = next == 0x7fffffff ? -1 : next;
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
        for (int c = 0; c < V; ++c) x[j][c] = qs[j].get(c);
    for (;;) {
        CT y[V];
#pragma unroll
        for (int c = 0; c < V; ++c) {
            x[W - 1][c] = q.get(c);
            CT s = bias[c];
#pragma unroll
            for (int j = 0; j < W; ++j) s = seq_fma(w[j][c], x[j][c], s);
            const CT g = s * seq_sigmoid(s);
            y[c] = p.silu ? g : s;
#pragma unroll
            for (int j = 0; j < W - 1; ++j) x[j][c] = x[j + 1][c];
        }
        if (on) conv_put<YT, V>(yp + r * (int64_t)p.y.rs * ES, d, y);
        if (nx < 0) break;
        r = nx;
        q.load((const char *)p.x.p + r * (int64_t)p.x.rs * ES, nullptr, d);
        __syncthreads();
        if (threadIdx.x == 0) next = 0x7fffffff;
        __syncthreads();
        seq_same_slot(p.slot, p.rows, r, &before, &next);
        __syncthreads();
        nx = next == 0x7fffffff ? -1 : next;
    }
    if (!on) return;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) conv_put<YT, V>(st + j * (int64_t)p.st.rs * ES, d, x[j]);
}

}  // namespace crnn
