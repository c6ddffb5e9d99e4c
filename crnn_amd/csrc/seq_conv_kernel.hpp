// crnn_amd/csrc/seq_conv_kernel.hpp -- gfx950: the short causal convolution over time, its gradient and its single step.
//
//     p[t, d] = bias[d] + sum_j w[d, j] x[t - W + 1 + j, d],   y = p or p sigmoid(p)
//
// x before a sequence's first row is its state (the last W - 1 rows before it), or 0.  Depthwise: a few multiply-adds per element read,
// bound by memory.  A thread owns kConvV neighbouring channels and walks down a strip of rows with the last W rows in registers, so that
// each row is read once but for the W - 1 rows in front of a strip.
#pragma once
#include "seq_common.hpp"

namespace crnn {

constexpr int kConvV = 4;        // channels of a thread
constexpr int kConvMaxW = 8;

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

template <int DT>
__device__ __forceinline__ void conv_load(const SeqV &v, int64_t off, int64_t soff, int d, int D, typename SeqT<DT>::C (&o)[kConvV]) {
    using CT = typename SeqT<DT>::C;
    if (DT == CRNN_DT_PACKED8) {
        const int8_t *q = (const int8_t *)v.p + off;
        if (v.vec && d + kConvV <= D) {
            const uint32_t b = *(const uint32_t *)q;       // four codes; kConvV divides 32: one scale
            const CT e = (CT)seq_scale(v.sc[soff + (d >> 5)]);
#pragma unroll
            for (int i = 0; i < kConvV; ++i) o[i] = (CT)(int32_t)(int8_t)(b >> (8 * i)) * e;
        } else {
#pragma unroll
            for (int i = 0; i < kConvV; ++i) o[i] = d + i < D ? (CT)(int32_t)q[i] * (CT)seq_scale(v.sc[soff + ((d + i) >> 5)]) : CT(0);
        }
    } else if (DT == CRNN_DT_F32 || DT == CRNN_DT_F64) {
        const CT *q = (const CT *)v.p + off;
        constexpr int L = 16 / (int)sizeof(CT);
        typedef CT V __attribute__((ext_vector_type(L)));
        if (v.vec && d + kConvV <= D) {
#pragma unroll
            for (int k = 0; k < kConvV / L; ++k) {
                const V b = *(const V *)(q + k * L);
#pragma unroll
                for (int i = 0; i < L; ++i) o[k * L + i] = b[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < kConvV; ++i) o[i] = d + i < D ? q[i] : CT(0);
        }
    } else {
        const uint16_t *q = (const uint16_t *)v.p + off;
        uint32_t b[kConvV];
        if (v.vec && d + kConvV <= D) {
            const uint64_t w = *(const uint64_t *)q;
#pragma unroll
            for (int i = 0; i < kConvV; ++i) b[i] = (uint32_t)(w >> (16 * i)) & 0xffffu;
        } else {
#pragma unroll
            for (int i = 0; i < kConvV; ++i) b[i] = d + i < D ? q[i] : 0u;
        }
#pragma unroll
        for (int i = 0; i < kConvV; ++i) o[i] = (CT)(DT == CRNN_DT_BF16 ? seq_as_float(b[i] << 16) : seq_from_f16(b[i]));
    }
}
template <int DT>
__device__ __forceinline__ void conv_store(const SeqV &v, int64_t off, int d, int D, const typename SeqT<DT>::C (&o)[kConvV]) {
    using CT = typename SeqT<DT>::C;
    if (DT == CRNN_DT_F32 || DT == CRNN_DT_F64) {
        CT *q = (CT *)v.p + off;
        constexpr int L = 16 / (int)sizeof(CT);
        typedef CT V __attribute__((ext_vector_type(L)));
        if (v.vec && d + kConvV <= D) {
#pragma unroll
            for (int k = 0; k < kConvV / L; ++k) {
                V b;
#pragma unroll
                for (int i = 0; i < L; ++i) b[i] = o[k * L + i];
                *(V *)(q + k * L) = b;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kConvV; ++i)
                if (d + i < D) q[i] = o[i];
        }
    } else {
        uint16_t *q = (uint16_t *)v.p + off;
        uint16_t b[kConvV];
#pragma unroll
        for (int i = 0; i < kConvV; ++i) b[i] = DT == CRNN_DT_BF16 ? seq_to_bf16((float)o[i]) : seq_to_f16((float)o[i]);
        if (v.vec && d + kConvV <= D) {
            *(uint64_t *)q = (uint64_t)b[0] | (uint64_t)b[1] << 16 | (uint64_t)b[2] << 32 | (uint64_t)b[3] << 48;
        } else {
#pragma unroll
            for (int i = 0; i < kConvV; ++i)
                if (d + i < D) q[i] = b[i];
        }
    }
}

// weights of a thread's channels, right-aligned in WM taps (tap WM - 1 is the row itself)
template <class CT, int WM>
__device__ __forceinline__ void conv_weights(const ConvP &p, int d, CT (&w)[WM][kConvV], CT (&bias)[kConvV]) {
#pragma unroll
    for (int i = 0; i < kConvV; ++i) {
        const int di = d + i < p.D ? d + i : p.D - 1;
        bias[i] = p.bias ? ((const CT *)p.bias)[di] : CT(0);
#pragma unroll
        for (int j = 0; j < WM; ++j) {
            const int k = j - (WM - p.W);
            w[j][i] = k >= 0 ? ((const CT *)p.w)[(int64_t)di * p.W + k] : CT(0);
        }
    }
}

// x of row t (negative: the state's)
template <int XT, int YT>
__device__ __forceinline__ void conv_x(const ConvP &p, const SeqChunk &k, int64_t t, int d, typename SeqT<YT>::C (&o)[kConvV]) {
    using CT = typename SeqT<YT>::C;
    if (t >= 0) {
        typename SeqT<XT>::C v[kConvV];
        conv_load<XT>(p.x, seq_off(p.m, p.x, k, t) + d, seq_soff(p.m, p.x, k, t), d, p.D, v);
#pragma unroll
        for (int i = 0; i < kConvV; ++i) o[i] = (CT)v[i];
    } else if (p.st_in.p && t >= -(p.W - 1)) {
        conv_load<YT>(p.st_in, (int64_t)k.s * p.st_in.bs + (t + p.W - 1) * p.st_in.rs + d, 0, d, p.D, o);
    } else {
#pragma unroll
        for (int i = 0; i < kConvV; ++i) o[i] = CT(0);
    }
}

// the place of a thread: blockIdx.x = group of channels + groups x group of blocks; threads (64, 4): 64 threads along the channels, 4 strips
struct ConvAt { SeqChunk k; int64_t b; int d; bool on; };
__device__ __forceinline__ ConvAt conv_at(const ConvP &p) {
    ConvAt a;
    const int64_t gx = (p.D + 64 * kConvV - 1) / (64 * kConvV);
    const int64_t by = (int64_t)blockIdx.x / gx;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    a.b = by * 4 + wave;
    a.d = (int)((int64_t)blockIdx.x - by * gx) * 64 * kConvV + (int)(threadIdx.x & 63) * kConvV;
    a.on = a.b < p.m.nblk;
    a.k = seq_locate(p.m, a.on ? a.b : p.m.nblk - 1);
    return a;
}

// the rows of the state behind a sequence: local rows len - (W - 1) .. len - 1 of (state, x)
template <int XT, int YT>
__device__ __forceinline__ void conv_state_out(const ConvP &p, const SeqChunk &k, int d) {
    for (int j = 0; j < p.W - 1; ++j) {
        typename SeqT<YT>::C v[kConvV];
        conv_x<XT, YT>(p, k, k.len - (p.W - 1) + j, d, v);
        conv_store<YT>(p.st_out, (int64_t)k.s * p.st_out.bs + j * p.st_out.rs + d, d, p.D, v);
    }
}

template <int XT, int YT, int WM>
__global__ __launch_bounds__(256) void seq_conv_fwd_kernel(const ConvP p) {
    using CT = typename SeqT<YT>::C;
    const ConvAt a = conv_at(p);
    if (!a.on || a.d >= p.D) return;
    if (p.zero_outside)
        for (int i = 0; i < kConvV; ++i) seq_zero_outside(p.m, p.y, a.b, a.d + i, a.d + i < p.D);
    if (!a.k.live) return;
    CT w[WM][kConvV], bias[kConvV], x[WM][kConvV];
    conv_weights<CT, WM>(p, a.d, w, bias);
#pragma unroll
    for (int j = 0; j < WM - 1; ++j) conv_x<XT, YT>(p, a.k, a.k.t0 - (WM - 1) + j, a.d, x[j]);
#pragma unroll 4
    for (int t = 0; t < a.k.n; ++t) {
        conv_x<XT, YT>(p, a.k, a.k.t0 + t, a.d, x[WM - 1]);
        CT y[kConvV];
#pragma unroll
        for (int i = 0; i < kConvV; ++i) {
            CT s = bias[i];
#pragma unroll
            for (int j = 0; j < WM; ++j) s = seq_fma(w[j][i], x[j][i], s);
            y[i] = p.silu ? s * seq_sigmoid(s) : s;
#pragma unroll
            for (int j = 0; j < WM - 1; ++j) x[j][i] = x[j + 1][i];
        }
        conv_store<YT>(p.y, seq_off(p.m, p.y, a.k, a.k.t0 + t) + a.d, a.d, p.D, y);
    }
    if (a.k.last && p.st_out.p) conv_state_out<XT, YT>(p, a.k, a.d);
}

// Gradient.  dp = dy act'(p) needs p once more; dx[t] = sum_j w[j] dp[t + W - 1 - j] needs the W - 1 rows behind t: the strip is walked W - 1
// rows past its end.  A sequence's first strip starts W - 1 rows early: those are the state's.  dw, db: a strip's part, summed in order.
template <int XT, int YT, int WM>
__global__ __launch_bounds__(256) void seq_conv_bwd_kernel(const ConvP p) {
    using CT = typename SeqT<YT>::C;
    const ConvAt a = conv_at(p);
    if (!a.on || a.d >= p.D) return;
    if (p.zero_outside)
        for (int i = 0; i < kConvV; ++i) seq_zero_outside(p.m, p.dx, a.b, a.d + i, a.d + i < p.D);
    CT dw[WM][kConvV], db[kConvV];
#pragma unroll
    for (int i = 0; i < kConvV; ++i) {
        db[i] = CT(0);
#pragma unroll
        for (int j = 0; j < WM; ++j) dw[j][i] = CT(0);
    }
    if (a.k.live) {
        CT w[WM][kConvV], bias[kConvV], x[WM][kConvV], dp[WM][kConvV];     // x[WM - 1]: row t; dp[j]: row t - j
        conv_weights<CT, WM>(p, a.d, w, bias);
#pragma unroll
        for (int j = 0; j < WM; ++j)
#pragma unroll
            for (int i = 0; i < kConvV; ++i) dp[j][i] = CT(0);
#pragma unroll
        for (int j = 0; j < WM - 1; ++j) conv_x<XT, YT>(p, a.k, a.k.t0 - (WM - 1) + j, a.d, x[j]);
        const int64_t end = a.k.t0 + a.k.n;
        const int back = p.W - 1;
        const int64_t from = a.k.t0 == 0 ? -(int64_t)back : a.k.t0;     // first row whose dx this strip writes
        for (int64_t t = a.k.t0; t < end + back; ++t) {
            const bool in = t < a.k.len;
            if (in) {
                CT y[kConvV];
                conv_x<XT, YT>(p, a.k, t, a.d, x[WM - 1]);
                conv_load<YT>(p.dy, seq_off(p.m, p.dy, a.k, t) + a.d, 0, a.d, p.D, y);
#pragma unroll
                for (int i = 0; i < kConvV; ++i) {
                    CT s = bias[i];
#pragma unroll
                    for (int j = 0; j < WM; ++j) s = seq_fma(w[j][i], x[j][i], s);
                    CT g = y[i];
                    if (p.silu) {
                        const CT sg = seq_sigmoid(s);
                        g *= sg * seq_fma(s, CT(1) - sg, CT(1));
                    }
                    dp[0][i] = g;
                    if (t < end) {
                        db[i] += g;
#pragma unroll
                        for (int j = 0; j < WM; ++j) dw[j][i] = seq_fma(g, x[j][i], dw[j][i]);
                    }
#pragma unroll
                    for (int j = 0; j < WM - 1; ++j) x[j][i] = x[j + 1][i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < kConvV; ++i) dp[0][i] = CT(0);
            }
            const int64_t row = t - back;                  // all its uses are in dp[0 .. back]
            if (row >= from) {
                CT g[kConvV];
#pragma unroll
                for (int i = 0; i < kConvV; ++i) {
                    g[i] = CT(0);
#pragma unroll
                    for (int j = 0; j < WM; ++j)           // tap j met row `row` in the output row t - (j - (WM - W)): dp[j - (WM - W)]
                        if (j >= WM - p.W) {
                            CT v = CT(0);
#pragma unroll
                            for (int k = 0; k < WM; ++k)
                                if (k == j - (WM - p.W)) v = dp[k][i];
                            g[i] = seq_fma(w[j][i], v, g[i]);
                        }
                }
                if (p.dst_out.p && row >= a.k.len - back) {
                    CT s[kConvV];
                    conv_load<YT>(p.dst_out, (int64_t)a.k.s * p.dst_out.bs + (row - (a.k.len - back)) * p.dst_out.rs + a.d, 0, a.d, p.D, s);
#pragma unroll
                    for (int i = 0; i < kConvV; ++i) g[i] += s[i];
                }
                if (row >= 0) conv_store<YT>(p.dx, seq_off(p.m, p.dx, a.k, row) + a.d, a.d, p.D, g);
                else if (p.dst_in.p) conv_store<YT>(p.dst_in, (int64_t)a.k.s * p.dst_in.bs + (row + back) * p.dst_in.rs + a.d, a.d, p.D, g);
            }
#pragma unroll
            for (int j = WM - 1; j >= 1; --j)
#pragma unroll
                for (int i = 0; i < kConvV; ++i) dp[j][i] = dp[j - 1][i];
        }
    }
    CT *part = (CT *)p.part + a.b * (p.W + 1) * p.D;
#pragma unroll
    for (int i = 0; i < kConvV; ++i) {
        if (a.d + i >= p.D) continue;
#pragma unroll
        for (int j = 0; j < WM; ++j) {
            const int k = j - (WM - p.W);
            if (k >= 0) part[(int64_t)k * p.D + a.d + i] = dw[j][i];
        }
        part[(int64_t)p.W * p.D + a.d + i] = db[i];
    }
}

// one row for each of many running sequences; the states (the last W - 1 rows) move up in place.  Rows that name one slot: seq_scan_step_kernel.
struct ConvStepP {
    SeqV x, y, st;                   // st.bs: between slots
    const void *w, *bias;
    const int32_t *slot;
    int64_t rows, n_slots;
    int32_t D, W, silu;
};
template <int YT, int WM>
__global__ __launch_bounds__(256) void seq_conv_step_kernel(const ConvStepP p) {
    using CT = typename SeqT<YT>::C;
    __shared__ int before, next;
    const int64_t gx = (p.D + 256 * kConvV - 1) / (256 * kConvV);
    int64_t r = (int64_t)blockIdx.x / gx;
    const int d = (int)((int64_t)blockIdx.x - r * gx) * 256 * kConvV + (int)threadIdx.x * kConvV;
    const bool on = d < p.D;
    const int64_t slot = p.slot ? p.slot[r] : r;
    const bool there = slot >= 0 && slot < p.n_slots;
    int64_t nx = -1;
    if (p.slot && there && p.rows > 1) {
        if (threadIdx.x == 0) { before = 0; next = 0x7fffffff; }
        __syncthreads();
        seq_same_slot(p.slot, p.rows, r, &before, &next);
        __syncthreads();
        if (before) return;
        nx = next == 0x7fffffff ? -1 : next;
    }
    CT w[WM][kConvV], bias[kConvV], x[WM][kConvV];
    if (!there) {
#pragma unroll
        for (int i = 0; i < kConvV; ++i) bias[i] = CT(0);
        if (on) conv_store<YT>(p.y, r * (int64_t)p.y.rs + d, d, p.D, bias);
        return;
    }
    ConvP q;
    q.D = p.D; q.W = p.W; q.w = p.w; q.bias = p.bias;
    conv_weights<CT, WM>(q, on ? d : 0, w, bias);
    const int at = on ? d : 0;
#pragma unroll
    for (int j = 0; j < WM - 1; ++j) {
        const int k = j - (WM - p.W);
        if (k >= 0) conv_load<YT>(p.st, slot * p.st.bs + k * p.st.rs + at, 0, at, p.D, x[j]);
        else
#pragma unroll
            for (int i = 0; i < kConvV; ++i) x[j][i] = CT(0);
    }
    for (;;) {
        CT y[kConvV];
        conv_load<YT>(p.x, r * (int64_t)p.x.rs + at, 0, at, p.D, x[WM - 1]);
#pragma unroll
        for (int i = 0; i < kConvV; ++i) {
            CT s = bias[i];
#pragma unroll
            for (int j = 0; j < WM; ++j) s = seq_fma(w[j][i], x[j][i], s);
            y[i] = p.silu ? s * seq_sigmoid(s) : s;
#pragma unroll
            for (int j = 0; j < WM - 1; ++j) x[j][i] = x[j + 1][i];
        }
        if (on) conv_store<YT>(p.y, r * (int64_t)p.y.rs + d, d, p.D, y);
        if (nx < 0) break;
        r = nx;
        __syncthreads();
        if (threadIdx.x == 0) next = 0x7fffffff;
        __syncthreads();
        seq_same_slot(p.slot, p.rows, r, &before, &next);
        __syncthreads();
        nx = next == 0x7fffffff ? -1 : next;
    }
    if (!on) return;
#pragma unroll
    for (int j = 0; j < WM - 1; ++j) {
        const int k = j - (WM - p.W);
        if (k >= 0) conv_store<YT>(p.st, slot * p.st.bs + k * p.st.rs + d, d, p.D, x[j]);
    }
}

}  // namespace crnn
