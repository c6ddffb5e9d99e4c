// crnn_amd/csrc/seq_common.hpp -- gfx950: what the sequence operators share (causal convolution, selective scan, 8-bit checkpoints):
// element types, views of caller-owned arrays, the map from a launch's blocks to pieces of sequences.
//
// Rows are time, channels run fastest in memory.  A view is addressed by sequence and row: a dense batch has a stride between sequences, a
// packed one holds all rows in one array and seq_start[s] .. seq_start[s + 1] - 1 are sequence s.  The offsets live on the device and are
// clamped to the array before use, so that no content of theirs can move an access outside the arrays of the call.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/crnn_hip.h"

namespace crnn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLog2eD = 1.4426950408889634;

__device__ __forceinline__ float seq_as_float(uint32_t b) { return __builtin_bit_cast(float, b); }
__device__ __forceinline__ uint32_t seq_as_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
// round to nearest even; a NaN stays one
__device__ __forceinline__ uint16_t seq_to_bf16(float f) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(uint16_t, (__bf16)f);
#else
    const uint32_t b = seq_as_bits(f);
    if ((b & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((b >> 16) | 0x40u);
    return (uint16_t)((b + 0x7fffu + ((b >> 16) & 1u)) >> 16);
#endif
}
__device__ __forceinline__ uint16_t seq_to_f16(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
__device__ __forceinline__ float seq_from_f16(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (uint16_t)b); }
// 2^(byte - 127), byte 255: NaN (E8M0).  byte 0 is the denormal 2^-127.
__device__ __forceinline__ float seq_scale(uint32_t byte) {
    return seq_as_float(byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23);
}

// code * 2^(byte - 127) with the byte at bit 23: 0 is the largest of it and 2^-127's bits, 255 (infinity here) adds 0 * infinity
__device__ __forceinline__ float seq_unpack(int32_t code, uint32_t byte23) {
    const float s = seq_as_float(byte23 > 0x00400000u ? byte23 : 0x00400000u);
    return __builtin_fmaf((float)code, s, s * 0.0f);
}

// ---- functions in the compute type.  The float forms use the hardware's exp2 and reciprocal (about one unit in the last place).
__device__ __forceinline__ float seq_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ double seq_exp2(double x) { return exp2(x); }
__device__ __forceinline__ float seq_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ double seq_rcp(double x) { return 1.0 / x; }
__device__ __forceinline__ float seq_fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double seq_fma(double a, double b, double c) { return __builtin_fma(a, b, c); }
__device__ __forceinline__ float seq_sigmoid(float x) { return seq_rcp(1.0f + seq_exp2(x * -kLog2e)); }
__device__ __forceinline__ double seq_sigmoid(double x) { return 1.0 / (1.0 + exp(-x)); }
// log(1 + e^x) = max(x, 0) + log1p(e^-|x|).  log1p(e) = 2 artanh(e / (2 + e)): the small values that step lengths usually have keep their
// relative accuracy, which log2(1 + e) would lose.  Polynomial in s^2 on [0, 1/9], off by less than 1e-9 (half a unit is 6e-8).
__device__ __forceinline__ float seq_softplus(float x) {
    const float e = seq_exp2(-__builtin_fabsf(x) * kLog2e);
    const float s = e * seq_rcp(2.0f + e), z = s * s;
    float p = 0.12204702f;
    p = seq_fma(p, z, 0.10697134f);
    p = seq_fma(p, z, 0.14310312f);
    p = seq_fma(p, z, 0.19999347f);
    p = seq_fma(p, z, 0.33333340f);
    p = seq_fma(p, z, 1.0f);
    return seq_fma(2.0f * s, p, x > 0.0f ? x : (x == x ? 0.0f : x));
}
__device__ __forceinline__ double seq_softplus(double x) {
    return (x > 0.0 ? x : (x == x ? 0.0 : x)) + log1p(exp(-fabs(x)));
}

__device__ __forceinline__ float seq_abs(float x) { return __builtin_fabsf(x); }
__device__ __forceinline__ double seq_abs(double x) { return __builtin_fabs(x); }
__device__ __forceinline__ float seq_max(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double seq_max(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ float seq_ldexp(float x, int e) { return __builtin_ldexpf(x, e); }
__device__ __forceinline__ double seq_ldexp(double x, int e) { return __builtin_ldexp(x, e); }
// h 2^x where 2^x alone may be out of the type's range (growth over a whole chunk: 0 stays 0, and a small h may come out in range)
template <class CT>
__device__ __forceinline__ CT seq_grow(CT h, CT x) {
    x = x > CT(10000) ? CT(10000) : x < CT(-10000) ? CT(-10000) : x;      // (behind either type's range; a NaN stays one)
    const CT w = __builtin_elementwise_rint(x);
    return seq_ldexp(h * seq_exp2(x - w), (int)w);
}

// ---- a caller-owned array [sequence][row][channel], channels contiguous
struct SeqV {
    void *p;
    const uint8_t *sc;      // CRNN_DT_PACKED8: one scale byte per 32 channels of a row
    int64_t bs, sbs;        // elements between sequences (dense), and of the scales
    int32_t rs, srs;        // elements between rows
    int32_t dt;
    int32_t vec;            // base and strides allow whole vectors to be loaded and stored (set by the host for the kernel's vector)
};

struct SeqMap {
    const int32_t *start;   // packed: [n_seq + 1] first rows; null: dense
    const int32_t *len;     // dense: rows of each sequence, or null (all of them)
    int64_t rows;           // packed: rows of the array; dense: rows of a sequence
    int64_t Q;              // rows of a chunk
    int64_t nch;            // dense: chunks of a sequence (at least 1)
    int64_t nblk;           // chunk blocks in all (an upper bound where packed), less than 2^31
    int64_t per;            // rows of the array a block looks after that belong to no sequence (packed)
    int32_t n_seq;
};

// A chunk block b: sequence s, its chunk c.  Packed sequences get their blocks from floor(first row / Q) + s on: sequence s then has at
// least max(1, ceil(rows / Q)) blocks and none is shared, whatever the lengths are, without a table.
struct SeqChunk {
    int64_t begin;          // packed: first row of the sequence in the array; dense: 0
    int64_t len;            // rows of the sequence
    int64_t t0;             // first row of the chunk, counted in its sequence
    int32_t n;              // rows of the chunk (0: an empty sequence's only chunk)
    int32_t s;
    bool live, last;
    int64_t flat;           // begin (packed) or s * rows (dense): row of the sequence's first row in arrays of the operators' own
};

__device__ __forceinline__ int64_t seq_clamp(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

__device__ __forceinline__ void seq_bounds(const SeqMap &m, int64_t s, int64_t &begin, int64_t &len) {
    if (m.start) {
        begin = seq_clamp(m.start[s], 0, m.rows);
        len = seq_clamp(m.start[s + 1], begin, m.rows) - begin;
    } else {
        begin = 0;
        len = m.len ? seq_clamp(m.len[s], 0, m.rows) : m.rows;
    }
}

__device__ __forceinline__ int64_t seq_first_block(const SeqMap &m, int64_t s) {
    if (!m.start) return s * m.nch;
    return (int64_t)((uint32_t)seq_clamp(m.start[s], 0, m.rows) / (uint32_t)m.Q) + s;
}

// all lanes of the wavefront call it with the same b
__device__ __forceinline__ SeqChunk seq_locate(const SeqMap &m, int64_t b) {
    SeqChunk k;
    int64_t s, c;
    if (!m.start) {
        s = (int64_t)((uint32_t)b / (uint32_t)m.nch);
        c = b - s * m.nch;
        if (s >= m.n_seq) s = -1;
    } else {
        const int lane = threadIdx.x & 63;
        int cnt = 0;
        for (int i0 = 0; i0 < m.n_seq; i0 += 64) {
            const int i = i0 + lane;
            const bool at = i < m.n_seq && seq_first_block(m, i) <= b;
            cnt += __popcll(__builtin_amdgcn_ballot_w64(at));
        }
        s = cnt - 1;
        c = s >= 0 ? b - seq_first_block(m, s) : 0;
    }
    k.live = s >= 0 && c >= 0;
    k.s = (int32_t)(s >= 0 ? s : 0);
    k.begin = k.len = 0;
    if (k.live) seq_bounds(m, s, k.begin, k.len);
    k.t0 = c * m.Q;
    k.live = k.live && (k.t0 < k.len || (c == 0 && k.len == 0));
    const int64_t left = k.len - k.t0;
    k.n = (int32_t)(k.live ? (left < m.Q ? left : m.Q) : 0);
    k.last = k.live && k.t0 + m.Q >= k.len;
    k.flat = m.start ? k.begin : (int64_t)k.s * m.rows;
    return k;
}

// element offset of a view's row t of the chunk's sequence
__device__ __forceinline__ int64_t seq_off(const SeqMap &m, const SeqV &v, const SeqChunk &k, int64_t t) {
    return (m.start ? k.begin * v.rs : (int64_t)k.s * v.bs) + t * (int64_t)v.rs;
}
__device__ __forceinline__ int64_t seq_soff(const SeqMap &m, const SeqV &v, const SeqChunk &k, int64_t t) {
    return (m.start ? k.begin * v.srs : (int64_t)k.s * v.sbs) + t * v.srs;
}
// whether row r of the array (packed: row; dense: s * rows + t) belongs to a sequence
__device__ __forceinline__ bool seq_inside(const SeqMap &m, int64_t r) {
    if (m.start) return m.n_seq > 0 && r >= seq_clamp(m.start[0], 0, m.rows) && r < seq_clamp(m.start[m.n_seq], 0, m.rows);
    if (!m.len) return true;
    const int64_t s = r / m.rows;
    return r - s * m.rows < seq_clamp(m.len[s], 0, m.rows);
}

__device__ __forceinline__ void seq_store(const SeqV &v, int64_t off, float x) {
    if (v.dt == CRNN_DT_F32) ((float *)v.p)[off] = x;
    else ((uint16_t *)v.p)[off] = v.dt == CRNN_DT_BF16 ? seq_to_bf16(x) : seq_to_f16(x);
}
__device__ __forceinline__ void seq_store(const SeqV &v, int64_t off, double x) { ((double *)v.p)[off] = x; }

__device__ __forceinline__ float seq_load1(const SeqV &v, int64_t off, float) {
    if (v.dt == CRNN_DT_F32) return ((const float *)v.p)[off];
    const uint32_t b = ((const uint16_t *)v.p)[off];
    return v.dt == CRNN_DT_BF16 ? seq_as_float(b << 16) : seq_from_f16(b);
}
__device__ __forceinline__ double seq_load1(const SeqV &v, int64_t off, double) { return ((const double *)v.p)[off]; }

// Rows of an output that belong to no sequence become 0 (the caller asked for it by SeqMap-wide flag): block b of the launch takes its
// share of the array's rows, a lane its channel.
__device__ __forceinline__ void seq_zero_outside(const SeqMap &m, const SeqV &v, int64_t b, int64_t d, bool valid) {
    if (!v.p) return;
    if (m.start) {
        const int64_t lo = b * m.per, hi = lo + m.per < m.rows ? lo + m.per : m.rows;
        const int64_t first = m.n_seq > 0 ? seq_clamp(m.start[0], 0, m.rows) : m.rows, end = m.n_seq > 0 ? seq_clamp(m.start[m.n_seq], 0, m.rows) : m.rows;
        if (lo >= first && hi <= end) return;
        for (int64_t r = lo; r < hi; ++r)
            if ((r < first || r >= end) && valid) {
                if (v.dt == CRNN_DT_F64) seq_store(v, r * v.rs + d, 0.0);
                else seq_store(v, r * v.rs + d, 0.0f);
            }
    } else if (m.len) {
        const int64_t s = (uint32_t)b / (uint32_t)m.nch, c = b - s * m.nch, n = seq_clamp(m.len[s], 0, m.rows);
        const int64_t hi = (c + 1) * m.Q < m.rows ? (c + 1) * m.Q : m.rows;
        for (int64_t r = c * m.Q > n ? c * m.Q : n; r < hi; ++r)
            if (valid) {
                if (v.dt == CRNN_DT_F64) seq_store(v, s * v.bs + r * v.rs + d, 0.0);
                else seq_store(v, s * v.bs + r * v.rs + d, 0.0f);
            }
    }
}

// TB consecutive rows of one channel on their way into registers: the loads of several arrays are issued before the first one is needed,
// conversion comes afterwards.  IO: bytes of an element (8: double).  PM: 0 plain, 1 a checkpoint, 2 either (looked at per launch).  Row
// addresses are uniform, the lane adds a 32-bit offset; rows behind the chunk's n-th are read as the n-th (n >= 1): no branch stands between
// the loads and stores of a loop, so that the wait for a load need not wait for the stores behind it.
template <int IO> struct SeqIO { using C = float; using E = uint32_t; };
template <> struct SeqIO<2> { using C = float; using E = uint16_t; };
template <> struct SeqIO<8> { using C = double; using E = double; };

template <int IO, int PM, int TB>
struct SeqRows {
    using CT = typename SeqIO<IO>::C;
    using E = typename SeqIO<IO>::E;
    E r[TB];                     // checkpoint: the code, its scale byte above it
    // rows t .. t + TB - 1 of the chunk
    __device__ __forceinline__ void load(const SeqMap &m, const SeqV &v, const SeqChunk &k, int t, uint32_t d) {
        if (PM == 1 || (PM == 2 && v.dt == CRNN_DT_PACKED8)) {
            const int8_t *c = (const int8_t *)v.p + seq_off(m, v, k, k.t0);
            const uint8_t *e = v.sc + seq_soff(m, v, k, k.t0);
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const int64_t ii = t + i < k.n ? t + i : k.n - 1;
                r[i] = (E)((uint32_t)(uint8_t)(c + ii * v.rs)[d] | (uint32_t)(e + ii * v.srs)[d >> 5] << 8);
            }
        } else {
            const E *c = (const E *)v.p + seq_off(m, v, k, k.t0);
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const int64_t ii = t + i < k.n ? t + i : k.n - 1;
                r[i] = (c + ii * v.rs)[d];
            }
        }
    }
    __device__ __forceinline__ void get(const SeqV &v, CT (&o)[TB]) const {
        if (PM == 1 || (PM == 2 && v.dt == CRNN_DT_PACKED8)) {
#pragma unroll
            for (int i = 0; i < TB; ++i) o[i] = (CT)seq_unpack((int8_t)((uint32_t)r[i] & 0xffu), (uint32_t)r[i] >> 8 << 23);
        } else if (IO == 8) {
#pragma unroll
            for (int i = 0; i < TB; ++i) o[i] = (CT)r[i];
        } else if (IO == 4) {
#pragma unroll
            for (int i = 0; i < TB; ++i) o[i] = (CT)seq_as_float((uint32_t)r[i]);
        } else if (v.dt == CRNN_DT_BF16) {
#pragma unroll
            for (int i = 0; i < TB; ++i) o[i] = (CT)seq_as_float((uint32_t)r[i] << 16);
        } else {
#pragma unroll
            for (int i = 0; i < TB; ++i) o[i] = (CT)seq_from_f16((uint32_t)r[i]);
        }
    }
};

// Rows t .. t + TB - 1 of the chunk to an output.  Rows behind the n-th store the n-th once more, and a lane without a channel of its own (its
// inputs are the last channel's) stores the last channel's value once more.
template <int IO, int TB>
__device__ __forceinline__ void seq_put_rows(const SeqMap &m, const SeqV &v, const SeqChunk &k, int t, uint32_t d, typename SeqIO<IO>::C (&x)[TB]) {
    using E = typename SeqIO<IO>::E;
    E *c = (E *)v.p + seq_off(m, v, k, k.t0);
    E b[TB];
#pragma unroll
    for (int i = 1; i < TB; ++i) x[i] = t + i < k.n ? x[i] : x[i - 1];
#pragma unroll
    for (int i = 0; i < TB; ++i) {
        if (IO == 8) b[i] = (E)x[i];
        else if (IO == 4) b[i] = (E)seq_as_bits((float)x[i]);
    }
    if (IO == 2) {
        if (v.dt == CRNN_DT_BF16) {
#pragma unroll
            for (int i = 0; i < TB; ++i) b[i] = (E)seq_to_bf16((float)x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < TB; ++i) b[i] = (E)seq_to_f16((float)x[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < TB; ++i) (c + (int64_t)(t + i < k.n ? t + i : k.n - 1) * v.rs)[d] = b[i];
}

// x as an index of the vector unit: an LDS address that the compiler knows to be uniform is kept in a scalar register, and moved for every read
__device__ __forceinline__ int seq_vector_index(int x) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm("" : "+v"(x));
#endif
    return x;
}
// what a wavefront wrote to its own part of the LDS is there for all its lanes
__device__ __forceinline__ void seq_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// sum over the wavefront's lanes of V values at once: every exchange halves how many values a lane still carries, about 2 V operations in
// all where separate sums would take 6 V.  Afterwards the lane holds the sum of value seq_spread_index<V>(lane).
template <int V>
__device__ __forceinline__ int seq_spread_index(int lane) {
    int idx = 0, w = V / 2;
    for (int bit = 32; w >= 1; bit >>= 1, w >>= 1) idx += (lane & bit) ? w : 0;
    return idx;
}
// float: the exchanges across 32 and 16 lanes are the swaps of half registers, the closer ones lane moves inside a row of 16 (DPP: by 8
// within the row, mirrored halves, pairs, neighbours; a mirrored partner differs in the bit in question and that is all it takes)
template <int CTRL>
__device__ __forceinline__ float seq_dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ float seq_fold(float a, float b, bool hi) {
    const float send = hi ? a : b, keep = hi ? b : a;
    return keep + seq_dpp<CTRL>(send);
}
// one exchange of the two largest: lanes below / from bit 32 on (16) carry a / b on
__device__ __forceinline__ float seq_fold32(float a, float b) {
    const auto s = __builtin_amdgcn_permlane32_swap(seq_as_bits(a), seq_as_bits(b), false, false);
    return seq_as_float(s[0]) + seq_as_float(s[1]);
}
__device__ __forceinline__ float seq_fold16(float a, float b) {
    const auto s = __builtin_amdgcn_permlane16_swap(seq_as_bits(a), seq_as_bits(b), false, false);
    return seq_as_float(s[0]) + seq_as_float(s[1]);
}
__device__ __forceinline__ double seq_fold32(double a, double b) {
    const bool hi = (threadIdx.x & 32) != 0;
    return (hi ? b : a) + __shfl_xor(hi ? a : b, 32);
}
__device__ __forceinline__ double seq_fold16(double a, double b) {
    const bool hi = (threadIdx.x & 16) != 0;
    return (hi ? b : a) + __shfl_xor(hi ? a : b, 16);
}
template <int CTRL>
__device__ __forceinline__ double seq_fold(double a, double b, bool hi) {
    constexpr int BIT = CTRL == 0x128 ? 8 : CTRL == 0x141 ? 4 : CTRL == 0x4e ? 2 : 1;
    return (hi ? b : a) + __shfl_xor(hi ? a : b, BIT);
}
template <int CTRL>
__device__ __forceinline__ double seq_dpp(double x) {
    constexpr int BIT = CTRL == 0x128 ? 8 : CTRL == 0x141 ? 4 : CTRL == 0x4e ? 2 : 1;
    return __shfl_xor(x, BIT);
}
// the exchanges within 16 lanes of the F values that are left after those across 32 and 16
template <int F, class CT>
__device__ __forceinline__ CT seq_spread_rest(CT (&v)[F]) {
    static_assert(F == 4 || F == 8, "values of a row");
    const int lane = threadIdx.x & 63;
    const bool b8 = (lane & 8) != 0, b4 = (lane & 4) != 0, b2 = (lane & 2) != 0;
#pragma unroll
    for (int j = 0; j < F / 2; ++j) v[j] = seq_fold<0x128>(v[j], v[j + F / 2], b8);
#pragma unroll
    for (int j = 0; j < F / 4; ++j) v[j] = seq_fold<0x141>(v[j], v[j + F / 4], b4);
    if (F == 8) v[0] = seq_fold<0x4e>(v[0], v[F == 8 ? 1 : 0], b2);
    else v[0] += seq_dpp<0x4e>(v[0]);
    return v[0] + seq_dpp<0xb1>(v[0]);
}
// Rows of one launch that name the same slot are consecutive rows of that sequence: the first of them in row order does them all.
// A thread finds for row r whether an earlier row has its slot, and which row is the next.
__device__ __forceinline__ void seq_same_slot(const int32_t *slot, int64_t rows, int64_t r, int *before, int *next) {
    const int32_t k = slot[r];
    for (int64_t j = threadIdx.x; j < rows; j += blockDim.x)
        if (j != r && slot[j] == k) {
            if (j < r) atomicMax(before, 1);
            else atomicMin(next, (int)j);
        }
}

}  // namespace crnn
