// crnn_amd/csrc/seq_scan_kernel.hpp -- gfx950: the selective state space scan, its discrete adjoint and its single step.
//
//     delta = softplus(dt + dt_bias) (or dt + dt_bias)
//     h[t, d, n] = exp(delta A[d, n]) h[t - 1, d, n] + delta u B[t, g, n],   v[t, d] = sum_n C[t, g, n] h[t, d, n] + D[d] u
//     y = v, or v z sigmoid(z);   g = d / (channels of a group)
//
// the diagonal linear ODE h' = A h + B u over steps of their own length: the decay exact, the input to first order in the step (delta u B).
//
// Split.  A block owns 64 channels of one group (a tile), a lane a channel.  Forward, four wavefronts share the states: each row's step length,
// input and gate are worked out by one of them and handed round in the LDS, so are the row's B and C (the same for all lanes of a tile: read
// back as broadcasts) and each wavefront's part of sum_n C h.  Per row, channel and state that is one multiplication and one exponential for
// the decay and three multiply-adds: bound by the vector units, not by memory.  The gradient needs every state's neighbours in registers and
// gives a wavefront all states of its tile.
// Where tiles and sequences do not fill the card, time is cut into chunks: their ends without what came before (the forward kernel without its
// outputs, seq_scan_ends2_kernel for the gradient), the carry over the chunks of a sequence (seq_scan_carry_kernel: the decay over a chunk is
// exp(A sum delta)), then the chunks proper.  Sums over channels and blocks are taken in a fixed order: results do not change from run to run.
#pragma once
#include "seq_common.hpp"

namespace crnn {

constexpr int kScanTB = 4;      // gradient: rows whose loads are in flight together
constexpr int kScanRows = 8;    // forward: rows of a batch, two for each wavefront
constexpr int kScanWaves = 4;   // wavefronts of a block (gradient: each on its own channel tile)

struct ScanP {
    SeqMap m;
    SeqV u, dt, z, y, dy, du, ddt, dz, B, C;
    int64_t Bg, Cg, Bn, Cn;                       // elements between groups, between states
    const void *A, *Dskip, *dt_bias;              // in the compute type
    const void *state_in, *dstate_out;            // [n_seq][D][N]
    void *state_out, *dstate_in;
    void *acc;                                    // N > NS: sums over the states so far, 3 x [rows of all sequences][D]
    int64_t acc_n;                                // elements of one of them
    int32_t D, N, G, Dg, tpg, ntile;              // Dg channels and tpg tiles of 64 a group
    int32_t n0;                                   // first state of this launch
    int32_t first, fin;                           // first / last launch over the states
    int32_t softplus, zero_outside;
    int32_t nvec;                                 // N and the arrays that end in it allow four states at a time
    int32_t gate;                                 // z is there (else its view is u's, and what it gives is not used)
};

// ---- dB and dC
struct ScanMapsP {
    SeqV B, C;              // rs: elements between rows, group stride below
    int64_t Bg, Cg;         // elements between groups
    int64_t Bn, Cn;         // elements between states
    int64_t rows;           // rows of all sequences
    int64_t srows;          // dense: rows of a sequence (0: packed)
    int32_t G, N, n0;
    int32_t zero_outside;   // rows that belong to no sequence: 0, or left as they are
};
// the plane of state n of chunk block b in an [block][state][D] array: uniform, the lane adds its channel
template <int NS, class T>
__device__ __forceinline__ T *scan_plane(T *x, int64_t b, int n, int D) { return x + (b * NS + n) * D; }

struct ScanAt {
    SeqChunk k;
    int64_t b;
    int32_t tile, g, d;
    bool on, valid;         // on: the wavefront has a tile; valid: the lane has a channel
};
// the place of a wavefront of the gradient's kernels: chunk block, channel tile, channel of the lane
__device__ __forceinline__ ScanAt scan_at(const ScanP &p) {
    ScanAt a;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const uint32_t tb = (uint32_t)(p.ntile + kScanWaves - 1) / kScanWaves, b = blockIdx.x / tb;
    a.b = b;
    a.tile = (int32_t)(blockIdx.x - b * tb) * kScanWaves + wave;
    a.on = a.tile < p.ntile;
    const int t = a.on ? a.tile : p.ntile - 1;
    a.g = t / p.tpg;
    const int dl = (t - a.g * p.tpg) * 64 + lane;
    a.valid = a.on && dl < p.Dg;
    a.d = a.g * p.Dg + (dl < p.Dg ? dl : p.Dg - 1);
    a.k = seq_locate(p.m, a.b);
    return a;
}

// K states from the n-th on of row `row` of a [..][N] array (null, or behind the last state: 0), four at a time where the arrays allow it: the lanes
// are N elements apart, a load of each state by itself touches as many lines as one of four
template <class CT, int K>
__device__ __forceinline__ void scan_get(const ScanP &p, const void *x, int64_t row, int n, CT (&o)[K]) {
    constexpr int V = K < 4 ? K : 4;
    typedef CT VV __attribute__((ext_vector_type(V)));
    const CT *q = (const CT *)x + row * p.N + n;
    if (sizeof(CT) == 4 && x && p.nvec && n + K <= p.N) {
#pragma unroll
        for (int j = 0; j < K; j += V) {
            const VV v = *(const VV *)(q + j);
#pragma unroll
            for (int i = 0; i < V; ++i) o[j + i] = v[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < K; ++j) o[j] = x && n + j < p.N ? q[j] : CT(0);
    }
}
// Rates for exp2.  An infinite one counts as the type's largest: rows behind a chunk's n-th are steps of length 0, and 0 times infinity is NaN.
template <class CT, int K>
__device__ __forceinline__ void scan_rates(const ScanP &p, int d, int n, CT (&A2)[K]) {
    constexpr CT top = CT(sizeof(CT) == 8 ? 1.7976931348623157e308 : 3.4028234663852886e38);
    scan_get<CT, K>(p, p.A, d, n, A2);
#pragma unroll
    for (int j = 0; j < K; ++j) A2[j] *= CT(kLog2eD);
    CT big = CT(0);
#pragma unroll
    for (int j = 0; j < K; ++j) big = seq_max(big, seq_abs(A2[j]));
    if (big > top)          // (looked at first: a gradient's chunk has 20 rows for what it does once; a NaN stays one)
#pragma unroll
        for (int j = 0; j < K; ++j) A2[j] = A2[j] < -top ? -top : A2[j] > top ? top : A2[j];
}
// PAD: N does not fill the launch's NS states.  The states behind the last one have rates, maps and first states of 0, but 0 times an infinite step length,
// input or gradient is NaN: they are put to 0 after every row, or what is summed over the states would take it up.
// what a launch may meet: 0 plain arrays, all states at once; 1 the same with u, and z if there is one, as checkpoints; 2 anything
constexpr int kScanAny = 2;

// step lengths and inputs of TB rows; rows behind the n-th become steps of length 0 with nothing to add, so that the rows need no branches
template <int IO, int TB>
__device__ __forceinline__ void scan_steps(const ScanP &p, int n, typename SeqIO<IO>::C bias, typename SeqIO<IO>::C (&x)[TB], typename SeqIO<IO>::C (&u)[TB],
                                           typename SeqIO<IO>::C (&dl)[TB]) {
    using CT = typename SeqIO<IO>::C;
#pragma unroll
    for (int i = 0; i < TB; ++i) x[i] += bias;
    if (p.softplus) {
#pragma unroll
        for (int i = 0; i < TB; ++i) dl[i] = seq_softplus(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < TB; ++i) dl[i] = x[i];
    }
#pragma unroll
    for (int i = 1; i < TB; ++i) {
        dl[i] = i < n ? dl[i] : CT(0);
        u[i] = i < n ? u[i] : CT(0);
    }
}

// B and C of TB rows on their way to a wavefront's own part of the LDS, [row][B: NS | C: NS] in the compute type, 0 behind the last state: loaded
// into registers while the rows before are worked on (a lane has TB NS / 32 of them), put down when those are done, read back as
// broadcasts.  (As scalar operands they are free of the vector registers, but every row then waits for its own scalar load: the forward
// scan of 8190 rows of 4096 channels took 316 us so and 279 us from the LDS, 2048 rows of one sequence left whole 1.83 and 1.07 ms.)
template <int IO, int NS, int TB>
struct ScanMapRows {
    using CT = typename SeqIO<IO>::C;
    using E = typename SeqIO<IO>::E;
    static constexpr int V = TB * 2 * NS / 64, RPV = 64 / (2 * NS);   // values of a lane, rows of 64 values
    const E *at;            // of the lane's value in the chunk's first row
    int32_t rs;
    int32_t row0;
    bool in;
    E v[V];
    __device__ __forceinline__ void init(const ScanP &p, const ScanAt &a) {
        const int lane = threadIdx.x & 63, j = lane % (2 * NS), n = p.n0 + j % NS;
        const bool b = j < NS;
        row0 = lane / (2 * NS);
        in = n < p.N;
        const int nn = in ? n : p.N - 1;
        const E *pb = (const E *)p.B.p + seq_off(p.m, p.B, a.k, a.k.t0) + a.g * p.Bg, *pc = (const E *)p.C.p + seq_off(p.m, p.C, a.k, a.k.t0) + a.g * p.Cg;
        at = b ? pb + nn * p.Bn : pc + nn * p.Cn;
        rs = b ? p.B.rs : p.C.rs;
    }
    // rows t .. t + TB - 1 of the chunk
    __device__ __forceinline__ void load(int t, int n) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int r = t + row0 + k * RPV;
            v[k] = at[(int64_t)(r < n ? r : n - 1) * rs];
        }
    }
    // nv: rows of the chunk from the first of these on.  Those behind are 0: they stand for the last row once more
    __device__ __forceinline__ void put(int dt, CT *lds, int nv) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            CT x;
            if (IO == 8) x = (CT)v[k];
            else if (IO == 4) x = (CT)seq_as_float((uint32_t)v[k]);
            else x = (CT)(dt == CRNN_DT_BF16 ? seq_as_float((uint32_t)v[k] << 16) : seq_from_f16((uint32_t)v[k]));
            lds[k * 64 + lane] = in && row0 + k * RPV < nv ? x : CT(0);
        }
        seq_wave_sync();
    }
};

// the place of a block of the forward kernels: chunk block, channel tile
__device__ __forceinline__ ScanAt scan_tile(const ScanP &p) {
    ScanAt a;
    const uint32_t b = blockIdx.x / (uint32_t)p.ntile;
    a.b = b;
    a.tile = (int32_t)(blockIdx.x - b * (uint32_t)p.ntile);
    a.on = true;
    a.g = a.tile / p.tpg;
    const int dl = (a.tile - a.g * p.tpg) * 64 + (int)(threadIdx.x & 63);
    a.valid = dl < p.Dg;
    a.d = a.g * p.Dg + (dl < p.Dg ? dl : p.Dg - 1);
    a.k = seq_locate(p.m, a.b);
    return a;
}

// What the wavefronts of a forward block hand each other: step length and delta u of a batch's rows, its B and C, the parts of its sums.
template <class CT, int NS, bool OUT>
struct ScanShare {
    CT dl[kScanRows][64], du[kScanRows][64], maps[kScanRows][2 * NS], v[OUT ? kScanWaves : 1][OUT ? kScanRows : 1][64];
};

// 8190 rows of 4096 channels, 16 states, bf16: 157 us with outputs, 107 without, vector unit busy 95 % of the time.  A row, channel and
// state cost 8.3 and 5.8 vector instructions, of which 5 and 4 are the recurrence itself, the exponential counting twice: a pass that did
// nothing else would take 83 and 69 us.  The rest is mostly the step lengths and gates of the rows (each worked out once a tile).  1 x 64 x 1536: 17 us.

// ---- forward, a chunk.  OUT: outputs from its first state (start[block][n][d]; null: one chunk a sequence, from state_in), and the sequence's
// last state.  Not OUT: S = the chunk's last state from zero and the sum of delta (a sequence's last chunk is not asked).
template <int IO, int NS, int MODE, bool OUT, bool PAD>
__global__ __launch_bounds__(64 * kScanWaves, IO == 8 ? 3 : 6) void seq_scan_fwd_kernel(const ScanP p, const typename SeqIO<IO>::C *__restrict__ start,
                                                                                      typename SeqIO<IO>::C *__restrict__ S, typename SeqIO<IO>::C *__restrict__ sdel) {
    using CT = typename SeqIO<IO>::C;
    using E = typename SeqIO<IO>::E;
    constexpr int R = kScanRows, RW = kScanRows / kScanWaves, NW = NS / kScanWaves;      // rows and states of a wavefront
    constexpr int MV = R * 2 * NS >= 256 ? R * 2 * NS / 256 : 1;                         // values of B and C a thread brings
    typedef CT VN __attribute__((ext_vector_type(NW)));
    __shared__ __align__(16) ScanShare<CT, NS, OUT> sh;
    const ScanAt a = scan_tile(p);
    const bool fin = MODE != kScanAny || p.fin;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (OUT && p.zero_outside && fin && wave == 0) seq_zero_outside(p.m, p.y, a.b, a.d, a.valid);
    if (!a.k.live || (!OUT && a.k.last)) return;
    const int lim = p.N - p.n0;
    CT A2[NW], h[NW], sd = CT(0);
    scan_rates<CT, NW>(p, a.d, p.n0 + wave * NW, A2);
    if (OUT && start) {
#pragma unroll
        for (int j = 0; j < NW; ++j) h[j] = p.n0 + wave * NW + j < p.N ? scan_plane<NS>(start, a.b, wave * NW + j, p.D)[(uint32_t)a.d] : CT(0);
    } else scan_get<CT, NW>(p, OUT ? p.state_in : nullptr, (int64_t)a.k.s * p.D + a.d, p.n0 + wave * NW, h);
    if (a.k.n > 0) {
        const CT bias = p.dt_bias ? ((const CT *)p.dt_bias)[a.d] : CT(0), skip = OUT && p.Dskip ? ((const CT *)p.Dskip)[a.d] : CT(0);
        // the thread's values of B and C: column j of rows row0, row0 + 256 / (2 NS), ..
        const int mj = threadIdx.x % (2 * NS), mrow = threadIdx.x / (2 * NS), mn = p.n0 + mj % NS;
        const bool min_ = mn < p.N, mb = mj < NS;
        const int mnn = min_ ? mn : p.N - 1;
        const E *pb = (const E *)p.B.p + seq_off(p.m, p.B, a.k, a.k.t0) + a.g * p.Bg, *pc = (const E *)p.C.p + seq_off(p.m, p.C, a.k, a.k.t0) + a.g * p.Cg;
        const E *mat = mb ? pb + mnn * p.Bn : pc + mnn * p.Cn;
        const int32_t mrs = mb ? p.B.rs : p.C.rs;
        E mv[MV];
        SeqRows<IO, MODE, RW> ru, rz;
        SeqRows<IO, 0, RW> rd;
        auto fetch = [&](int t) {
#pragma unroll
            for (int k = 0; k < MV; ++k) {
                const int r = t + mrow + k * (256 / (2 * NS));
                mv[k] = mat[(int64_t)(r < a.k.n ? r : a.k.n - 1) * mrs];
            }
            ru.load(p.m, p.u, a.k, t + wave * RW, a.d);
            rd.load(p.m, p.dt, a.k, t + wave * RW, a.d);
            if (OUT) rz.load(p.m, p.z, a.k, t + wave * RW, a.d);
        };
        const CT *bc = &sh.maps[0][0] + seq_vector_index(wave * NW);        // the wavefront's states in B, NS further in C
        fetch(0);
#pragma unroll 1
        for (int t = 0; t < a.k.n; t += R) {
            const int mine = t + wave * RW;              // the wavefront's first row of the batch
            CT u[RW], x[RW], z[RW], dl[RW];
            ru.get(p.u, u);
            rd.get(p.dt, x);
            if (OUT) rz.get(p.z, z);
#pragma unroll
            for (int k = 0; k < MV; ++k) {
                CT m;
                if (IO == 8) m = (CT)mv[k];
                else if (IO == 4) m = (CT)seq_as_float((uint32_t)mv[k]);
                else m = (CT)(p.B.dt == CRNN_DT_BF16 ? seq_as_float((uint32_t)mv[k] << 16) : seq_from_f16((uint32_t)mv[k]));
                if (R * 2 * NS >= 256 || mrow < R) sh.maps[(mrow + k * (256 / (2 * NS))) % R][mj] = min_ && t + mrow + k * (256 / (2 * NS)) < a.k.n ? m : CT(0);
            }
            fetch(t + R);
#pragma unroll
            for (int i = 0; i < RW; ++i) {
                x[i] += bias;
                dl[i] = p.softplus ? seq_softplus(x[i]) : x[i];
                const bool in = mine + i < a.k.n;
                dl[i] = in ? dl[i] : CT(0);
                sh.dl[wave * RW + i][lane] = dl[i];
                sh.du[wave * RW + i][lane] = in ? dl[i] * u[i] : CT(0);
                if (!OUT) sd += dl[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const CT d = sh.dl[i][lane], du = sh.du[i][lane];
                const VN b = *(const VN *)(bc + i * (2 * NS)), c = *(const VN *)(bc + i * (2 * NS) + (OUT ? NS : 0));
                CT v = CT(0);
#pragma unroll
                for (int j = 0; j < NW; ++j) {
                    h[j] = seq_fma(seq_exp2(d * A2[j]), h[j], du * b[j]);
                    if (PAD) h[j] = wave * NW + j < lim ? h[j] : CT(0);
                    if (OUT) v = seq_fma(h[j], c[j], v);
                }
                if (OUT) sh.v[OUT ? wave : 0][OUT ? i : 0][lane] = v;
            }
            __syncthreads();
            if (OUT) {
#pragma unroll
                for (int i = 0; i < RW; ++i) {
                    CT v = CT(0);
#pragma unroll
                    for (int w = 0; w < kScanWaves; ++w) v += sh.v[OUT ? w : 0][OUT ? wave * RW + i : 0][lane];
                    const int row = mine + i;
                    if (row >= a.k.n) break;
                    if (MODE == kScanAny && p.acc) {
                        CT *acc = (CT *)p.acc + (a.k.flat + a.k.t0 + row) * p.D + a.d;
                        if (!p.first) v += *acc;
                        if (!fin && a.valid) *acc = v;
                    }
                    if (!fin) continue;
                    v = p.Dskip ? seq_fma(skip, u[i], v) : v;        // (absent: not 0 times an infinite input)
                    const CT g = z[i] * seq_sigmoid(z[i]);
                    v = p.gate ? v * g : v;
                    seq_store(p.y, seq_off(p.m, p.y, a.k, a.k.t0 + row) + a.d, v);     // (lanes without a channel: the last channel's value again)
                }
            }
        }
    }
    if (OUT) {
        if (a.k.last && p.state_out && a.valid)
#pragma unroll
            for (int j = 0; j < NW; ++j) {
                const int n = p.n0 + wave * NW + j;
                if (n < p.N) ((CT *)p.state_out)[((int64_t)a.k.s * p.D + a.d) * p.N + n] = h[j];
            }
        return;
    }
    // every wavefront summed its own rows' step lengths
    sh.dl[wave][lane] = sd;
    __syncthreads();
    if (!a.valid) return;
#pragma unroll
    for (int j = 0; j < NW; ++j) scan_plane<NS>(S, a.b, wave * NW + j, p.D)[(uint32_t)a.d] = h[j];
    if (wave == 0) sdel[a.b * p.D + a.d] = (sh.dl[0][lane] + sh.dl[1][lane]) + (sh.dl[2][lane] + sh.dl[3][lane]);
}

// whether one of these products of decays is infinite or NaN (none is negative: their bits are ordered like the values, infinities and NaN above all)
template <int NS>
__device__ __forceinline__ bool scan_left_range(const float (&P)[NS]) {
    uint32_t m = 0;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const uint32_t b = seq_as_bits(P[n]) & 0x7fffffffu;
        m = b > m ? b : m;
    }
    return m >= 0x7f800000u;
}
template <int NS>
__device__ __forceinline__ bool scan_left_range(const double (&P)[NS]) {
    bool out = false;
#pragma unroll
    for (int n = 0; n < NS; ++n) out = out || !(P[n] <= 1.7976931348623157e308);
    return out;
}

// ---- gradient, a chunk by itself: S = its last state from zero, the sum of delta, and G = what its outputs' gradients r pass back to the state
// before it, sum_t (prod of the decays up to t) r C -- taken in the forward direction, so that one exponential serves both.
// 6144 rows of 2048 channels, 16 states, u and z in 8 bits: 82 us, vector unit busy 84 %.
template <int IO, int NS, int MODE>
__global__ __launch_bounds__(64 * kScanWaves, IO == 8 ? 2 : 3) void seq_scan_ends2_kernel(const ScanP p, typename SeqIO<IO>::C *__restrict__ S,
                                                                                                  typename SeqIO<IO>::C *__restrict__ Gb,
                                                                                                  typename SeqIO<IO>::C *__restrict__ sdel) {
    using CT = typename SeqIO<IO>::C;
    constexpr int TB = kScanTB;
    __shared__ CT smaps[kScanWaves][TB * 2 * NS];
    CT *maps = smaps[threadIdx.x >> 6];
    const ScanAt a = scan_at(p);
    if (!a.on || !a.k.live) return;
    CT A2[NS], h[NS], P[NS], g[NS];
    scan_rates<CT, NS>(p, a.d, p.n0, A2);
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        h[n] = CT(0);
        P[n] = CT(1);
        g[n] = CT(0);
    }
    CT sd = CT(0);
    if (a.k.n > 0) {
        const CT bias = p.dt_bias ? ((const CT *)p.dt_bias)[a.d] : CT(0);
        SeqRows<IO, MODE, TB> ru, rz;
        SeqRows<IO, 0, TB> rd, ry;
        ScanMapRows<IO, NS, TB> rm;
        rm.init(p, a);
        rm.load(0, a.k.n);
        ru.load(p.m, p.u, a.k, 0, a.d);
        rd.load(p.m, p.dt, a.k, 0, a.d);
        ry.load(p.m, p.dy, a.k, 0, a.d);
        rz.load(p.m, p.z, a.k, 0, a.d);
#pragma unroll 1
        for (int t = 0; t < a.k.n; t += TB) {
            CT u[TB], x[TB], z[TB], y[TB], dl[TB];
            ru.get(p.u, u);
            rd.get(p.dt, x);
            ry.get(p.dy, y);
            rz.get(p.z, z);
            rm.put(p.B.dt, maps, a.k.n - t);
            rm.load(t + TB, a.k.n);
            ru.load(p.m, p.u, a.k, t + TB, a.d);
            rd.load(p.m, p.dt, a.k, t + TB, a.d);
            ry.load(p.m, p.dy, a.k, t + TB, a.d);
            rz.load(p.m, p.z, a.k, t + TB, a.d);
            scan_steps<IO, TB>(p, a.k.n - t, bias, x, u, dl);
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const CT gz = z[i] * seq_sigmoid(z[i]);
                y[i] = p.gate ? y[i] * gz : y[i];
                y[i] = t + i < a.k.n ? y[i] : CT(0);
            }
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const CT *bc = maps + i * (2 * NS);
                const CT du = dl[i] * u[i];
                sd += dl[i];
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    const CT e = seq_exp2(dl[i] * A2[n]);
                    h[n] = seq_fma(e, h[n], du * bc[n]);
                    P[n] *= e;
                    g[n] = seq_fma(P[n], y[i] * bc[NS + n], g[n]);
                }
            }
            seq_wave_sync();
        }
        // decays above one (a positive rate, a negative step length) may have taken P out of range, where it makes NaN of an r C of 0: then G row by row
        // from the last to the first, as the formula has it (only the channels that need it: the others keep their bits)
        if (scan_left_range(P)) {
#pragma unroll
            for (int n = 0; n < NS; ++n) g[n] = CT(0);
#pragma unroll 1
            for (int t = a.k.n - 1; t >= 0; --t) {
                SeqRows<IO, MODE, 1> qz;
                SeqRows<IO, 0, 1> qd, qy;
                CT z[1], x[1], y[1];
                qd.load(p.m, p.dt, a.k, t, a.d);
                qy.load(p.m, p.dy, a.k, t, a.d);
                qz.load(p.m, p.z, a.k, t, a.d);
                qd.get(p.dt, x);
                qy.get(p.dy, y);
                qz.get(p.z, z);
                const CT dl = p.softplus ? seq_softplus(x[0] + bias) : x[0] + bias, r = p.gate ? y[0] * (z[0] * seq_sigmoid(z[0])) : y[0];
                const int64_t c0 = seq_off(p.m, p.C, a.k, a.k.t0 + t) + a.g * p.Cg;
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    const CT c = p.n0 + n < p.N ? seq_load1(p.C, c0 + (p.n0 + n) * p.Cn, CT(0)) : CT(0);
                    g[n] = seq_fma(r, c, g[n]) * seq_exp2(dl * A2[n]);
                }
            }
        }
    }
    if (!a.valid) return;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        scan_plane<NS>(S, a.b, n, p.D)[(uint32_t)a.d] = h[n];
        scan_plane<NS>(Gb, a.b, n, p.D)[(uint32_t)a.d] = g[n];
    }
    sdel[a.b * p.D + a.d] = sd;
}

// ---- carry over the chunks of a sequence: S becomes each chunk's first state, G (may be null) what reaches each chunk's last state from
// the rows behind it.  A thread per (sequence, state, channel).  Bound by memory: S and G of 308 chunks x 16 states x 2048 channels once in and once
// out, 161 MB in 38 us (4.2 TB/s).
template <class CT, int NS>
__global__ __launch_bounds__(256) void seq_scan_carry_kernel(const ScanP p, CT *__restrict__ S, CT *__restrict__ Gb, const CT *__restrict__ sdel) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (int64_t)NS * p.D;
    if (i >= per * p.m.n_seq) return;
    const int64_t s = i / per;
    const int n = (int)((i - s * per) / p.D), d = (int)(i % p.D);
    if (p.n0 + n >= p.N) return;      // behind the last state S and G are 0 and stay so
    int64_t begin, len;
    seq_bounds(p.m, s, begin, len);
    const int64_t b0 = seq_first_block(p.m, s), nc = len > 0 ? (len + p.m.Q - 1) / p.m.Q : 1;
    const int64_t at = (s * p.D + d) * p.N + p.n0 + n;
    const CT A2 = ((const CT *)p.A)[(int64_t)d * p.N + p.n0 + n] * CT(kLog2eD);
    // the loads of eight chunks at once; the sequence of chunks itself is a scaled product (seq_grow) and a sum each
    constexpr int CB = 8;
    const int64_t stride = (int64_t)NS * p.D;
    CT *Sp = S + (b0 * NS + n) * p.D + d;
    const CT *dp = sdel + b0 * p.D + d;
    CT h = p.state_in ? ((const CT *)p.state_in)[at] : CT(0);
    for (int64_t c0 = 0; c0 < nc; c0 += CB) {
        CT own[CB], e[CB];
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            const int64_t c = c0 + i < nc ? c0 + i : nc - 1;
            own[i] = Sp[c * stride];
            e[i] = dp[c * p.D];
        }
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            if (c0 + i < nc) Sp[(c0 + i) * stride] = h;
            h = seq_grow(h, A2 * e[i]) + own[i];
        }
    }
    if (!Gb) return;
    CT *Gp = Gb + (b0 * NS + n) * p.D + d;
    CT q = p.dstate_out ? ((const CT *)p.dstate_out)[at] : CT(0);
    for (int64_t c0 = nc - 1; len > 0 && c0 >= 0; c0 -= CB) {
        CT own[CB], e[CB];
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            const int64_t c = c0 - i >= 0 ? c0 - i : 0;
            own[i] = Gp[c * stride];
            e[i] = dp[c * p.D];
        }
#pragma unroll
        for (int i = 0; i < CB; ++i)
            if (c0 - i >= 0) {
                Gp[(c0 - i) * stride] = q;
                q = seq_grow(q, A2 * e[i]) + own[i];
            }
    }
    if (p.dstate_in) ((CT *)p.dstate_in)[at] = q;
}

// ---- adjoint of a chunk of at most kScanBwdQ rows.  Forward over the chunk once, keeping the state in front of every kScanBwdTB rows in LDS; then,
// from the last kScanBwdTB rows to the first: those rows once more, each row's decay a and a h[t - 1] kept in registers (2 NS x kScanBwdTB;
// h[t] is one multiply-add away, and dA needs the product itself), and the reverse sweep over them.  dB and dC are sums over channels: a
// wavefront's part goes to part[tile][row][B: NS | C: NS], summed over the tiles in a fixed order by seq_scan_sum_maps_kernel.
// Four rows and five times four a chunk: two wavefronts a SIMD fill the registers (256 a lane) and the LDS (16.5 KB each) about together.
// 6144 rows of 2048 channels, 16 states, u and z in 8 bits: 276 to 294 us, vector unit busy 69 %: 33 vector instructions a row, channel and state (21 of
// them the reverse row, folds of dB and dC included), the rest of the time both wavefronts of a SIMD wait (a row's maps from the LDS, the next rows).
constexpr int kScanBwdTB = 4, kScanBwdSub = 5, kScanBwdQ = kScanBwdTB * kScanBwdSub;
template <int IO, int NS, int MODE, bool PAD>
__global__ __launch_bounds__(64 * kScanWaves, 2) void seq_scan_bwd_kernel(const ScanP p, const typename SeqIO<IO>::C *__restrict__ start,
                                                                          const typename SeqIO<IO>::C *__restrict__ back, typename SeqIO<IO>::C *__restrict__ part,
                                                                          typename SeqIO<IO>::C *__restrict__ ppart) {
    using CT = typename SeqIO<IO>::C;
    constexpr int TB = kScanBwdTB, H = NS / 2;
    __shared__ CT keep[kScanWaves][kScanBwdSub - 1][NS][64];
    __shared__ CT smaps[kScanWaves][TB * 2 * NS];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    CT *maps = smaps[wave];
    const ScanAt a = scan_at(p);
    if (!a.on) return;
    const bool fin = MODE != kScanAny || p.fin;
    if (p.zero_outside && fin) {
        seq_zero_outside(p.m, p.du, a.b, a.d, a.valid);
        seq_zero_outside(p.m, p.ddt, a.b, a.d, a.valid);
        seq_zero_outside(p.m, p.dz, a.b, a.d, a.valid);
    }
    CT dA[NS], dD = CT(0), db = CT(0);
#pragma unroll
    for (int n = 0; n < NS; ++n) dA[n] = CT(0);
    if (a.k.live && a.k.n > 0) {
        const int lim = p.N - p.n0;
        auto real = [&](int n, CT x) { return !PAD || n < lim ? x : CT(0); };
        CT A2[NS], h[NS], q[NS];
        scan_rates<CT, NS>(p, a.d, p.n0, A2);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            h[n] = scan_plane<NS>(start, a.b, n, p.D)[(uint32_t)a.d];
            q[n] = scan_plane<NS>(back, a.b, n, p.D)[(uint32_t)a.d];
        }
        const CT bias = p.dt_bias ? ((const CT *)p.dt_bias)[a.d] : CT(0), skip = p.Dskip ? ((const CT *)p.Dskip)[a.d] : CT(0);
        const int nsub = (a.k.n + TB - 1) / TB;
        SeqRows<IO, MODE, TB> ru, rz;
        SeqRows<IO, 0, TB> rd, ry;
        ScanMapRows<IO, NS, TB> rm;
        rm.init(p, a);
        rm.load(0, a.k.n);
        ru.load(p.m, p.u, a.k, 0, a.d);
        rd.load(p.m, p.dt, a.k, 0, a.d);
#pragma unroll 1
        for (int k = 0; k < nsub - 1; ++k) {
            CT u[TB], x[TB], dl[TB];
            ru.get(p.u, u);
            rd.get(p.dt, x);
            rm.put(p.B.dt, maps, TB);
            // the next rows; the last ones of the chunk stay for the way back
            rm.load((k + 1) * TB, a.k.n);
            ru.load(p.m, p.u, a.k, (k + 1) * TB, a.d);
            rd.load(p.m, p.dt, a.k, (k + 1) * TB, a.d);
            scan_steps<IO, TB>(p, TB, bias, x, u, dl);
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const CT *bc = maps + i * (2 * NS);
                const CT du = dl[i] * u[i];
#pragma unroll
                for (int n = 0; n < NS; ++n) h[n] = seq_fma(seq_exp2(dl[i] * A2[n]), h[n], du * bc[n]);
            }
#pragma unroll
            for (int n = 0; n < NS; ++n) keep[wave][k][n][lane] = h[n];
            seq_wave_sync();
        }
        ry.load(p.m, p.dy, a.k, (nsub - 1) * TB, a.d);
        rz.load(p.m, p.z, a.k, (nsub - 1) * TB, a.d);
        CT *prow = part + ((int64_t)a.tile * p.acc_n + a.k.flat + a.k.t0) * (2 * NS);
        const uint32_t pidx = (uint32_t)seq_spread_index<2 * NS>(lane);
#pragma unroll 1
        for (int k = nsub - 1; k >= 0; --k) {
            const int t = k * TB, nv = a.k.n - t, before = k > 0 ? t - TB : 0;
            CT u[TB], x[TB], z[TB], y[TB], dl[TB], ah[TB][NS];
            ru.get(p.u, u);
            rd.get(p.dt, x);
            rm.put(p.B.dt, maps, nv);
            rm.load(before, a.k.n);
            ru.load(p.m, p.u, a.k, before, a.d);
            rd.load(p.m, p.dt, a.k, before, a.d);
            if (k > 0) {
#pragma unroll
                for (int n = 0; n < NS; ++n) h[n] = keep[wave][k - 1][n][lane];
            } else {
#pragma unroll
                for (int n = 0; n < NS; ++n) h[n] = scan_plane<NS>(start, a.b, n, p.D)[(uint32_t)a.d];
            }
            scan_steps<IO, TB>(p, nv, bias, x, u, dl);
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                const CT *bc = maps + i * (2 * NS);
                const CT du = dl[i] * u[i];
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    ah[i][n] = real(n, seq_exp2(dl[i] * A2[n]) * h[n]);
                    h[n] = seq_fma(du, bc[n], ah[i][n]);
                }
            }
            ry.get(p.dy, y);
            rz.get(p.z, z);
            ry.load(p.m, p.dy, a.k, before, a.d);
            rz.load(p.m, p.z, a.k, before, a.d);
            CT odu[TB], odt[TB], odz[TB];
#pragma unroll
            for (int i = TB - 1; i >= 0; --i) {
                __builtin_amdgcn_sched_barrier(0);      // a row after the other: interleaved they would not fit the registers
                const bool in = i < nv;
                const int64_t ii = t + (in ? i : nv - 1);
                const CT du = dl[i] * u[i], yi = in ? y[i] : CT(0), zi = in ? z[i] : CT(0);
                const CT sg = seq_sigmoid(zi), gz = zi * sg, r = p.gate ? yi * gz : yi;
                const CT *bc = maps + i * (2 * NS);
                CT v = CT(0), qb = CT(0), qa = CT(0), f[H], dle = dl[i];
                asm volatile("" : "+v"(dle));      // the decays are formed again rather than kept: NS registers a row
                const CT duv = a.valid ? du : CT(0), rv = a.valid ? r : CT(0);
#pragma unroll
                for (int j = 0; j < H; ++j) {       // states j and j + NS / 2 together: their parts of dB, dC fold at once
                    CT w[2];
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const int n = j + s * H;
                        const CT hn = real(n, seq_fma(du, bc[n], ah[i][n]));
                        q[n] = real(n, seq_fma(r, bc[NS + n], q[n]));
                        v = seq_fma(hn, bc[NS + n], v);
                        qb = seq_fma(q[n], bc[n], qb);
                        const CT m = q[n] * ah[i][n];
                        qa = seq_fma(m, A2[n], qa);
                        dA[n] = seq_fma(m, dl[i], dA[n]);
                        w[s] = seq_fold32(q[n] * duv, rv * hn);
                        q[n] *= seq_exp2(dle * A2[n]);
                    }
                    f[j] = seq_fold16(w[0], w[1]);
                }
                asm volatile("" : "+v"(v), "+v"(qb), "+v"(qa));      // here, not where they are used: a sum moved there keeps its terms alive
                // lanes that hold the same sum store it together; rows behind the n-th come first and are overwritten by the n-th
                (prow + ii * (2 * NS))[pidx] = seq_spread_rest(f);
                if (MODE == kScanAny && p.acc && in) {
                    CT *acc = (CT *)p.acc + (a.k.flat + a.k.t0 + ii) * p.D + a.d;
                    const int64_t stride = p.acc_n * p.D;
                    if (!p.first) { v += acc[0]; qb += acc[stride]; qa += acc[2 * stride]; }
                    if (!fin && a.valid) { acc[0] = v; acc[stride] = qb; acc[2 * stride] = qa; }
                }
                CT ddt = seq_fma(qa, CT(0.6931471805599453), qb * u[i]);
                const CT sx = seq_sigmoid(x[i]);
                ddt = p.softplus ? ddt * sx : ddt;
                ddt = in ? ddt : CT(0);
                dD = seq_fma(r, u[i], dD);
                db += ddt;
                odu[i] = seq_fma(dl[i], qb, p.Dskip ? r * skip : CT(0));
                odt[i] = ddt;
                v = p.Dskip ? seq_fma(skip, u[i], v) : v;
                odz[i] = yi * v * (sg * seq_fma(zi, CT(1) - sg, CT(1)));
            }
            seq_wave_sync();
            if (fin) {
                seq_put_rows<IO, TB>(p.m, p.du, a.k, t, a.d, odu);
                seq_put_rows<IO, TB>(p.m, p.ddt, a.k, t, a.d, odt);
                if (p.gate) seq_put_rows<IO, TB>(p.m, p.dz, a.k, t, a.d, odz);
            }
        }
    }
    if (!a.valid) return;
#pragma unroll
    for (int n = 0; n < NS; ++n) scan_plane<NS + 2>(ppart, a.b, n, p.D)[(uint32_t)a.d] = dA[n];
    scan_plane<NS + 2>(ppart, a.b, NS, p.D)[(uint32_t)a.d] = dD;
    scan_plane<NS + 2>(ppart, a.b, NS + 1, p.D)[(uint32_t)a.d] = db;
}

// ---- dB, dC: the tiles of a group in order.  dst: views like B and C.  (6144 rows, 32 tiles of 2 x 16 sums: 25 MB in 7.5 us.)
template <class CT, int NS>
__global__ __launch_bounds__(256) void seq_scan_sum_maps_kernel(const SeqMap m, const ScanMapsP p, const CT *__restrict__ part, int32_t tpg) {
    const int64_t total = p.rows * p.G * 2 * NS;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int j = (int)(i % (2 * NS));
        const int64_t rg = i / (2 * NS), g = rg % p.G, r = rg / p.G;
        const int n = p.n0 + (j % NS);
        if (n >= p.N) continue;
        const bool inside = seq_inside(m, r);
        if (!inside && !p.zero_outside) continue;
        CT sum = CT(0);
        if (inside)
            for (int k = 0; k < tpg; k += 8) {
                CT x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = part[((g * tpg + (k + e < tpg ? k + e : tpg - 1)) * p.rows + r) * (2 * NS) + j];
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += k + e < tpg ? x[e] : CT(0);
            }
        const SeqV &v = j < NS ? p.B : p.C;
        const int64_t at = p.srows ? (r / p.srows) * v.bs + (r % p.srows) * v.rs : r * v.rs;
        seq_store(v, at + g * (j < NS ? p.Bg : p.Cg) + n * (j < NS ? p.Bn : p.Cn), sum);
    }
}

// ---- sums over the blocks of a launch, in double and in a fixed order: in[block][count] -> out.  A thread block takes 32 neighbouring columns, eight
// threads each every eighth block of its own, then one of them adds the eight.  in is [block][planes][D]: the first `lim` planes go to
// out[d width + off + plane], plane p0 to out0[d], plane p0 + 1 to out1[d] (either may be null).  (308 blocks x 18 planes x 2048: 45 MB in 10 us.)
template <class CT>
__global__ __launch_bounds__(256) void seq_sum_blocks_kernel(const CT *__restrict__ in, int64_t nblk, int64_t count, CT *__restrict__ out, CT *__restrict__ out0, CT *__restrict__ out1,
                                                             int32_t D, int32_t width, int32_t off, int32_t lim, int32_t p0) {
    __shared__ double sh[8][32];
    const int col = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int64_t i = (int64_t)blockIdx.x * 32 + col;
    double s = 0.0;
    if (i < count) {
        int64_t b = k;
        for (; b + 24 < nblk; b += 32) {
            const CT x0 = in[b * count + i], x1 = in[(b + 8) * count + i], x2 = in[(b + 16) * count + i], x3 = in[(b + 24) * count + i];
            s += (double)x0;
            s += (double)x1;
            s += (double)x2;
            s += (double)x3;
        }
        for (; b < nblk; b += 8) s += (double)in[b * count + i];
    }
    sh[k][col] = s;
    __syncthreads();
    if (k || i >= count) return;
    for (int j = 1; j < 8; ++j) s += sh[j][col];
    const int64_t j = i / D, d = i % D;
    if (j < lim) out[d * width + off + j] = (CT)s;
    if (j == p0 && out0) out0[d] = (CT)s;
    if (j == p0 + 1 && out1) out1[d] = (CT)s;
}

// ---- one row for each of many running sequences, states updated in place.  LPC lanes share a channel, four states each (16-byte loads of
// the state where its rows are so aligned), so that a wavefront's state accesses are contiguous: the step is bound by them.  250 rows of
// 4096 channels, 16 states: 140 MB in 34.6 us (4.0 TB/s; a copy of as much reaches 4.7).  One row of 2048 channels: 4.2 us, a chain of three loads.
struct ScanStepP {
    SeqV u, dt, z, y, B, C;             // rs: between rows
    int64_t Bg, Cg, Bn, Cn;
    const void *A, *Dskip, *dt_bias;
    void *state;                        // [n_slots][D][N]
    const int32_t *slot;                // null: row r has slot r
    int64_t rows, n_slots;
    int32_t D, N, G, Dg, softplus, gate, lpc, vec;
};
// CPT channels a thread, 256 / lpc apart.  All that the row reads is on its way before the first of it is used or another row's slot is looked
// at, and what belongs to the row is looked up once for the CPT channels.
template <int IO>
__device__ __forceinline__ typename SeqIO<IO>::C scan_value(typename SeqIO<IO>::E e, int dt) {
    using CT = typename SeqIO<IO>::C;
    if (IO == 8) return (CT)e;
    if (IO == 4) return (CT)seq_as_float((uint32_t)e);
    return (CT)(dt == CRNN_DT_BF16 ? seq_as_float((uint32_t)e << 16) : seq_from_f16((uint32_t)e));
}
template <int IO, int CPT>
struct ScanStepRow {
    using E = typename SeqIO<IO>::E;
    E u[CPT], x[CPT], z[CPT], b[4], c[4];
    __device__ __forceinline__ void maps(const ScanStepP &p, int64_t r, int g, int n0) {
        const E *pb = (const E *)p.B.p + r * p.B.rs + g * p.Bg, *pc = (const E *)p.C.p + r * p.C.rs + g * p.Cg;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = n0 + i < p.N ? n0 + i : p.N - 1;
            b[i] = pb[n * p.Bn];
            c[i] = pc[n * p.Cn];
        }
    }
    __device__ __forceinline__ void load(const ScanStepP &p, int64_t r, const int (&d)[CPT], int n0) {
#pragma unroll
        for (int k = 0; k < CPT; ++k) {
            u[k] = ((const E *)p.u.p + r * p.u.rs)[(uint32_t)d[k]];
            x[k] = ((const E *)p.dt.p + r * p.dt.rs)[(uint32_t)d[k]];
            z[k] = ((const E *)p.z.p + r * p.z.rs)[(uint32_t)d[k]];      // (u's where there is no gate)
        }
        maps(p, r, p.G > 1 ? d[0] / p.Dg : 0, n0);
    }
};
template <int IO, int CPT>
__global__ __launch_bounds__(256) void seq_scan_step_kernel(const ScanStepP p) {
    using CT = typename SeqIO<IO>::C;
    __shared__ int before, next;
    typedef CT V4 __attribute__((ext_vector_type(4)));
    const int cpb = 256 / p.lpc, sub = threadIdx.x % p.lpc, dl = threadIdx.x / p.lpc;
    const uint32_t cb = (uint32_t)(p.D + cpb * CPT - 1) / (uint32_t)(cpb * CPT), r0 = blockIdx.x / cb;
    int64_t r = r0;
    const int d0 = (int)(blockIdx.x - r0 * cb) * cpb * CPT + dl;
    int d[CPT];
#pragma unroll
    for (int c = 0; c < CPT; ++c) d[c] = d0 + c * cpb < p.D ? d0 + c * cpb : p.D - 1;
    const int64_t slot = p.slot ? p.slot[r] : r;
    const bool there = slot >= 0 && slot < p.n_slots;
    if (!there) {
        if (sub == 0)
#pragma unroll
            for (int c = 0; c < CPT; ++c)
                if (d0 + c * cpb < p.D) seq_store(p.y, r * (int64_t)p.y.rs + d[c], CT(0));
        return;
    }
    const int n0 = sub * 4;
    CT A2[CPT][4], h[CPT][4], bias[CPT], skip[CPT];
    CT *st = (CT *)p.state + slot * (int64_t)p.D * p.N + n0;
    const CT *pa = (const CT *)p.A + n0;
    if (p.vec) {
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const V4 s = *(const V4 *)(st + (int64_t)d[c] * p.N), a = *(const V4 *)(pa + (int64_t)d[c] * p.N);
#pragma unroll
            for (int i = 0; i < 4; ++i) { A2[c][i] = a[i]; h[c][i] = s[i]; }
        }
    } else {
#pragma unroll
        for (int c = 0; c < CPT; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = n0 + i < p.N;
                A2[c][i] = in ? pa[(int64_t)d[c] * p.N + i] : CT(0);
                h[c][i] = in ? st[(int64_t)d[c] * p.N + i] : CT(0);
            }
    }
    ScanStepRow<IO, CPT> row;
    row.load(p, r, d, n0);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
        bias[c] = p.dt_bias ? ((const CT *)p.dt_bias)[d[c]] : CT(0);
        skip[c] = p.Dskip ? ((const CT *)p.Dskip)[d[c]] : CT(0);
    }
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
    for (int c = 0; c < CPT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) A2[c][i] *= CT(kLog2eD);
    for (;;) {
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            if (c > 0 && p.G > 1) row.maps(p, r, d[c] / p.Dg, n0);
            const CT u = scan_value<IO>(row.u[c], p.u.dt), pre = scan_value<IO>(row.x[c], p.u.dt) + bias[c], z = scan_value<IO>(row.z[c], p.u.dt);
            const CT dlt = p.softplus ? seq_softplus(pre) : pre, du = dlt * u;
            CT v = CT(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = n0 + i < p.N;
                h[c][i] = in ? seq_fma(seq_exp2(dlt * A2[c][i]), h[c][i], du * scan_value<IO>(row.b[i], p.u.dt)) : CT(0);
                v = seq_fma(h[c][i], in ? scan_value<IO>(row.c[i], p.u.dt) : CT(0), v);
            }
            if (p.lpc > 1) v += seq_dpp<0xb1>(v);
            if (p.lpc > 2) v += seq_dpp<0x4e>(v);
            for (int k = 4; k < p.lpc; k <<= 1) v += __shfl_xor(v, k);
            v = p.Dskip ? seq_fma(skip[c], u, v) : v;
            const CT vz = v * (z * seq_sigmoid(z));
            v = p.gate ? vz : v;
            if (sub == 0 && d0 + c * cpb < p.D) seq_store(p.y, r * (int64_t)p.y.rs + d[c], v);
        }
        if (nx < 0) break;
        r = nx;
        row.load(p, r, d, n0);
        __syncthreads();
        if (threadIdx.x == 0) next = 0x7fffffff;
        __syncthreads();
        seq_same_slot(p.slot, p.rows, r, &before, &next);
        __syncthreads();
        nx = next == 0x7fffffff ? -1 : next;
    }
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
        if (d0 + c * cpb >= p.D) continue;
        CT *o = st + (int64_t)d[c] * p.N;
        if (p.vec) {
            V4 s;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = h[c][i];
            *(V4 *)o = s;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n0 + i < p.N) o[i] = h[c][i];
        }
    }
}

}  // namespace crnn
