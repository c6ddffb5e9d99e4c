// crnn_amd/csrc/seq_capi.hpp -- the sequence operators' entry points of include/crnn_hip.h (part of crnn_capi.hip's translation unit).
// Device pointers in and out, everything enqueued on the caller's stream, workspace from the caller: a call may be captured.
#pragma once
#include "seq_common.hpp"
#include "seq_scan_kernel.hpp"
#include "seq_conv_kernel.hpp"
#include "seq_pack_kernel.hpp"

namespace {

int32_t sfail(const std::string &msg) {
    g_last_error = msg;
    return -1;
}

// the caller's device for the length of a call
struct SeqDevice {
    int prev = -1;
    bool moved = false;
    hipError_t enter(int device) {
        hipError_t e = hipGetDevice(&prev);
        if (e != hipSuccess || prev == device) return e;
        int n = 0;
        e = hipGetDeviceCount(&n);
        if (e != hipSuccess) return e;
        if (device < 0 || device >= n) return hipErrorInvalidValue;
        e = hipSetDevice(device);
        moved = e == hipSuccess;
        return e;
    }
    ~SeqDevice() {
        if (moved) (void)hipSetDevice(prev);
    }
};

int seq_size(int dt) { return dt == CRNN_DT_F64 ? 8 : dt == CRNN_DT_F32 ? 4 : dt == CRNN_DT_PACKED8 ? 1 : 2; }

crnn::SeqV seq_view(const crnn_view &v, int nvec) {
    crnn::SeqV o{};
    o.p = v.ptr;
    o.sc = (const uint8_t *)v.scales;
    o.bs = v.seq_stride; o.rs = (int32_t)v.row_stride; o.sbs = v.scale_seq_stride; o.srs = (int32_t)v.scale_row_stride;
    o.dt = v.dtype;
    const int64_t bytes = (int64_t)nvec * seq_size(v.dtype);
    o.vec = (uintptr_t)v.ptr % (uintptr_t)bytes == 0 && v.row_stride % nvec == 0 && v.seq_stride % nvec == 0;
    return o;
}

struct SeqCheck {
    const char *who;
    std::string err;
    bool bad(const std::string &what) {
        if (err.empty()) err = std::string(who) + ": " + what;
        return false;
    }
    // a view of the call's type (or, where allowed, a checkpoint); out: rows of `width` elements may not overlap (0: there is one row, its stride means nothing)
    bool view(const crnn_view &v, const char *name, int dtype, bool needed, bool packed_ok, bool out, int64_t width) {
        if (!v.ptr) return needed ? bad(std::string(name) + " is missing") : true;
        if (v.dtype == CRNN_DT_PACKED8) {
            if (!packed_ok || dtype == CRNN_DT_F64) return bad(std::string(name) + " cannot be an 8-bit checkpoint here");
            if (!v.scales) return bad(std::string(name) + ": a checkpoint needs its scales");
            if (v.scale_seq_stride < 0 || v.scale_row_stride < 0) return bad(std::string(name) + ": negative stride");
        } else if (v.dtype != dtype) return bad(std::string(name) + " has another element type than the call");
        if (v.seq_stride < 0 || v.row_stride < 0) return bad(std::string(name) + ": negative stride");
        if (v.row_stride > 0x7fffffff || v.scale_row_stride > 0x7fffffff) return bad(std::string(name) + ": rows are too far apart");
        if (out && v.row_stride < width) return bad(std::string(name) + ": rows of an output overlap");
        return true;
    }
    // an output's sequences (n of `rows` rows) may lie one behind another or row by row side by side, but not over one another
    bool apart(const crnn_view &v, const char *name, int64_t n, int64_t rows, int64_t width) {
        if (!v.ptr || n < 2 || rows < 1 || v.seq_stride >= (rows - 1) * v.row_stride + width) return true;
        if (v.seq_stride >= width && v.row_stride >= (n - 1) * v.seq_stride + width) return true;
        return bad(std::string(name) + ": sequences of an output overlap");
    }
    // an output is written while other lanes and blocks still read the inputs (the pointers alone; what else they may share: SeqShare)
    bool other(std::initializer_list<const crnn_view *> outs, std::initializer_list<const crnn_view *> ins, int64_t rows) {
        for (const crnn_view *y : outs)
            for (const crnn_view *x : ins)
                if (rows > 0 && y->ptr && y->ptr == x->ptr) return bad("an output is also an input");
        return true;
    }
};

// Where an array lies: `width` bytes, `n[0]` times `s[0]` bytes apart, all that `n[1]` times `s[1]` bytes apart (s[0] <= s[1]).
struct SeqSpan {
    uintptr_t at = 0;
    int64_t width = 0, n[2] = {0, 0}, s[2] = {0, 0};
    SeqSpan() = default;
    SeqSpan(const void *p, int64_t bytes) : SeqSpan(p, bytes, 1, 0, 1, 0) {}
    SeqSpan(const void *p, int64_t bytes, int64_t rows, int64_t row_bytes, int64_t seqs, int64_t seq_bytes) {
        if (!p || bytes <= 0 || rows <= 0 || seqs <= 0) return;
        at = (uintptr_t)p; width = bytes;
        n[0] = row_bytes ? rows : 1; s[0] = n[0] > 1 ? row_bytes : 0;
        n[1] = seq_bytes ? seqs : 1; s[1] = n[1] > 1 ? seq_bytes : 0;
        if (n[0] == 1 || (n[1] > 1 && s[1] < s[0])) { std::swap(n[0], n[1]); std::swap(s[0], s[1]); }
    }
    __int128 end() const { return (__int128)at + (__int128)(n[0] - 1) * s[0] + (__int128)(n[1] - 1) * s[1] + width; }
    bool one(int k) const { return n[k] <= 1; }
};
// a and b, each pieces of `wa` and `wb` bytes some multiples of `every` bytes apart, never meet
inline bool seq_beside(const SeqSpan &a, const SeqSpan &b, __int128 wa, __int128 wb, int64_t every) {
    if (every <= 0) return false;
    const int64_t d = (int64_t)((((__int128)b.at - (__int128)a.at) % every + every) % every);
    return d >= wa && d + wb <= every;
}
// Arrays whose ranges of addresses meet are still apart where both are columns of one wider array (row by row side by side), or blocks of rows side by side.
// What else meets counts as shared.
inline bool seq_shared(const SeqSpan &a, const SeqSpan &b) {
    if (!a.at || !b.at || a.end() <= (__int128)b.at || b.end() <= (__int128)a.at) return false;
    const int64_t in = a.one(0) ? b.s[0] : a.s[0], out = a.one(1) ? b.s[1] : a.s[1];
    const bool rows = (a.one(0) || a.s[0] == in) && (b.one(0) || b.s[0] == in) && in > 0 && a.s[1] % in == 0 && b.s[1] % in == 0;
    if (rows && seq_beside(a, b, a.width, b.width, in)) return false;
    const bool blocks = (a.one(1) || a.s[1] == out) && (b.one(1) || b.s[1] == out);
    const __int128 wa = (__int128)(a.n[0] - 1) * a.s[0] + a.width, wb = (__int128)(b.n[0] - 1) * b.s[0] + b.width;
    return !(blocks && seq_beside(a, b, wa, wb, out));
}
// The arrays of a call.  Outputs may share memory neither with inputs nor with one another; `same`: an input that an output may be, as a whole
// (each of its elements is read by the thread that writes it, before).
struct SeqShare {
    SeqSpan ins[16], outs[10];
    int n_in = 0, n_out = 0;
    void put_in(const SeqSpan &x) { if (x.at) ins[n_in++] = x; }
    void put_out(const SeqSpan &x) { if (x.at) outs[n_out++] = x; }
    // rows of `width` elements
    static SeqSpan span(const crnn_view &v, int64_t width, int64_t rows, int64_t n) {
        const int64_t e = seq_size(v.dtype);
        return SeqSpan(v.ptr, width * e, rows, v.row_stride * e, n, v.seq_stride * e);
    }
    void in(const crnn_view &v, int64_t width, int64_t rows, int64_t n) {
        put_in(span(v, width, rows, n));
        if (v.ptr && v.dtype == CRNN_DT_PACKED8) put_in(SeqSpan(v.scales, (width + 31) / 32, rows, v.scale_row_stride, n, v.scale_seq_stride));
    }
    void in(const void *p, int64_t bytes) { put_in(SeqSpan(p, bytes)); }
    void out(const crnn_view &v, int64_t width, int64_t rows, int64_t n) { put_out(span(v, width, rows, n)); }
    void out(const void *p, int64_t bytes) { put_out(SeqSpan(p, bytes)); }
    bool ok(SeqCheck &c, const void *same = nullptr, const void *same2 = nullptr) const {
        for (int i = 0; i < n_out; ++i) {
            const SeqSpan &y = outs[i];
            for (int j = 0; j < n_in; ++j)
                if (seq_shared(y, ins[j]) && !(y.at == ins[j].at && (y.at == (uintptr_t)same || y.at == (uintptr_t)same2))) return c.bad("an output shares memory with an input");
            for (int j = 0; j < i; ++j)
                if (seq_shared(y, outs[j])) return c.bad("two outputs share memory");
        }
        return true;
    }
};

bool seq_rows_ok(SeqCheck &c, int32_t n_seq, int64_t rows, const int32_t *start, const int32_t *len, int32_t D, int32_t dtype) {
    if (n_seq < 0 || rows < 0) return c.bad("negative number of sequences or rows");
    if (rows > 0x7fffffc0LL) return c.bad("more than 2^31 - 64 rows");
    if (start && len) return c.bad("seq_start and seq_len exclude each other");
    if (D < 1 || D > (1 << 24)) return c.bad("D must be in 1 .. 2^24");
    if (dtype < CRNN_DT_F32 || dtype > CRNN_DT_F64) return c.bad("unknown element type");
    return true;
}

// chunks of Q rows; Q <= 0: one chunk a sequence
crnn::SeqMap seq_map(int32_t n_seq, int64_t rows, const int32_t *start, const int32_t *len, int64_t Q) {
    crnn::SeqMap m{};
    m.start = start; m.len = len; m.rows = rows; m.n_seq = n_seq;
    m.Q = Q > 0 ? Q : rows + 1;
    m.nch = rows > 0 ? (rows + m.Q - 1) / m.Q : 1;
    m.nblk = start ? rows / m.Q + n_seq : m.nch * n_seq;
    m.per = m.nblk > 0 ? (rows + m.nblk - 1) / m.nblk : 0;
    return m;
}
int64_t seq_flat(int32_t n_seq, int64_t rows, bool packed) { return packed ? rows : rows * n_seq; }
// Blocks of 256 threads a launch may have: the hardware counts threads in 32 bits, and a larger grid is cut off without an error (524296 x 32 blocks ran as 256)
constexpr int64_t kSeqMaxGrid = 0xffffffffLL / 256;
constexpr int64_t kSeqMaxChunks = 0x7fffffff;      // chunks are counted in 31 bits on the device

#define SEQ_ENTER(a, who)                                                                                                   \
    if (!(a)) return sfail(who ": null arguments");                                                                          \
    if ((a)->struct_size != (int32_t)sizeof(*(a))) return sfail(who ": struct_size does not match this library's struct");
#define SEQ_DEVICE(device, who)                                                                                             \
    SeqDevice guard;                                                                                                         \
    {                                                                                                                        \
        const hipError_t e_ = guard.enter(device);                                                                           \
        if (e_ != hipSuccess) return sfail(std::string(who ": device: ") + hipGetErrorString(e_));                           \
    }
#define SEQ_DONE(who)                                                                                                       \
    do {                                                                                                                     \
        const hipError_t e_ = hipGetLastError();                                                                             \
        if (e_ != hipSuccess) return sfail(std::string(who ": ") + hipGetErrorString(e_));                                   \
        return 0;                                                                                                            \
    } while (0)

// ------------------------------------------------------------------ scan
struct ScanPlan {
    bool f64, p8, split;
    int mode;                   // the kernels' MODE
    int NS, nb;                 // states of a launch, launches over the states
    int64_t flat;
    crnn::ScanP p;
    // workspace, in elements of the compute type
    int64_t S, G, sdel, part, dA, acc, total;
};

// Rows of a chunk of the forward scan; 0: sequences are not cut.  Cutting costs a second look at all but a sequence's last chunk and two launches; a
// block alone takes 0.18 us a row.  So short sequences stay whole, and so do a dense batch's where they give every SIMD a wavefront; packed ones are cut
// even then, since their lengths are not known here.  Else chunks are as long as they still fill the card.  Measured (bf16, 16 states; sequences x
// rows x channels: us a call at 16 / 32 / 64 / 128 / 512 rows a chunk, whole): 1 x 64 x 1536 - / 27 / 26 / 27 / 26, 18; 1 x 256 x 1536 25 / 25 / 32 / 50 / 57, 52;
// 1 x 512 x 4096 45 / 38 / 39 / 51 / 104, 98; 1 x 2048 x 2048 73 / 59 / 56 / 61 / 161, 375; 1 x 16384 x 1024 285 / 191 / 156 / 143 / 189, 2952; 9 x 910 x 4096 422 /
// 291 / 253 / 248 / 294, 486; 8 x 1024 x 4096 415 / 286 / 249 / 232 / 242, 224; 32 x 512 x 4096 773 / 558 / 488 / 447 / 319, 289.
int64_t scan_forward_rows(int64_t flat, int32_t n_seq, int64_t rows, bool packed, int64_t ntile) {
    if (rows <= 64) return 0;                      // (packed: no sequence has more)
    const bool many = (int64_t)n_seq * ntile >= 1024;
    if (many && !packed) return 0;
    const int64_t total = flat * ntile;
    const int64_t q = many ? 512 : total <= 8192 ? 16 : total <= 49152 ? 32 : total <= 131072 ? 64 : 128;
    return std::max(q, (total / 8192 + 7) / 8 * 8);
}

// step: only what a single row has to do with (its launch is checked by itself)
bool scan_plan(SeqCheck &c, const crnn_scan_args *a, bool backward, ScanPlan &s, bool step = false) {
    if (!seq_rows_ok(c, a->n_seq, a->rows, a->seq_start, a->seq_len, a->D, a->dtype)) return false;
    if (a->N < 1 || a->N > CRNN_SEQ_MAX_STATES) return c.bad("N must be in 1 .. 256");
    if (a->G < 1 || a->D % a->G) return c.bad("G must divide D");
    s.f64 = a->dtype == CRNN_DT_F64;
    const bool pu = a->u.dtype == CRNN_DT_PACKED8, pz = a->z.ptr ? a->z.dtype == CRNN_DT_PACKED8 : pu;
    s.p8 = pu || (a->z.ptr && pz);
    s.mode = s.f64 || a->N > 16 || pu != pz ? crnn::kScanAny : pu ? 1 : 0;
    s.NS = s.f64 || (s.mode != crnn::kScanAny && a->N <= 8) ? 8 : 16;
    s.nb = (a->N + s.NS - 1) / s.NS;
    s.flat = seq_flat(a->n_seq, a->rows, a->seq_start != nullptr);
    crnn::ScanP &p = s.p;
    p = crnn::ScanP{};
    p.D = a->D; p.N = a->N; p.G = a->G; p.Dg = a->D / a->G;
    p.tpg = (p.Dg + 63) / 64;
    p.ntile = p.tpg * a->G;
    const int64_t Q = backward ? crnn::kScanBwdQ : scan_forward_rows(s.flat, a->n_seq, a->rows, a->seq_start != nullptr, p.ntile);
    p.m = seq_map(a->n_seq, a->rows, a->seq_start, a->seq_len, Q);
    s.split = backward || Q > 0;
    const int64_t blk = p.m.nblk * a->D;
    const int64_t tiles = backward ? (p.ntile + crnn::kScanWaves - 1) / crnn::kScanWaves : p.ntile;
    if (!step && (p.m.nblk > kSeqMaxChunks || p.m.nblk * tiles > kSeqMaxGrid || (s.split && ((int64_t)a->n_seq * s.NS * a->D + 255) / 256 > kSeqMaxGrid)))
        return c.bad("too many sequences, rows and channels for one launch");
    int64_t at = 0;
    auto take = [&](int64_t n) { const int64_t o = at; at += (n + 31) / 32 * 32; return o; };
    s.S = take(s.split ? blk * s.NS : 0);
    s.sdel = take(s.split ? blk : 0);
    s.G = take(backward ? blk * s.NS : 0);
    s.part = take(backward ? (int64_t)p.ntile * s.flat * 2 * s.NS : 0);
    s.dA = take(backward ? blk * (s.NS + 2) : 0);
    s.acc = take(s.nb > 1 ? s.flat * a->D * (backward ? 3 : 1) : 0);
    s.total = at * (s.f64 ? 8 : 4);
    return true;
}

void scan_fill(const crnn_scan_args *a, ScanPlan &s) {
    crnn::ScanP &p = s.p;
    p.u = seq_view(a->u, 4); p.dt = seq_view(a->dt, 4); p.z = seq_view(a->z, 4); p.y = seq_view(a->y, 4);
    p.gate = a->z.ptr != nullptr;
    if (!p.gate) p.z = p.u;
    p.dy = seq_view(a->dy, 4); p.du = seq_view(a->du, 4); p.ddt = seq_view(a->ddt, 4); p.dz = seq_view(a->dz, 4);
    p.B = seq_view(a->B, 1); p.C = seq_view(a->C, 1);
    p.Bg = a->B_group; p.Bn = a->B_state; p.Cg = a->C_group; p.Cn = a->C_state;
    p.A = a->A; p.Dskip = a->skip; p.dt_bias = a->dt_bias;
    p.state_in = a->state_in; p.state_out = a->state_out; p.dstate_out = a->dstate_out; p.dstate_in = a->dstate_in;
    p.softplus = a->softplus; p.zero_outside = a->zero_outside;
    p.acc_n = s.flat;
    p.nvec = a->N % 4 == 0 && (uintptr_t)a->A % 16 == 0 && (uintptr_t)a->state_in % 16 == 0;
}
crnn::ScanMapsP scan_maps(const crnn_scan_args *a, const ScanPlan &s, const crnn_view &B, const crnn_view &C, int64_t Bg, int64_t Bn, int64_t Cg, int64_t Cn) {
    crnn::ScanMapsP m{};
    m.B = seq_view(B, 1); m.C = seq_view(C, 1);
    m.Bg = Bg; m.Cg = Cg; m.Bn = Bn; m.Cn = Cn;
    m.rows = s.flat;
    m.srows = a->seq_start ? 0 : a->rows;
    m.G = a->G; m.N = a->N;
    m.zero_outside = a->zero_outside;
    return m;
}

unsigned seq_grid(int64_t n) { return (unsigned)std::min<int64_t>((n + 255) / 256, 65536); }

template <int IO, int NS, int MODE>
void scan_forward_run(const crnn_scan_args *a, ScanPlan &s, hipStream_t st) {
    using CT = typename crnn::SeqIO<IO>::C;
    crnn::ScanP p = s.p;
    CT *ws = (CT *)a->workspace, *S = ws + s.S, *sdel = ws + s.sdel;
    p.acc = s.nb > 1 ? ws + s.acc : nullptr;
    const dim3 grid((unsigned)(p.m.nblk * p.ntile)), block(64 * crnn::kScanWaves);
    for (int b = 0; b < s.nb; ++b) {
        p.n0 = b * NS;
        p.first = b == 0;
        p.fin = b == s.nb - 1;
        if (s.split) {
            hipLaunchKernelGGL((crnn::seq_scan_fwd_kernel<IO, NS, MODE, false, false>), grid, block, 0, st, p, (const CT *)nullptr, S, sdel);
            hipLaunchKernelGGL((crnn::seq_scan_carry_kernel<CT, NS>), dim3((unsigned)(((int64_t)p.m.n_seq * NS * p.D + 255) / 256)), dim3(256), 0, st, p, S,
                               (CT *)nullptr, (const CT *)sdel);
        }
        const CT *start = s.split ? S : nullptr;
        if (p.n0 + NS <= p.N) hipLaunchKernelGGL((crnn::seq_scan_fwd_kernel<IO, NS, MODE, true, false>), grid, block, 0, st, p, start, (CT *)nullptr, (CT *)nullptr);
        else hipLaunchKernelGGL((crnn::seq_scan_fwd_kernel<IO, NS, MODE, true, true>), grid, block, 0, st, p, start, (CT *)nullptr, (CT *)nullptr);
    }
}

template <int IO, int NS, int MODE>
void scan_backward_run(const crnn_scan_args *a, ScanPlan &s, hipStream_t st) {
    using CT = typename crnn::SeqIO<IO>::C;
    crnn::ScanP p = s.p;
    CT *ws = (CT *)a->workspace, *S = ws + s.S, *Gb = ws + s.G, *sdel = ws + s.sdel, *part = ws + s.part, *pp = ws + s.dA;
    p.acc = s.nb > 1 ? ws + s.acc : nullptr;
    const dim3 grid((unsigned)(p.m.nblk * ((p.ntile + crnn::kScanWaves - 1) / crnn::kScanWaves))), block(64 * crnn::kScanWaves);
    crnn::ScanMapsP mo = scan_maps(a, s, a->dB, a->dC, a->N, 1, a->N, 1);
    const int64_t cA = (int64_t)(NS + 2) * p.D;      // dA's states, then the gradients of the skip and of the step lengths' bias
    for (int b = 0; b < s.nb; ++b) {
        p.n0 = mo.n0 = b * NS;
        p.first = b == 0;
        p.fin = b == s.nb - 1;
        hipLaunchKernelGGL((crnn::seq_scan_ends2_kernel<IO, NS, MODE>), grid, block, 0, st, p, S, Gb, sdel);
        hipLaunchKernelGGL((crnn::seq_scan_carry_kernel<CT, NS>), dim3((unsigned)(((int64_t)p.m.n_seq * NS * p.D + 255) / 256)), dim3(256), 0, st, p, S, Gb,
                           (const CT *)sdel);
        if (p.n0 + NS <= p.N) hipLaunchKernelGGL((crnn::seq_scan_bwd_kernel<IO, NS, MODE, false>), grid, block, 0, st, p, (const CT *)S, (const CT *)Gb, part, pp);
        else hipLaunchKernelGGL((crnn::seq_scan_bwd_kernel<IO, NS, MODE, true>), grid, block, 0, st, p, (const CT *)S, (const CT *)Gb, part, pp);
        if (s.flat > 0)
            hipLaunchKernelGGL((crnn::seq_scan_sum_maps_kernel<CT, NS>), dim3(seq_grid(s.flat * p.G * 2 * NS)), dim3(256), 0, st, p.m, mo, (const CT *)part, p.tpg);
        hipLaunchKernelGGL((crnn::seq_sum_blocks_kernel<CT>), dim3((unsigned)((cA + 31) / 32)), dim3(256), 0, st, (const CT *)pp, p.m.nblk, cA, (CT *)a->dA,
                           (CT *)(p.fin ? a->dskip : nullptr), (CT *)(p.fin ? a->ddt_bias : nullptr), p.D, p.N, p.n0, std::min(NS, p.N - p.n0), NS);
    }
}

// (the arrays of a step have one row a sequence, row_stride apart)
bool scan_views(SeqCheck &c, const crnn_scan_args *a, bool backward, bool step = false) {
    const int dt = a->dtype;
    const int64_t D = a->D, GN = (int64_t)a->G * a->N;
    if (!a->A) return c.bad("A is missing");
    if (!c.view(a->u, "u", dt, true, true, false, D) || !c.view(a->dt, "dt", dt, true, false, false, D) || !c.view(a->z, "z", dt, false, true, false, D) ||
        !c.view(a->B, "B", dt, true, false, false, 0) || !c.view(a->C, "C", dt, true, false, false, 0))
        return false;
    if (a->B_group < 0 || a->B_state < 0 || a->C_group < 0 || a->C_state < 0) return c.bad("negative stride of B or C");
    const int64_t n = a->seq_start || step ? 1 : a->n_seq, rows = a->rows, flat = step ? a->n_seq : seq_flat(a->n_seq, rows, a->seq_start != nullptr);
    const bool many = (step ? a->n_seq : rows) > 1;
    const int64_t Dw = many ? D : 0, GNw = many ? GN : 0;
    if (!backward)
        return c.view(a->y, "y", dt, true, false, true, Dw) && c.apart(a->y, "y", n, rows, D) && c.other({&a->y}, {&a->u, &a->dt, &a->z, &a->B, &a->C}, flat);
    if (!a->dA) return c.bad("dA is missing");
    if ((a->z.ptr != nullptr) != (a->dz.ptr != nullptr)) return c.bad("dz goes with z");
    return c.view(a->dy, "dy", dt, true, false, false, D) && c.view(a->du, "du", dt, true, false, true, Dw) && c.view(a->ddt, "ddt", dt, true, false, true, Dw) &&
           c.view(a->dz, "dz", dt, false, false, true, Dw) && c.view(a->dB, "dB", dt, true, false, true, GNw) && c.view(a->dC, "dC", dt, true, false, true, GNw) &&
           c.apart(a->du, "du", n, rows, D) && c.apart(a->ddt, "ddt", n, rows, D) && c.apart(a->dz, "dz", n, rows, D) && c.apart(a->dB, "dB", n, rows, GN) &&
           c.apart(a->dC, "dC", n, rows, GN) && c.other({&a->du, &a->ddt, &a->dz, &a->dB, &a->dC}, {&a->dy, &a->u, &a->dt, &a->z, &a->B, &a->C}, flat);
}

bool scan_apart(SeqCheck &c, const crnn_scan_args *a, bool backward, bool step = false) {
    SeqShare m;
    const int64_t pe = a->dtype == CRNN_DT_F64 ? 8 : 4, D = a->D, N = a->N, G = a->G;
    const int64_t rows = step ? a->n_seq : a->rows, n = step || a->seq_start ? 1 : a->n_seq, states = (step ? a->n_slots : (int64_t)a->n_seq) * D * N * pe;
    m.in(a->u, D, rows, n); m.in(a->dt, D, rows, n); m.in(a->z, D, rows, n);
    m.in(a->B, (G - 1) * a->B_group + (N - 1) * a->B_state + 1, rows, n); m.in(a->C, (G - 1) * a->C_group + (N - 1) * a->C_state + 1, rows, n);
    m.in(a->A, D * N * pe); m.in(a->skip, D * pe); m.in(a->dt_bias, D * pe);
    m.in(a->seq_start, ((int64_t)a->n_seq + 1) * 4); m.in(a->seq_len, (int64_t)a->n_seq * 4);
    if (step) {
        m.in(a->slot, (int64_t)a->n_seq * 4);
        m.out(a->y, D, rows, n); m.out(a->state_out, states);
        return m.ok(c);
    }
    m.in(a->state_in, states);
    if (!backward) {
        m.out(a->y, D, rows, n); m.out(a->state_out, states);
        return m.ok(c, a->state_in);
    }
    m.in(a->dy, D, rows, n); m.in(a->dstate_out, states);
    m.out(a->du, D, rows, n); m.out(a->ddt, D, rows, n); m.out(a->dz, D, rows, n); m.out(a->dB, G * N, rows, n); m.out(a->dC, G * N, rows, n);
    m.out(a->dA, D * N * pe); m.out(a->dskip, D * pe); m.out(a->ddt_bias, D * pe); m.out(a->dstate_in, states);
    return m.ok(c, a->state_in, a->dstate_out);
}

// the launches' template: MODE 2 (anything: several launches over the states, one of u and z a checkpoint) has 16 states a launch, 8 in double
#define SCAN_RUN(run)                                                                                                         \
    do {                                                                                                                      \
        const hipStream_t st_ = (hipStream_t)a->stream;                                                                       \
        if (s.f64) run<8, 8, 2>(a, s, st_);                                                                                   \
        else if (a->dtype == CRNN_DT_F32) SCAN_RUN_IO(run, 4);                                                                \
        else SCAN_RUN_IO(run, 2);                                                                                             \
    } while (0)
#define SCAN_RUN_IO(run, IO)                                                                                                  \
    do {                                                                                                                      \
        if (s.mode == 2) run<IO, 16, 2>(a, s, st_);                                                                           \
        else if (s.NS == 8) { if (s.mode) run<IO, 8, 1>(a, s, st_); else run<IO, 8, 0>(a, s, st_); }                           \
        else { if (s.mode) run<IO, 16, 1>(a, s, st_); else run<IO, 16, 0>(a, s, st_); }                                        \
    } while (0)

// ------------------------------------------------------------------ convolution
// channels of a thread, one where an array of the call does not allow more.  Four of two bytes beat eight (12001 x 4096, W = 4: 37 against 41 us):
// half the registers are twice the wavefronts.
int conv_wide(int dtype, int W, bool backward) {
    if (dtype == CRNN_DT_F64) return 2;
    if (dtype == CRNN_DT_F32) return W > 4 && backward ? 2 : 4;
    return 4;
}
// Rows of a strip: strips and channels together give some wavefronts to each SIMD; a strip reads W - 1 rows twice, the gradient 2 (W - 1).
// Measured, bf16 (us a call at 8 / 16 / 24 / 32 / 48 / 64 / 128 rows): forward 12001 x 4096 43 / 36 / 38 / 39 / 40 / 40 / 42, 1024 x 2048 12 / 12 / 12 / 12 / 13 /
// 16 / 26; gradient 8192 x 2048 from 8 bits 60 / 46 / 39 / 42 / 41 / 48 / 56, 12000 x 4096 148 / 99 / 83 / 80 / 72 / 71 / 83, 1024 x 2048 23 / 23 / 23 / 23 / 27 / 31 / 51.
int64_t conv_strip(int64_t flat, int32_t D, int V, bool backward) {
    const int64_t waves = (D + 64 * V - 1) / (64 * V);
    const int64_t q = (flat * waves / 4096 + 3) / 4 * 4;
    const int64_t lo = backward ? 24 : 8, hi = backward ? 64 : 16;
    return q < lo ? lo : q > hi ? hi : q;
}
bool conv_fits(const crnn_view &v, int V) { return !v.ptr || seq_view(v, V).vec; }
bool conv_weights_fit(const crnn_conv_args *a, int V) {
    const uintptr_t b = (uintptr_t)V * (a->dtype == CRNN_DT_F64 ? 8 : 4);
    return (uintptr_t)a->weight % b == 0 && (uintptr_t)a->bias % b == 0;
}
int conv_channels(const crnn_conv_args *a, bool backward) {
    const int V = conv_wide(a->dtype, a->W, backward);
    const bool fits = a->D % V == 0 && conv_weights_fit(a, V) && conv_fits(a->x, V) && conv_fits(a->y, V) && conv_fits(a->state_in, V) && conv_fits(a->state_out, V) && conv_fits(a->dy, V) &&
                      conv_fits(a->dx, V) && conv_fits(a->dstate_out, V) && conv_fits(a->dstate_in, V);
    return fits ? V : 1;
}
// chunks do not depend on V (the workspace is asked for before the arrays are known)
bool conv_check(SeqCheck &c, const crnn_conv_args *a, bool backward, crnn::ConvP &p) {
    if (!seq_rows_ok(c, a->n_seq, a->rows, a->seq_start, a->seq_len, a->D, a->dtype)) return false;
    if (a->W < 1 || a->W > CRNN_SEQ_MAX_TAPS) return c.bad("W must be in 1 .. 8");
    p = crnn::ConvP{};
    p.D = a->D; p.W = a->W; p.silu = a->silu; p.zero_outside = a->zero_outside;
    p.m = seq_map(a->n_seq, a->rows, a->seq_start, a->seq_len,
                  conv_strip(seq_flat(a->n_seq, a->rows, a->seq_start != nullptr), a->D, conv_wide(a->dtype, a->W, backward), backward));
    if (p.m.nblk > kSeqMaxChunks) return c.bad("too many sequences, rows and channels for one launch");
    return true;
}
bool conv_views(SeqCheck &c, const crnn_conv_args *a, bool backward, crnn::ConvP &p) {
    const int dt = a->dtype;
    if (!a->weight) return c.bad("weight is missing");
    const int64_t n = a->seq_start ? 1 : a->n_seq, flat = seq_flat(a->n_seq, a->rows, a->seq_start != nullptr);
    const int64_t Dw = a->rows > 1 ? a->D : 0, Sw = a->W > 2 ? a->D : 0;
    if (!c.view(a->x, "x", dt, true, true, false, a->D) || !c.view(a->state_in, "state_in", dt, false, false, false, a->D)) return false;
    if (backward) {
        if (!a->dweight) return c.bad("dweight is missing");
        if (!c.view(a->dy, "dy", dt, true, false, false, a->D) || !c.view(a->dx, "dx", dt, true, false, true, Dw) ||
            !c.view(a->dstate_out, "dstate_out", dt, false, false, false, a->D) || !c.view(a->dstate_in, "dstate_in", dt, false, false, true, Sw) ||
            !c.apart(a->dx, "dx", n, a->rows, a->D) || !c.apart(a->dstate_in, "dstate_in", a->n_seq, a->W - 1, a->D) || !c.other({&a->dx}, {&a->x, &a->dy}, flat))
            return false;
    } else {
        if (!c.view(a->y, "y", dt, true, false, true, Dw) || !c.view(a->state_out, "state_out", dt, false, false, true, Sw) ||
            !c.apart(a->y, "y", n, a->rows, a->D) || !c.apart(a->state_out, "state_out", a->n_seq, a->W - 1, a->D) || !c.other({&a->y}, {&a->x}, flat))
            return false;
        if (a->state_out.ptr && a->state_out.ptr == a->state_in.ptr) return c.bad("state_out may not be state_in");
    }
    p.x = seq_view(a->x, 1); p.y = seq_view(a->y, 1); p.dy = seq_view(a->dy, 1); p.dx = seq_view(a->dx, 1);
    p.st_in = seq_view(a->state_in, 1); p.st_out = seq_view(a->state_out, 1); p.dst_out = seq_view(a->dstate_out, 1); p.dst_in = seq_view(a->dstate_in, 1);
    p.w = a->weight; p.bias = a->bias;
    return true;
}
bool conv_apart(SeqCheck &c, const crnn_conv_args *a, bool backward, bool step = false) {
    SeqShare m;
    const int64_t pe = a->dtype == CRNN_DT_F64 ? 8 : 4, D = a->D, W = a->W, rows = step ? a->n_seq : a->rows, n = step || a->seq_start ? 1 : a->n_seq;
    m.in(a->x, D, rows, n); m.in(a->weight, D * W * pe); m.in(a->bias, D * pe);
    m.in(a->seq_start, ((int64_t)a->n_seq + 1) * 4); m.in(a->seq_len, (int64_t)a->n_seq * 4);
    if (step) {
        m.in(a->slot, (int64_t)a->n_seq * 4);
        m.out(a->y, D, rows, n); m.out(a->state_in, D, W - 1, a->n_slots);
        return m.ok(c);
    }
    m.in(a->state_in, D, W - 1, a->n_seq);
    if (!backward) {
        m.out(a->y, D, rows, n); m.out(a->state_out, D, W - 1, a->n_seq);
        return m.ok(c);
    }
    m.in(a->dy, D, rows, n); m.in(a->dstate_out, D, W - 1, a->n_seq);
    m.out(a->dx, D, rows, n); m.out(a->dstate_in, D, W - 1, a->n_seq); m.out(a->dweight, D * W * pe); m.out(a->dbias, D * pe);
    return m.ok(c);
}
int64_t conv_grid(const crnn::ConvP &p, int V) { return (p.m.nblk + 3) / 4 * ((p.D + 64 * V - 1) / (64 * V)); }
template <int XT, int YT, int W, int V>
void conv_launch(const crnn::ConvP &p, bool backward, hipStream_t st) {
    const dim3 grid((unsigned)conv_grid(p, V));
    if (backward) hipLaunchKernelGGL((crnn::seq_conv_bwd_kernel<XT, YT, W, V>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((crnn::seq_conv_fwd_kernel<XT, YT, W, V>), grid, dim3(256), 0, st, p);
}
// VF, VB: the wide forms' channels forward and backward (conv_wide)
template <int XT, int YT, int W, int VF, int VB>
void conv_launch_v(const crnn::ConvP &p, int V, bool backward, hipStream_t st) {
    if (V == 1) conv_launch<XT, YT, W, 1>(p, backward, st);
    else if (backward) conv_launch<XT, YT, W, VB>(p, true, st);
    else conv_launch<XT, YT, W, VF>(p, false, st);
}
// VB8: the gradient's channels from five taps on
template <int XT, int YT, int VF, int VB, int VB8>
void conv_launch_w(const crnn::ConvP &p, int V, bool backward, hipStream_t st) {
    switch (p.W) {
        case 1: return conv_launch_v<XT, YT, 1, VF, VB>(p, V, backward, st);
        case 2: return conv_launch_v<XT, YT, 2, VF, VB>(p, V, backward, st);
        case 3: return conv_launch_v<XT, YT, 3, VF, VB>(p, V, backward, st);
        case 4: return conv_launch_v<XT, YT, 4, VF, VB>(p, V, backward, st);
        case 5: return conv_launch_v<XT, YT, 5, VF, VB8>(p, V, backward, st);
        case 6: return conv_launch_v<XT, YT, 6, VF, VB8>(p, V, backward, st);
        case 7: return conv_launch_v<XT, YT, 7, VF, VB8>(p, V, backward, st);
        default: return conv_launch_v<XT, YT, 8, VF, VB8>(p, V, backward, st);
    }
}
template <int YT>
void conv_launch_x(const crnn::ConvP &p, int V, bool backward, hipStream_t st) {
    constexpr int VB8 = YT == CRNN_DT_F32 ? 2 : 4;
    if (p.x.dt == CRNN_DT_PACKED8) conv_launch_w<CRNN_DT_PACKED8, YT, 4, 4, VB8>(p, V, backward, st);
    else conv_launch_w<YT, YT, 4, 4, VB8>(p, V, backward, st);
}
void conv_launch_t(const crnn::ConvP &p, int dtype, int V, bool backward, hipStream_t st) {
    if (dtype == CRNN_DT_F64) conv_launch_w<CRNN_DT_F64, CRNN_DT_F64, 2, 2, 2>(p, V, backward, st);
    else if (dtype == CRNN_DT_F32) conv_launch_x<CRNN_DT_F32>(p, V, backward, st);
    else if (dtype == CRNN_DT_BF16) conv_launch_x<CRNN_DT_BF16>(p, V, backward, st);
    else conv_launch_x<CRNN_DT_F16>(p, V, backward, st);
}
template <int YT, int W, int V>
void conv_step_launch(const crnn::ConvStepP &p, hipStream_t st) {
    const int64_t gx = (p.D + 256 * V - 1) / (256 * V);
    hipLaunchKernelGGL((crnn::seq_conv_step_kernel<YT, W, V>), dim3((unsigned)(p.rows * gx)), dim3(256), 0, st, p);
}
// (four channels of a thread at most: the rows are few, the wavefronts should not be)
template <int YT>
void conv_step_launch_w(const crnn::ConvStepP &p, int V, hipStream_t st) {
    constexpr int VW = YT == CRNN_DT_F64 ? 2 : 4;
    auto run = [&](auto w) {
        constexpr int W = decltype(w)::value;
        if (V == 1) conv_step_launch<YT, W, 1>(p, st);
        else conv_step_launch<YT, W, VW>(p, st);
    };
    switch (p.W) {
        case 1: return run(std::integral_constant<int, 1>{});
        case 2: return run(std::integral_constant<int, 2>{});
        case 3: return run(std::integral_constant<int, 3>{});
        case 4: return run(std::integral_constant<int, 4>{});
        case 5: return run(std::integral_constant<int, 5>{});
        case 6: return run(std::integral_constant<int, 6>{});
        case 7: return run(std::integral_constant<int, 7>{});
        default: return run(std::integral_constant<int, 8>{});
    }
}

}  // namespace

extern "C" {

int64_t crnn_conv_workspace(const crnn_conv_args *a) {
    try {
        SEQ_ENTER(a, "crnn_conv_workspace");
        SeqCheck c{"crnn_conv_workspace", {}};
        crnn::ConvP p;
        if (!conv_check(c, a, true, p)) return sfail(c.err);
        return p.m.nblk * (a->W + 1) * a->D * (a->dtype == CRNN_DT_F64 ? 8 : 4);
    } catch (...) { return -1; }
}

int32_t crnn_conv_forward(const crnn_conv_args *a) {
    try {
        SEQ_ENTER(a, "crnn_conv_forward");
        SeqCheck c{"crnn_conv_forward", {}};
        crnn::ConvP p;
        if (!conv_check(c, a, false, p)) return sfail(c.err);
        if (a->n_seq == 0) return 0;
        if (!conv_views(c, a, false, p) || !conv_apart(c, a, false)) return sfail(c.err);
        const int V = conv_channels(a, false);
        if (conv_grid(p, V) > kSeqMaxGrid) return sfail("crnn_conv_forward: too many sequences, rows and channels for one launch");
        SEQ_DEVICE(a->device, "crnn_conv_forward");
        conv_launch_t(p, a->dtype, V, false, (hipStream_t)a->stream);
        SEQ_DONE("crnn_conv_forward");
    } catch (...) { return -1; }
}

int32_t crnn_conv_backward(const crnn_conv_args *a) {
    try {
        SEQ_ENTER(a, "crnn_conv_backward");
        SeqCheck c{"crnn_conv_backward", {}};
        crnn::ConvP p;
        if (!conv_check(c, a, true, p) || !conv_views(c, a, true, p)) return sfail(c.err);
        if (a->n_seq == 0) return sfail("crnn_conv_backward: no sequences");
        const bool f64 = a->dtype == CRNN_DT_F64;
        const int64_t need = p.m.nblk * (a->W + 1) * a->D * (f64 ? 8 : 4);
        if (need > 0 && (!a->workspace || a->workspace_bytes < need)) return sfail("crnn_conv_backward: workspace is missing or too small");
        if (!conv_apart(c, a, true)) return sfail(c.err);
        const int V = conv_channels(a, true);
        if (conv_grid(p, V) > kSeqMaxGrid) return sfail("crnn_conv_backward: too many sequences, rows and channels for one launch");
        SEQ_DEVICE(a->device, "crnn_conv_backward");
        p.part = a->workspace;
        const hipStream_t st = (hipStream_t)a->stream;
        conv_launch_t(p, a->dtype, V, true, st);
        const int64_t count = (int64_t)(a->W + 1) * a->D;       // [tap][D], then the bias
        const dim3 grid((unsigned)((count + 31) / 32));
        if (f64)
            hipLaunchKernelGGL((crnn::seq_sum_blocks_kernel<double>), grid, dim3(256), 0, st, (const double *)p.part, p.m.nblk, count, (double *)a->dweight, (double *)a->dbias,
                               (double *)nullptr, a->D, a->W, 0, a->W, a->W);
        else
            hipLaunchKernelGGL((crnn::seq_sum_blocks_kernel<float>), grid, dim3(256), 0, st, (const float *)p.part, p.m.nblk, count, (float *)a->dweight, (float *)a->dbias,
                               (float *)nullptr, a->D, a->W, 0, a->W, a->W);
        SEQ_DONE("crnn_conv_backward");
    } catch (...) { return -1; }
}

int32_t crnn_conv_step(const crnn_conv_args *a) {
    try {
        SEQ_ENTER(a, "crnn_conv_step");
        SeqCheck c{"crnn_conv_step", {}};
        crnn::ConvP q;
        if (!conv_check(c, a, false, q)) return sfail(c.err);
        if (a->seq_start || a->seq_len) return sfail("crnn_conv_step: rows are one per sequence (no seq_start, seq_len)");
        if (a->n_slots < 0 || a->n_slots > 0x7fffffff || (!a->slot && a->n_seq > a->n_slots)) return sfail("crnn_conv_step: n_slots does not fit the rows");
        if (a->n_seq == 0) return 0;
        if (!c.view(a->x, "x", a->dtype, true, false, false, a->D) || !c.view(a->y, "y", a->dtype, true, false, true, a->n_seq > 1 ? a->D : 0) ||
            !c.view(a->state_in, "state_in", a->dtype, a->W > 1 && a->n_slots > 0, false, true, a->W > 2 ? a->D : 0) || !c.other({&a->y}, {&a->x}, 1) ||
            !c.apart(a->state_in, "state_in", a->n_slots, a->W - 1, a->D))
            return sfail(c.err);
        if (!a->weight) return sfail("crnn_conv_step: weight is missing");
        if (!conv_apart(c, a, false, true)) return sfail(c.err);
        crnn::ConvStepP p{};
        p.x = seq_view(a->x, 1); p.y = seq_view(a->y, 1); p.st = seq_view(a->state_in, 1);
        p.w = a->weight; p.bias = a->bias; p.slot = a->slot; p.rows = a->n_seq; p.n_slots = a->n_slots;
        p.D = a->D; p.W = a->W; p.silu = a->silu;
        const hipStream_t st = (hipStream_t)a->stream;
        const int VW = a->dtype == CRNN_DT_F64 ? 2 : 4;
        const int V = a->D % VW == 0 && conv_weights_fit(a, VW) && conv_fits(a->x, VW) && conv_fits(a->y, VW) && conv_fits(a->state_in, VW) ? VW : 1;
        if (a->n_seq * (int64_t)((a->D + 256 * V - 1) / (256 * V)) > kSeqMaxGrid) return sfail("crnn_conv_step: too many rows and channels for one launch");
        SEQ_DEVICE(a->device, "crnn_conv_step");
        if (a->dtype == CRNN_DT_F64) conv_step_launch_w<CRNN_DT_F64>(p, V, st);
        else if (a->dtype == CRNN_DT_F32) conv_step_launch_w<CRNN_DT_F32>(p, V, st);
        else if (a->dtype == CRNN_DT_BF16) conv_step_launch_w<CRNN_DT_BF16>(p, V, st);
        else conv_step_launch_w<CRNN_DT_F16>(p, V, st);
        SEQ_DONE("crnn_conv_step");
    } catch (...) { return -1; }
}

int64_t crnn_scan_workspace(const crnn_scan_args *a, int32_t which) {
    try {
        SEQ_ENTER(a, "crnn_scan_workspace");
        if (which < 0 || which > 1) return sfail("crnn_scan_workspace: which must be 0 or 1");
        SeqCheck c{"crnn_scan_workspace", {}};
        ScanPlan s;
        if (!scan_plan(c, a, which == 1, s)) return sfail(c.err);
        return s.total;
    } catch (...) { return -1; }
}

int32_t crnn_scan_forward(const crnn_scan_args *a) {
    try {
        SEQ_ENTER(a, "crnn_scan_forward");
        SeqCheck c{"crnn_scan_forward", {}};
        ScanPlan s;
        if (!scan_plan(c, a, false, s)) return sfail(c.err);
        if (a->n_seq == 0) return 0;
        if (!scan_views(c, a, false)) return sfail(c.err);
        if (s.total > 0 && (!a->workspace || a->workspace_bytes < s.total)) return sfail("crnn_scan_forward: workspace is missing or too small");
        if (!scan_apart(c, a, false)) return sfail(c.err);
        SEQ_DEVICE(a->device, "crnn_scan_forward");
        scan_fill(a, s);
        SCAN_RUN(scan_forward_run);
        SEQ_DONE("crnn_scan_forward");
    } catch (...) { return -1; }
}

int32_t crnn_scan_backward(const crnn_scan_args *a) {
    try {
        SEQ_ENTER(a, "crnn_scan_backward");
        SeqCheck c{"crnn_scan_backward", {}};
        ScanPlan s;
        if (!scan_plan(c, a, true, s) || !scan_views(c, a, true)) return sfail(c.err);
        if (s.total > 0 && (!a->workspace || a->workspace_bytes < s.total)) return sfail("crnn_scan_backward: workspace is missing or too small");
        if (a->n_seq == 0) return sfail("crnn_scan_backward: no sequences");
        if (!scan_apart(c, a, true)) return sfail(c.err);
        SEQ_DEVICE(a->device, "crnn_scan_backward");
        scan_fill(a, s);
        SCAN_RUN(scan_backward_run);
        SEQ_DONE("crnn_scan_backward");
    } catch (...) { return -1; }
}

int32_t crnn_scan_step(const crnn_scan_args *a) {
    try {
        SEQ_ENTER(a, "crnn_scan_step");
        SeqCheck c{"crnn_scan_step", {}};
        ScanPlan s;
        if (!scan_plan(c, a, false, s, true)) return sfail(c.err);
        if (a->seq_start || a->seq_len) return sfail("crnn_scan_step: rows are one per sequence (no seq_start, seq_len)");
        if (a->n_slots < 0 || a->n_slots > 0x7fffffff || (!a->slot && a->n_seq > a->n_slots)) return sfail("crnn_scan_step: n_slots does not fit the rows");
        if (a->n_seq == 0) return 0;
        if (!scan_views(c, a, false, true)) return sfail(c.err);
        if (s.p8) return sfail("crnn_scan_step: u and z cannot be 8-bit checkpoints here");
        if (!a->state_out && a->n_slots > 0) return sfail("crnn_scan_step: the states are missing");
        if (!scan_apart(c, a, false, true)) return sfail(c.err);
        crnn::ScanStepP p{};
        p.u = seq_view(a->u, 4); p.dt = seq_view(a->dt, 4); p.z = seq_view(a->z, 4); p.y = seq_view(a->y, 4); p.B = seq_view(a->B, 1); p.C = seq_view(a->C, 1);
        p.Bg = a->B_group; p.Cg = a->C_group; p.Bn = a->B_state; p.Cn = a->C_state;
        p.A = a->A; p.Dskip = a->skip; p.dt_bias = a->dt_bias; p.state = a->state_out; p.slot = a->slot;
        p.rows = a->n_seq; p.n_slots = a->n_slots;
        p.D = a->D; p.N = a->N; p.G = a->G; p.Dg = a->D / a->G; p.softplus = a->softplus;
        p.gate = a->z.ptr != nullptr;
        if (!p.gate) p.z = p.u;
        for (p.lpc = 1; p.lpc * 4 < a->N;) p.lpc *= 2;
        const uintptr_t align = s.f64 ? 32 : 16;
        p.vec = a->N == 4 * p.lpc && (uintptr_t)a->A % align == 0 && (uintptr_t)a->state_out % align == 0;
        // four channels a thread where that still gives every SIMD a wavefront
        const int cpb = 256 / p.lpc;
        const int cpt = !s.f64 && (int64_t)a->n_seq * ((a->D + 4 * cpb - 1) / (4 * cpb)) >= 1024 ? 4 : 1;
        const int64_t grid = (int64_t)a->n_seq * ((a->D + cpt * cpb - 1) / (cpt * cpb));
        if (grid > kSeqMaxGrid) return sfail("crnn_scan_step: too many rows and channels for one launch");
        SEQ_DEVICE(a->device, "crnn_scan_step");
        const hipStream_t st = (hipStream_t)a->stream;
        if (s.f64) hipLaunchKernelGGL((crnn::seq_scan_step_kernel<8, 1>), dim3((unsigned)grid), dim3(256), 0, st, p);
        else if (a->dtype == CRNN_DT_F32) {
            if (cpt == 4) hipLaunchKernelGGL((crnn::seq_scan_step_kernel<4, 4>), dim3((unsigned)grid), dim3(256), 0, st, p);
            else hipLaunchKernelGGL((crnn::seq_scan_step_kernel<4, 1>), dim3((unsigned)grid), dim3(256), 0, st, p);
        } else {
            if (cpt == 4) hipLaunchKernelGGL((crnn::seq_scan_step_kernel<2, 4>), dim3((unsigned)grid), dim3(256), 0, st, p);
            else hipLaunchKernelGGL((crnn::seq_scan_step_kernel<2, 1>), dim3((unsigned)grid), dim3(256), 0, st, p);
        }
        SEQ_DONE("crnn_scan_step");
    } catch (...) { return -1; }
}

static bool pack_plan(SeqCheck &c, const crnn_view *x, int64_t rows, int32_t D, const void *codes, const void *scales, bool out, crnn::PackP &p) {
    if (!x) return c.bad("null view");
    if (rows < 0 || D < 1 || D > (1 << 24)) return c.bad("bad sizes");
    if (x->dtype < CRNN_DT_F32 || x->dtype > CRNN_DT_F16) return c.bad("float, bfloat16 or half only");
    p = crnn::PackP{};
    p.rows = rows; p.D = D; p.nb = (D + 31) / 32;
    if (rows == 0) return true;
    if (!codes || !scales) return c.bad("codes or scales are missing");
    if (!c.view(*x, "x", x->dtype, true, false, out, rows > 1 ? D : 0)) return false;
    SeqShare m;
    if (out) {
        m.out(*x, D, rows, 1); m.in(codes, rows * D); m.in(scales, rows * p.nb);
    } else {
        m.in(*x, D, rows, 1); m.out(codes, rows * D); m.out(scales, rows * p.nb);
    }
    if (!m.ok(c)) return false;
    p.x = seq_view(*x, 16 / seq_size(x->dtype));
    p.q = (int8_t *)codes; p.sc = (uint8_t *)scales;
    p.vecq = (uintptr_t)codes % 16 == 0 && D % 16 == 0 ? 16 : (uintptr_t)codes % 4 == 0 && D % 4 == 0 ? 4 : 1;
    if ((rows * 2 * p.nb + 255) / 256 > kSeqMaxGrid) return c.bad("too many rows and channels for one launch");
    return true;
}

int32_t crnn_pack8(int32_t device, void *stream, const crnn_view *x, int64_t rows, int32_t D, void *codes, void *scales) {
    try {
        SeqCheck c{"crnn_pack8", {}};
        crnn::PackP p;
        if (!pack_plan(c, x, rows, D, codes, scales, false, p)) return sfail(c.err);
        if (rows == 0) return 0;
        SEQ_DEVICE(device, "crnn_pack8");
        const dim3 grid((unsigned)((rows * 2 * p.nb + 255) / 256));
        const hipStream_t st = (hipStream_t)stream;
        if (x->dtype == CRNN_DT_F32) hipLaunchKernelGGL((crnn::seq_pack_kernel<CRNN_DT_F32>), grid, dim3(256), 0, st, p);
        else if (x->dtype == CRNN_DT_BF16) hipLaunchKernelGGL((crnn::seq_pack_kernel<CRNN_DT_BF16>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((crnn::seq_pack_kernel<CRNN_DT_F16>), grid, dim3(256), 0, st, p);
        SEQ_DONE("crnn_pack8");
    } catch (...) { return -1; }
}

int32_t crnn_unpack8(int32_t device, void *stream, const void *codes, const void *scales, int64_t rows, int32_t D, const crnn_view *x) {
    try {
        SeqCheck c{"crnn_unpack8", {}};
        crnn::PackP p;
        if (!pack_plan(c, x, rows, D, codes, scales, true, p)) return sfail(c.err);
        if (rows == 0) return 0;
        SEQ_DEVICE(device, "crnn_unpack8");
        const dim3 grid((unsigned)((rows * 2 * p.nb + 255) / 256));
        const hipStream_t st = (hipStream_t)stream;
        if (x->dtype == CRNN_DT_F32) hipLaunchKernelGGL((crnn::seq_unpack_kernel<CRNN_DT_F32>), grid, dim3(256), 0, st, p);
        else if (x->dtype == CRNN_DT_BF16) hipLaunchKernelGGL((crnn::seq_unpack_kernel<CRNN_DT_BF16>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((crnn::seq_unpack_kernel<CRNN_DT_F16>), grid, dim3(256), 0, st, p);
        SEQ_DONE("crnn_unpack8");
    } catch (...) { return -1; }
}

}  // extern "C"
