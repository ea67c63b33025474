// Drafted tokens checked against the target's logits (speculative sampling), a
// batch of sequences at once.  No counterpart in the reference, which decodes one
// token a step; the target's distribution is that of its sampler without the
// nucleus, softmax(x / T) (runtime.rs:534-601).
//
// Sequence s has k drafts y_0 .. y_{k-1} and k + 1 rows of logits: row i is the
// target's at the place of draft i, row k the one after them.  With p_i =
// softmax(x_i / T) (T <= 0: certain of the first largest logit), q_i the draft's
// own probabilities (none given: the draft was certain) and a uniform u_i per row:
//   draft i is accepted while  u_i q_i(y_i) < p_i(y_i);
//   at the first rejected i the token is drawn from  max(p_i - q_i, 0)  normalised,
//   after k accepted drafts from p_k: the first index whose cumulative weight
//   exceeds u_k of the whole.
// Then every emitted token has the target's distribution.
//
// A token changes where two cumulative sums of a vocabulary's weights change
// places: the emission row's weights and sums are held in f64 (a sum off by 1e-8
// would change one token in a thousand of a vocabulary of 128256; these are off by
// about 1e-13).  A draft's test has one border alone, so the other rows' sums Z are
// f32 weights' (1e-7 of Z): of k + 1 rows one is weighed in f64, whose exp costs
// about 20 f64 operations a logit, more than the logit's bytes (stats in f64: 56 us
// of 64 x 5 rows x 128256, in f32 at the rate of the bytes).
//
// Three launches (us of 64 sequences with 4 drafts of 128256 columns, of one with 4
// of 32000, measured one after another; the latter's last two are one of 11.6):
//   verify_stats_kernel  one pass over all logits: per chunk of a row its largest
//                        logit, the first place of it, and the f32 sum of weights
//                        relative to it.  HBM bound (27.5: 6 TB/s; 3.6).
//   verify_rest_kernel   the tests, then per chunk of the emission row in f64:
//                        W = sum w, and over A = {w > q Z} the sums of w and q.
//                        The rest's weight is then W_A - Q_A Z with the f64 Z =
//                        sum W: a column that the f32 Z puts on the wrong side of A
//                        weighs below 1e-7 of itself.  Bound by f64 rates and by the
//                        tests' chain of loads before it (20.8; 6.0).
//   verify_emit_kernel   the crossing's chunk by the chunks' sums, then its place in
//                        the chunk, which is weighed again: a chain of latencies
//                        (5.1; 5.2)
#include "zr_internal.h"

namespace zr {

namespace {

constexpr int kSeqs = 256;        // sequences a launch (their lengths and temperatures are kernel arguments)
constexpr int kMaxDrafts = 255;   // drafts of one sequence
constexpr int kRestChunk = 2048;  // columns of an emission row's chunk
constexpr float kLog2E = 1.44269504088896341f;

// Sequences of a launch, as a kernel argument: N = 16 or kSeqs (2 KiB of arguments
// cost the host half a microsecond a launch: 5 rows of 32000 15.5 us with them, 13.7 without).
constexpr int kFewSeqs = 16;
template <int N> struct VerifyArgs {
    int row[N + 1];    // first logits row of each sequence, and the end; drafts before it: row[s] - s
    float temp[N];
};

struct VerifyBufs {
    const float* logits;   // [rows, cols]
    int cols, chunk, chunks;
    const uint32_t* drafts;
    const float* probs;    // [drafts, cols] or null
    const float* u;        // [rows]
    struct ChunkStat* stat;  // [rows][chunks]
    struct RestSum* rest;    // [n][rest_chunks]
    struct Decision* dec;    // [n]
    int* done;               // [n] workgroups of a sequence that have their sums (0 between calls)
    int rest_chunks;
    uint32_t* out;
    int out_stride;
    int* accepted;
};

struct ChunkStat {
    float m;    // largest logit of the chunk (-inf: none)
    int at;     // its first column
    float sum;  // of exp((x - m) / T)
    int pad;
};

struct RestSum {
    double w, wa, qa;  // sum of w; over the columns with w > q Z: of w and of q
};

// What the tests of a sequence come to: where its token is drawn from.
struct Decision {
    float m;       // the row's largest logit
    int at;        // the first place of it
    float z;       // the f32 sum of its weights (0: none weighs)
    float t;
    int row;       // of the logits
    int probs;     // ... of the rejected draft's probabilities, or -1: p ...
    uint32_t out;  // ... without a certain draft's own column (none: 0xffffffff)
    float u;
    int first, accepted;  // the sequence's first draft; how many were accepted
};

// Weights exp((x - m) / T) = 2^z, z = (x - m) log2(e) / T, in f64.  z = k + f
// with k by adding and taking away 1.5 2^52 (which leaves it in the sum's low
// bits), |f| <= 1/2, and 2^f by its Taylor series to f^10 (the next term is below
// 2.3e-13); the factor and the product round by 2^-53 of |z|, below 100 or so.
struct Weigher {
    double c, top;
    bool inf;  // the largest logit is +inf: it weighs 1, all others 0
    __device__ Weigher(float m, float t) : c(1.4426950408889634074 / (double)t), top(m), inf(m == INFINITY) {}
    // 0 for -inf and for what is not a number (z at least -2000: scaled to 0)
    __device__ __forceinline__ double operator()(float x) const {
        constexpr double kRound = 6755399441055744.0, l = 0.69314718055994530942;
        constexpr double c2 = l * l / 2, c3 = c2 * l / 3, c4 = c3 * l / 4, c5 = c4 * l / 5, c6 = c5 * l / 6,
                         c7 = c6 * l / 7, c8 = c7 * l / 8, c9 = c8 * l / 9, c10 = c9 * l / 10;
        const double z = __builtin_fmax(((double)x - top) * c, -2000.0);  // (NaN: -2000)
        const double t = z + kRound, f = z - (t - kRound);
        double e = __builtin_fma(c10, f, c9);
        e = __builtin_fma(e, f, c8);
        e = __builtin_fma(e, f, c7);
        e = __builtin_fma(e, f, c6);
        e = __builtin_fma(e, f, c5);
        e = __builtin_fma(e, f, c4);
        e = __builtin_fma(e, f, c3);
        e = __builtin_fma(e, f, c2);
        e = __builtin_fma(e, f, l);
        e = __builtin_fma(e, f, 1.0);
        return __builtin_ldexp(e, __double2loint(t));
    }
};
// the same in f32: c = log2(e) / T
__device__ inline float weight32(float x, float m, float c) {
    const float y = fmaxf((x - m) * c, -1000.0f);  // (NaN: nothing)
    return x == m ? 1.0f : __builtin_amdgcn_exp2f(y);
}

// Lanes meet over DPP (rows of 16 lanes, every lane active in a row that takes
// part) and, between rows, over readlane: a step costs tens of cycles less than a
// shuffle through LDS, and these kernels are chains of such steps.
constexpr int kRowRor = 0x120, kRowShr = 0x110;  // + lanes; shr fills with 0
template <int CTRL> __device__ inline int dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }
template <int CTRL> __device__ inline float dpp(float v) { return __int_as_float(dpp<CTRL>(__float_as_int(v))); }
template <int CTRL> __device__ inline double dpp(double v) {
    return __hiloint2double(dpp<CTRL>(__double2hiint(v)), dpp<CTRL>(__double2loint(v)));
}
__device__ inline int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ inline float lane_of(float v, int lane) { return __int_as_float(lane_of(__float_as_int(v), lane)); }
__device__ inline double lane_of(double v, int lane) {
    return __hiloint2double(lane_of(__double2hiint(v), lane), lane_of(__double2loint(v), lane));
}
// sums: of a row of 16 lanes, of the wave (the same bits in every lane)
template <typename T> __device__ inline T row_sum(T v) {
    v += dpp<kRowRor + 8>(v);
    v += dpp<kRowRor + 4>(v);
    v += dpp<kRowRor + 2>(v);
    v += dpp<kRowRor + 1>(v);
    return v;
}
template <typename T> __device__ inline T wave_sum(T v) {
    v = row_sum(v);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
// the sum of the lanes up to and with this one
__device__ inline double wave_scan(double v, int lane) {
    v += dpp<kRowShr + 1>(v);
    v += dpp<kRowShr + 2>(v);
    v += dpp<kRowShr + 4>(v);
    v += dpp<kRowShr + 8>(v);
    const double r0 = lane_of(v, 15), r1 = r0 + lane_of(v, 31), r2 = r1 + lane_of(v, 47);
    return v + (lane < 16 ? 0.0 : lane < 32 ? r0 : lane < 48 ? r1 : r2);
}
// the larger logit, the lower column among equals
__device__ inline void take_larger(float& m, int& at, float m2, int at2) {
    if (m2 > m || (m2 == m && at2 < at)) {
        m = m2;
        at = at2;
    }
}
__device__ inline void row_larger(float& m, int& at) {
    take_larger(m, at, dpp<kRowRor + 8>(m), dpp<kRowRor + 8>(at));
    take_larger(m, at, dpp<kRowRor + 4>(m), dpp<kRowRor + 4>(at));
    take_larger(m, at, dpp<kRowRor + 2>(m), dpp<kRowRor + 2>(at));
    take_larger(m, at, dpp<kRowRor + 1>(m), dpp<kRowRor + 1>(at));
}
__device__ inline void wave_larger(float& m, int& at) {
    row_larger(m, at);
    float top = lane_of(m, 0);
    int col = lane_of(at, 0);
#pragma unroll
    for (int r = 16; r < 64; r += 16) take_larger(top, col, lane_of(m, r), lane_of(at, r));
    m = top;
    at = col;
}

template <int N> __device__ inline int seq_of(const VerifyArgs<N>& v, int n, int row) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (v.row[mid] <= row) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Four columns from c on; the ones past the row's end are `none`.  Rows of an odd
// length start at any multiple of 4 bytes: so do these 16-byte loads.
struct __attribute__((packed, aligned(4))) Four {
    float x, y, z, w;
};
__device__ inline float4 four(const float* x, int c) {
    const Four f = *(const Four*)(x + c);
    return make_float4(f.x, f.y, f.z, f.w);
}
__device__ inline float4 four_to(const float* x, int c, int cols, float none) {
    if (c + 4 <= cols) return four(x, c);
    return make_float4(c < cols ? x[c] : none, c + 1 < cols ? x[c + 1] : none, c + 2 < cols ? x[c + 2] : none, none);
}

// A workgroup of 4 waves takes one chunk of 1024 E columns of one row; every
// load of a lane goes out before the first is used.
template <int E, int N>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyBufs b, VerifyArgs<N> v, int n) {
    __shared__ float sm[4];
    __shared__ int sat[4];
    __shared__ float ss[4];
    const int row = blockIdx.x / b.chunks, ch = blockIdx.x - row * b.chunks;
    const int c0 = ch * b.chunk, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* x = b.logits + (size_t)row * b.cols;
    float4 d[E];
    if (c0 + b.chunk <= b.cols) {
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = four(x, c0 + (e * 256 + tid) * 4);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = four_to(x, c0 + (e * 256 + tid) * 4, b.cols, -INFINITY);
    }
    const float t = v.temp[seq_of(v, n, row)];  // (behind the loads' issue: a chain of scalar loads)
    float m = -INFINITY;
    int at = c0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float f[4] = {d[e].x, d[e].y, d[e].z, d[e].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + (e * 256 + tid) * 4 + j;
            if (f[j] > m) {  // (a lane's columns ascend: the first of equals stays)
                m = f[j];
                at = c;
            }
        }
    }
    wave_larger(m, at);
    float sum = 0.0f;
    const float c = kLog2E / t;
    if (t > 0.0f && m != -INFINITY) {
        float s2 = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            sum += weight32(d[e].x, m, c);
            s2 += weight32(d[e].y, m, c);
            sum += weight32(d[e].z, m, c);
            s2 += weight32(d[e].w, m, c);
        }
        sum = wave_sum(sum + s2);
    }
    if (lane == 0) {
        sm[wave] = m;
        sat[wave] = at;
        ss[wave] = sum;
    }
    __syncthreads();
    if (tid) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) take_larger(m, at, sm[w], sat[w]);
    float all = 0.0f;
    if (t > 0.0f && m != -INFINITY)
#pragma unroll
        for (int w = 0; w < 4; ++w)
            if (sm[w] != -INFINITY) all += ss[w] * weight32(sm[w], m, c);
    b.stat[(size_t)row * b.chunks + ch] = {m, at, all, 0};
}

// The tests of a sequence, by 16 groups of 16 lanes, a row each in turn: the
// chunks' sums joined in one order, so every workgroup gets the same bits.  The
// draft's own logit and probability come beside them.
template <int N> __device__ inline Decision decide(const VerifyBufs& b, const VerifyArgs<N>& v, int s) {
    __shared__ float sm[kMaxDrafts + 1], sz[kMaxDrafts + 1];
    __shared__ int sat[kMaxDrafts + 1], ok[kMaxDrafts + 1];
    const int tid = threadIdx.x, lane = tid & 15;
    const int row0 = v.row[s], k = v.row[s + 1] - row0 - 1, d0 = row0 - s;
    const float t = v.temp[s], c32 = kLog2E / t;
    for (int i = tid >> 4; i <= k; i += 16) {
        const uint32_t y = i < k ? b.drafts[d0 + i] : 0xffffffffu;
        const bool in = y < (uint32_t)b.cols;  // (an id outside the vocabulary has no probability)
        const float xy = in ? b.logits[(size_t)(row0 + i) * b.cols + y] : -INFINITY;
        const float qy = !in ? 0.0f : b.probs ? fmaxf(b.probs[(size_t)(d0 + i) * b.cols + y], 0.0f) : 1.0f;
        const float u = b.u[row0 + i];
        const ChunkStat* st = b.stat + (size_t)(row0 + i) * b.chunks;
        float m = -INFINITY;
        int at = 0x7fffffff;
        for (int c = lane; c < b.chunks; c += 16) {
            const ChunkStat x = st[c];
            if (x.m > m) {
                m = x.m;
                at = x.at;
            }
        }
        row_larger(m, at);
        if (m == -INFINITY) at = 0;  // a row without a finite logit: the first place, as the argmax has it
        float z = 0.0f;
        if (t > 0.0f && m != -INFINITY)
            for (int c = lane; c < b.chunks; c += 16) {
                const ChunkStat x = st[c];
                if (x.m != -INFINITY) z += x.sum * weight32(x.m, m, c32);
            }
        z = row_sum(z);
        if (lane == 0) {
            sm[i] = m;
            sat[i] = at;
            sz[i] = z;
            ok[i] = t <= 0.0f ? y == (uint32_t)at
                              : m != -INFINITY && (double)u * (double)qy * (double)z < (m == INFINITY ? (xy == m ? 1.0 : 0.0) : Weigher(m, t)(xy));
        }
    }
    __syncthreads();
    int a = 0;
    for (;;) {  // (64 drafts at a time: the first rejected one)
        const int i = a + (tid & 63);
        const unsigned long long no = __ballot(i >= k || !ok[i]);
        if (no) {
            a += __ffsll(no) - 1;
            break;
        }
        a += 64;
    }
    const bool left = a < k;  // a draft was rejected
    return {sm[a], sat[a], sz[a], t, row0 + a, left && b.probs ? d0 + a : -1, left && !b.probs ? b.drafts[d0 + a] : 0xffffffffu,
            b.u[row0 + k], d0, a};
}

// Finds the token of a sequence by a workgroup of THREADS (mine: the chunk sums of
// this lane's first chunk) and writes what the sequence comes to.  A chain of
// latencies: what can be loaded before the decision is known is.
template <int THREADS>
__device__ inline void draw(const VerifyBufs& b, int s, const Decision& d, const RestSum* rs, const RestSum mine) {
    __shared__ double sw[THREADS / 64];
    __shared__ double s_before, s_target, s_z;
    __shared__ int s_chunk, s_first, s_last;
    __shared__ bool s_whole;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t y = tid < d.accepted ? b.drafts[d.first + tid] : 0;  // (at most 255 drafts)
    uint32_t token = (uint32_t)d.at;
    if (d.t > 0.0f && d.z > 0.0f) {
        const float* xr = b.logits + (size_t)d.row * b.cols;
        const float* qr = d.probs >= 0 ? b.probs + (size_t)d.probs * b.cols : nullptr;
        const Weigher weight(d.m, d.t);
        if (wave == 0) {
            auto sum_of = [&](int c) { return c < 64 ? mine : rs[c]; };
            double z = 0.0, total = 0.0;
            for (int c = lane; c < b.rest_chunks; c += 64) z += sum_of(c).w;
            z = wave_sum(z);
            bool whole = false;  // the rest weighs nothing (by rounding): the token comes from p
            auto chunk_sum = [&](int c) {
                const RestSum x = sum_of(c);
                return whole ? x.w : qr ? __builtin_fmax(__builtin_fma(-x.qa, z, x.wa), 0.0) : x.wa;
            };
            for (int pass = 0; pass < 2; ++pass) {
                total = 0.0;
                for (int c = lane; c < b.rest_chunks; c += 64) total += chunk_sum(c);
                total = wave_sum(total);
                if (total > 0.0) break;
                whole = true;
            }
            const double target = (double)d.u * total;
            // the first chunk whose end exceeds the target; none (u >= 1 or not a number): the last that weighs
            double before = 0.0, pick_before = 0.0;
            int chunk = 0;
            bool found = false;
            for (int c0 = 0; c0 < b.rest_chunks && !found; c0 += 64) {
                const double w = c0 + lane < b.rest_chunks ? chunk_sum(c0 + lane) : 0.0;
                const double run = wave_scan(w, lane);
                const unsigned long long hit = __ballot(w > 0.0 && before + run > target), some = __ballot(w > 0.0);
                if (some) {
                    const int pick = hit ? __ffsll(hit) - 1 : 63 - __clzll(some);
                    chunk = c0 + pick;
                    pick_before = before + (pick ? lane_of(run, pick - 1) : 0.0);
                    found = hit != 0;
                }
                before += lane_of(run, 63);
            }
            if (lane == 0) {
                s_chunk = chunk;
                s_before = pick_before;
                s_target = target;
                s_z = z;
                s_whole = whole;
                s_first = 0x7fffffff;
                s_last = -1;
            }
        }
        __syncthreads();
        // the chunk's columns, E to a thread, in order
        constexpr int E = kRestChunk / THREADS;
        const int c0 = s_chunk * kRestChunk + tid * E;
        const double z = s_z;
        const bool whole = s_whole;
        float x[E], q[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = c0 + e < b.cols ? xr[c0 + e] : -INFINITY;
            q[e] = qr && c0 + e < b.cols ? fmaxf(qr[c0 + e], 0.0f) : 0.0f;
        }
        double w[E], sum = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            w[e] = weight.inf ? (x[e] == d.m ? 1.0 : 0.0) : weight(x[e]);
            if (!whole) w[e] = qr ? __builtin_fmax(w[e] - (double)q[e] * z, 0.0) : (uint32_t)(c0 + e) == d.out ? 0.0 : w[e];
            sum += w[e];
        }
        const double run = wave_scan(sum, lane);
        if (lane == 63) sw[wave] = run;
        __syncthreads();
        double cum = s_before;
        for (int i = 0; i < wave; ++i) cum += sw[i];
        cum += run - sum;
        int first = 0x7fffffff, last = -1;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            cum += w[e];
            if (w[e] > 0.0) {
                last = c0 + e;
                if (first == 0x7fffffff && cum > s_target) first = c0 + e;
            }
        }
        // (a wave's columns ascend with its lanes; one atomic a wave: every lane's own took 5 us)
        const unsigned long long hit = __ballot(first != 0x7fffffff), some = __ballot(last >= 0);
        if (hit && lane == __ffsll(hit) - 1) atomicMin(&s_first, first);
        if (some && lane == 63 - __clzll(some)) atomicMax(&s_last, last);
        __syncthreads();
        // (no crossing: the chunk's sum and this one's order differ in their last bits, or u >= 1)
        token = s_first != 0x7fffffff ? (uint32_t)s_first : s_last >= 0 ? (uint32_t)s_last : (uint32_t)d.at;
    }
    for (int i = tid; i < b.out_stride; i += THREADS)
        b.out[(size_t)s * b.out_stride + i] = i < d.accepted ? y : i == d.accepted ? token : 0xffffffffu;
    if (tid == 0) b.accepted[s] = d.accepted;
}

// A workgroup takes `per` chunks of one sequence's emission row in turn: as many as
// leave no more workgroups than the chip holds at once, for each has the tests to do first.
// DRAW: few workgroups in all; the last of a sequence's draws its token as well, and
// a third launch is saved.  It knows that it is by a count (its own chunk sums are
// released by its addition to it, the others' acquired with it); many workgroups would
// pay a write-back of an XCD's L2 each.
template <int N, bool DRAW>
__global__ __launch_bounds__(256) void verify_rest_kernel(VerifyBufs b, VerifyArgs<N> v, int per, int groups) {
    __shared__ double ss[2][3][4];
    constexpr int E = kRestChunk / 256;
    const int s = blockIdx.x / groups, g = blockIdx.x - s * groups, tid = threadIdx.x;
    const Decision d = decide(b, v, s);
    RestSum* rs = b.rest + (size_t)s * b.rest_chunks;
    if (!DRAW && g == 0 && tid == 0) b.dec[s] = d;
    if (d.t <= 0.0f || d.z <= 0.0f) {  // greedy, or nothing weighs: the first largest logit
        if (DRAW && g == 0) draw<256>(b, s, d, rs, RestSum{});
        return;
    }
    const float* xr = b.logits + (size_t)d.row * b.cols;
    const float* qr = d.probs >= 0 ? b.probs + (size_t)d.probs * b.cols : nullptr;
    const Weigher weight(d.m, d.t);
    const int end = min((g + 1) * per, b.rest_chunks);
    for (int ch = g * per; ch < end; ++ch) {
        const int c0 = ch * kRestChunk, buf = ch & 1;
        float x[E], q[E];
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const int c = c0 + e * 256 + tid * 4;
            float4 xv, qv = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (c0 + kRestChunk <= b.cols) {
                xv = four(xr, c);
                if (qr) qv = four(qr, c);
            } else {
                xv = four_to(xr, c, b.cols, -INFINITY);
                if (qr) qv = four_to(qr, c, b.cols, 0.0f);
            }
            x[e] = xv.x, x[e + 1] = xv.y, x[e + 2] = xv.z, x[e + 3] = xv.w;
            q[e] = qv.x, q[e + 1] = qv.y, q[e + 2] = qv.z, q[e + 3] = qv.w;
        }
        double w = 0.0, wa = 0.0, qa = 0.0;
        if (qr) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const double we = weight.inf ? (x[e] == d.m ? 1.0 : 0.0) : weight(x[e]);
                const float qe = fmaxf(q[e], 0.0f);
                w += we;
                const bool in = (float)we > qe * d.z;
                wa += in ? we : 0.0;
                qa += (double)(in ? qe : 0.0f);
            }
            wa = wave_sum(wa);
            qa = wave_sum(qa);
        } else {  // p, without a certain draft's own column (alone in weighing, it is drawn as the largest)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float xe = (uint32_t)(c0 + (e / 4) * 1024 + tid * 4 + (e & 3)) == d.out ? -INFINITY : x[e];
                w += weight.inf ? (xe == d.m ? 1.0 : 0.0) : weight(xe);
            }
        }
        w = wave_sum(w);
        if (!qr) wa = w;
        if ((tid & 63) == 0) {
            ss[buf][0][tid >> 6] = w;
            ss[buf][1][tid >> 6] = wa;
            ss[buf][2][tid >> 6] = qa;
        }
        __syncthreads();  // (one a chunk: two buffers, in turn)
        if (tid == 0) {
            double o[3];
#pragma unroll
            for (int i = 0; i < 3; ++i) o[i] = (ss[buf][i][0] + ss[buf][i][1]) + (ss[buf][i][2] + ss[buf][i][3]);
            rs[ch] = {o[0], o[1], o[2]};
        }
    }
    if constexpr (DRAW) {
        __shared__ bool s_mine;
        if (tid == 0) {
            const int before = __hip_atomic_fetch_add(b.done + s, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
            s_mine = before == groups - 1;
            if (s_mine) b.done[s] = 0;  // for the next call
        }
        __syncthreads();
        if (!s_mine) return;
        draw<256>(b, s, d, rs, rs[min(tid & 63, b.rest_chunks - 1)]);
    }
}

// A workgroup of 16 waves per sequence: two columns a thread keep the code short
// (its first pass waits for every line of it).
constexpr int kEmitThreads = 1024;
__global__ __launch_bounds__(kEmitThreads) void verify_emit_kernel(VerifyBufs b) {
    const int s = blockIdx.x;
    const RestSum* rs = b.rest + (size_t)s * b.rest_chunks;
    const RestSum mine = rs[min((int)(threadIdx.x & 63), b.rest_chunks - 1)];  // (of a greedy row: not used)
    const Decision d = b.dec[s];
    draw<kEmitThreads>(b, s, d, rs, mine);
}

// Workgroups up to which the rest's kernel draws too (us a call, three launches / two:
// 16 workgroups 13.7 / 10.5, 63 13.0 / 11.6, 64 12.2 / 11.6, 126 12.5 / 14.6, 128 12.2 /
// 13.3, 504 14.6 / 23.4, 1008 18.3 / 41.9).
constexpr int kDrawWgs = 64;

// The launches of m <= N sequences.
template <int N>
void launch_passes(zr_context* ctx, const VerifyBufs& b, const int* draft_len, const float* temperature, int m, int e) {
    VerifyArgs<N> v;
    int r = 0;
    for (int s = 0; s < N; ++s) {
        v.row[s] = r;
        v.temp[s] = s < m ? temperature[s] : 0.0f;
        if (s < m) r += draft_len[s] + 1;
    }
    v.row[N] = r;
    auto stats = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(r * b.chunks), dim3(256), 0, ctx->stream, b, v, m);
    };
    switch (e) {
        case 1: stats(verify_stats_kernel<1, N>); break;
        case 2: stats(verify_stats_kernel<2, N>); break;
        case 4: stats(verify_stats_kernel<4, N>); break;
        default: stats(verify_stats_kernel<8, N>); break;
    }
    const int per = (m * b.rest_chunks + 2047) / 2048, groups = (b.rest_chunks + per - 1) / per;
    auto rest = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(m * groups), dim3(256), 0, ctx->stream, b, v, per, groups);
    };
    if (m * groups <= kDrawWgs) {
        rest(verify_rest_kernel<N, true>);
    } else {
        rest(verify_rest_kernel<N, false>);
        hipLaunchKernelGGL(verify_emit_kernel, dim3(m), dim3(kEmitThreads), 0, ctx->stream, b);
    }
}

}  // namespace

zr_status launch_verify(zr_context* ctx, const float* d_logits, int cols, const zr_verify_batch* vb, uint32_t* d_out,
                        int out_stride, int* d_accepted) {
    const int n = vb->num_seqs;
    long rows = 0;
    for (int s = 0; s < n; ++s) rows += vb->draft_len[s] + 1;
    // Chunks of a power of two of 1024 columns, at most 8: large ones where the rows
    // fill the chip by themselves, small ones where few rows would leave it idle
    // (5 rows of 32000: 160 workgroups).
    int e = 8;
    while (e > 1 && rows * ((cols + 1024 * e - 1) / (1024 * e)) < 1024) e /= 2;
    const int chunk = 1024 * e, chunks = (cols + chunk - 1) / chunk;
    const int rest_chunks = (cols + kRestChunk - 1) / kRestChunk;
    constexpr size_t done_bytes = sizeof(int) * kSeqs;  // (first, whatever the call: 0 between calls)
    const size_t stat_bytes = done_bytes + sizeof(ChunkStat) * (size_t)rows * chunks;
    const size_t dec_bytes = sizeof(Decision) * (size_t)n, need = stat_bytes + dec_bytes + sizeof(RestSum) * (size_t)n * rest_chunks;
    if (need > ctx->verify_ws_bytes) {
        ZR_HIP(ctx, hipStreamSynchronize(ctx->stream));
        if (ctx->verify_ws) (void)hipFree(ctx->verify_ws);
        ctx->verify_ws = nullptr;
        ctx->verify_ws_bytes = 0;
        const hipError_t err = hipMalloc(&ctx->verify_ws, need);
        if (err != hipSuccess)
            return set_err(ctx, err == hipErrorOutOfMemory ? ZR_E_OOM : ZR_E_HIP, "verification workspace of %zu bytes: %s",
                           need, hipGetErrorString(err));
        ZR_HIP(ctx, hipMemsetAsync(ctx->verify_ws, 0, done_bytes, ctx->stream));
        ctx->verify_ws_bytes = need;
    }
    hipEvent_t ev;
    timing_mark_begin(ctx, kClassOther, &ev);
    size_t row0 = 0, draft0 = 0;
    for (int s0 = 0; s0 < n; s0 += kSeqs) {
        const int m = std::min(kSeqs, n - s0);
        int r = 0;
        for (int s = 0; s < m; ++s) r += vb->draft_len[s0 + s] + 1;
        VerifyBufs b;
        b.logits = d_logits + row0 * cols;
        b.cols = cols;
        b.chunk = chunk;
        b.chunks = chunks;
        b.drafts = vb->d_drafts + draft0;
        b.probs = vb->d_draft_probs ? vb->d_draft_probs + draft0 * cols : nullptr;
        b.u = vb->d_uniforms + row0;
        b.done = (int*)ctx->verify_ws;
        b.stat = (ChunkStat*)((char*)ctx->verify_ws + done_bytes) + row0 * chunks;
        b.dec = (Decision*)((char*)ctx->verify_ws + stat_bytes) + s0;
        b.rest = (RestSum*)((char*)ctx->verify_ws + stat_bytes + dec_bytes) + (size_t)s0 * rest_chunks;
        b.rest_chunks = rest_chunks;
        b.out = d_out + (size_t)s0 * out_stride;
        b.out_stride = out_stride;
        b.accepted = d_accepted + s0;
        const int *lens = vb->draft_len + s0;
        const float* temps = vb->temperature + s0;
        if (m <= kFewSeqs)
            launch_passes<kFewSeqs>(ctx, b, lens, temps, m, e);
        else
            launch_passes<kSeqs>(ctx, b, lens, temps, m, e);
        ZR_LAUNCH_CHECK(ctx);
        row0 += r;
        draft0 += r - m;
    }
    timing_mark_end(ctx, kClassOther, ev);
    return ZR_OK;
}

}  // namespace zr
