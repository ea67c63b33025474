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
//   verify_stats_kernel  one pass over all logits: per chunk of a row its largest
//                        logit, the first place of it, and the f32 sum of weights
//                        relative to it.  HBM bound.
//   verify_rest_kernel   the tests, then per chunk of the emission row in f64:
//                        W = sum w, and over A = {w > q Z} the sums of w and q.
//                        The rest's weight is then W_A - Q_A Z with the f64 Z =
//                        sum W: a column that the f32 Z puts on the wrong side of A
//                        weighs below 1e-7 of itself.
//   verify_emit_kernel   the crossing's chunk by the chunks' sums, then its place in
//                        the chunk, which is weighed again
#include "zr_internal.h"

namespace zr {

namespace {

constexpr int kSeqs = 256;        // sequences a launch (their lengths and temperatures are kernel arguments)
constexpr int kMaxDrafts = 255;   // drafts of one sequence
constexpr int kRestChunk = 2048;  // columns of an emission row's chunk
constexpr double kNothing = -1000.0;  // exp of it is 0
constexpr float kLog2E = 1.44269504088896341f;

struct VerifyArgs {
    int row[kSeqs + 1];    // first logits row of each sequence, and the end; drafts before it: row[s] - s
    float temp[kSeqs];
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

// What the tests of a sequence come to.
struct Decision {
    int drafts, accepted, row;  // drafts of the sequence; accepted ones; the row the token comes from
    float m;                    // ... its largest logit
    int at;                     // ... the first place of it
    float z;                    // ... the f32 sum of its weights (0: none weighs)
    float t;
    int pad;
};

// exp(y) for y <= 0: y = k ln 2 + r, |r| <= ln 2 / 2 (k by adding and taking away
// 1.5 2^52, which leaves it in the sum's low bits; ln 2 in two parts, Cody and
// Waite's, k times the first exact), and the Taylor series of exp(r) to r^10 (the
// next term is below 2.2e-13).  0 below -700.
__device__ inline double exp_neg(double y) {
    constexpr double kRound = 6755399441055744.0;
    const double t = __builtin_fma(y, 1.4426950408889634074, kRound), k = t - kRound;
    double r = __builtin_fma(-k, 0.693147180369123816490, y);
    r = __builtin_fma(-k, 1.90821492927058770002e-10, r);
    double e = 1.0 / 3628800;
    e = __builtin_fma(e, r, 1.0 / 362880);
    e = __builtin_fma(e, r, 1.0 / 40320);
    e = __builtin_fma(e, r, 1.0 / 5040);
    e = __builtin_fma(e, r, 1.0 / 720);
    e = __builtin_fma(e, r, 1.0 / 120);
    e = __builtin_fma(e, r, 1.0 / 24);
    e = __builtin_fma(e, r, 1.0 / 6);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    const double scaled = __hiloint2double(__double2hiint(e) + (__double2loint(t) << 20), __double2loint(e));  // e 2^k
    return y >= -700.0 ? scaled : 0.0;
}

// weight of a logit against the largest one, m: exp((x - m) / T); 0 for -inf and
// for what is not a number, 1 for m itself (also where it is +inf)
__device__ inline double weight(float x, float m, double inv_t) {
    const double y = __builtin_fmax(((double)x - (double)m) * inv_t, kNothing);  // (NaN: kNothing)
    return x == m ? 1.0 : exp_neg(y);
}
// the same in f32: c = log2(e) / T
__device__ inline float weight32(float x, float m, float c) {
    const float y = fmaxf((x - m) * c, -1000.0f);  // (NaN: nothing)
    return x == m ? 1.0f : __builtin_amdgcn_exp2f(y);
}

__device__ inline double shfl_xor64(double v, int mask) {
    return __hiloint2double(__shfl_xor(__double2hiint(v), mask, 64), __shfl_xor(__double2loint(v), mask, 64));
}
__device__ inline double shfl_up64(double v, int by) {
    return __hiloint2double(__shfl_up(__double2hiint(v), by, 64), __shfl_up(__double2loint(v), by, 64));
}
// the larger logit, the lower column among equals
__device__ inline void take_larger(float& m, int& at, float m2, int at2) {
    if (m2 > m || (m2 == m && at2 < at)) {
        m = m2;
        at = at2;
    }
}
__device__ inline void wave_larger(float& m, int& at) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) take_larger(m, at, __shfl_xor(m, off, 64), __shfl_xor(at, off, 64));
}

__device__ inline int seq_of(const VerifyArgs& v, int n, int row) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (v.row[mid] <= row) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// A workgroup of 4 waves takes one chunk of 1024 E columns of one row; every
// load of a lane goes out before the first is used.
template <int E, bool VEC>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyBufs b, VerifyArgs v, int n) {
    __shared__ float sm[4];
    __shared__ int sat[4];
    __shared__ float ss[4];
    const int row = blockIdx.x / b.chunks, ch = blockIdx.x - row * b.chunks;
    const float t = v.temp[seq_of(v, n, row)];
    const int c0 = ch * b.chunk, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* x = b.logits + (size_t)row * b.cols;
    float4 d[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = c0 + (e * 256 + tid) * 4;
        const float none = -INFINITY;
        if constexpr (VEC) {
            d[e] = c < b.cols ? *(const float4*)(x + c) : make_float4(none, none, none, none);
        } else {  // rows that are not 16-byte aligned: the same columns in another order (c0 + 256 of a lane's four apart)
            const int c1 = c0 + e * 1024 + tid;
            d[e].x = c1 < b.cols ? x[c1] : none;
            d[e].y = c1 + 256 < b.cols ? x[c1 + 256] : none;
            d[e].z = c1 + 512 < b.cols ? x[c1 + 512] : none;
            d[e].w = c1 + 768 < b.cols ? x[c1 + 768] : none;
        }
    }
    float m = -INFINITY;
    int at = c0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float f[4] = {d[e].x, d[e].y, d[e].z, d[e].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = VEC ? c0 + (e * 256 + tid) * 4 + j : c0 + e * 1024 + tid + 256 * j;
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
        sum += s2;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
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
__device__ inline Decision decide(const VerifyBufs& b, const VerifyArgs& v, int s) {
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
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) take_larger(m, at, __shfl_xor(m, off, 64), __shfl_xor(at, off, 64));
        if (m == -INFINITY) at = 0;  // a row without a finite logit: the first place, as the argmax has it
        float z = 0.0f;
        if (t > 0.0f && m != -INFINITY)
            for (int c = lane; c < b.chunks; c += 16) {
                const ChunkStat x = st[c];
                if (x.m != -INFINITY) z += x.sum * weight32(x.m, m, c32);
            }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) z += __shfl_xor(z, off, 64);
        if (lane == 0) {
            sm[i] = m;
            sat[i] = at;
            sz[i] = z;
            ok[i] = t <= 0.0f ? y == (uint32_t)at
                              : m != -INFINITY && (double)u * (double)qy * (double)z < weight(xy, m, 1.0 / (double)t);
        }
    }
    __syncthreads();
    int a = 0;
    while (a < k && ok[a]) ++a;
    return {k, a, row0 + a, sm[a], sat[a], sz[a], t, 0};
}

// Where the emission row's weights come from: of p, or of the rest that the
// rejected draft leaves.
struct Rest {
    const float* x;
    const float* q;  // the rejected draft's probabilities, or null: p ...
    uint32_t out;    // ... without a certain draft's own column (none: 0xffffffff)
};
__device__ inline Rest rest_of(const VerifyBufs& b, const VerifyArgs& v, int s, const Decision& d) {
    const size_t at = (size_t)(v.row[s] - s + d.accepted);
    const bool left = d.accepted < d.drafts;
    return {b.logits + (size_t)d.row * b.cols, left && b.probs ? b.probs + at * b.cols : nullptr,
            left && !b.probs ? b.drafts[at] : 0xffffffffu};
}

__device__ inline double wave_sum(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += shfl_xor64(v, off);
    return v;
}

template <bool VEC>
__global__ __launch_bounds__(256) void verify_rest_kernel(VerifyBufs b, VerifyArgs v) {
    __shared__ double ss[3][4];
    constexpr int E = kRestChunk / 256;
    const int s = blockIdx.x / b.rest_chunks, ch = blockIdx.x - s * b.rest_chunks, tid = threadIdx.x;
    const Decision d = decide(b, v, s);
    if (ch == 0 && tid == 0) b.dec[s] = d;
    if (d.t <= 0.0f || d.z <= 0.0f) return;  // greedy, or nothing weighs: the first largest logit
    const Rest r = rest_of(b, v, s, d);
    const int c0 = ch * kRestChunk;
    float x[E], q[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        x[e] = -INFINITY;
        q[e] = 0.0f;
    }
    if constexpr (VEC) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const int c = c0 + e * 256 + tid * 4;
            if (c < b.cols) {
                *(float4*)(x + e) = *(const float4*)(r.x + c);
                if (r.q) *(float4*)(q + e) = *(const float4*)(r.q + c);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = c0 + e * 256 + tid;
            if (c < b.cols) {
                x[e] = r.x[c];
                if (r.q) q[e] = r.q[c];
            }
        }
    }
    const double inv_t = 1.0 / (double)d.t, z = d.z;
    double w = 0.0, wa = 0.0, qa = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = VEC ? c0 + (e / 4) * 1024 + tid * 4 + (e & 3) : c0 + e * 256 + tid;
        const double we = weight(x[e], d.m, inv_t), qe = fmaxf(q[e], 0.0f);
        w += we;
        const bool in = r.q ? we > qe * z : (uint32_t)c != r.out;
        wa += in ? we : 0.0;
        qa += in ? qe : 0.0;
    }
    w = wave_sum(w);
    wa = wave_sum(wa);
    qa = wave_sum(qa);
    if ((tid & 63) == 0) {
        ss[0][tid >> 6] = w;
        ss[1][tid >> 6] = wa;
        ss[2][tid >> 6] = qa;
    }
    __syncthreads();
    if (tid == 0) {
        double o[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) o[i] = (ss[i][0] + ss[i][1]) + (ss[i][2] + ss[i][3]);
        b.rest[(size_t)s * b.rest_chunks + ch] = {o[0], o[1], o[2]};
    }
}

// A workgroup of 4 waves per sequence.
__global__ __launch_bounds__(256) void verify_emit_kernel(VerifyBufs b, VerifyArgs v) {
    __shared__ double sw[4];
    __shared__ double s_before, s_target, s_z;
    __shared__ int s_chunk, s_first, s_last;
    __shared__ bool s_whole;
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Decision d = b.dec[s];
    uint32_t token = (uint32_t)d.at;
    if (d.t > 0.0f && d.z > 0.0f) {
        const Rest r = rest_of(b, v, s, d);
        if (wave == 0) {
            const RestSum* rs = b.rest + (size_t)s * b.rest_chunks;
            const double u = b.u[v.row[s] + d.drafts];
            double z = 0.0, total = 0.0;
            for (int c = lane; c < b.rest_chunks; c += 64) z += rs[c].w;
            z = wave_sum(z);
            bool whole = false;  // the rest weighs nothing (by rounding): the token comes from p
            auto chunk_sum = [&](int c) {
                const RestSum x = rs[c];
                return whole ? x.w : r.q ? __builtin_fmax(__builtin_fma(-x.qa, z, x.wa), 0.0) : x.wa;
            };
            for (int pass = 0; pass < 2; ++pass) {
                total = 0.0;
                for (int c = lane; c < b.rest_chunks; c += 64) total += chunk_sum(c);
                total = wave_sum(total);
                if (total > 0.0) break;
                whole = true;
            }
            const double target = u * total;
            // the first chunk whose end exceeds the target; none (u >= 1 or not a number): the last that weighs
            double before = 0.0, pick_before = 0.0;
            int chunk = 0;
            bool found = false;
            for (int c0 = 0; c0 < b.rest_chunks && !found; c0 += 64) {
                const double w = c0 + lane < b.rest_chunks ? chunk_sum(c0 + lane) : 0.0;
                double run = w;
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) {
                    const double up = shfl_up64(run, off);
                    if (lane >= off) run += up;
                }
                const unsigned long long hit = __ballot(w > 0.0 && before + run > target), some = __ballot(w > 0.0);
                const double up1 = shfl_up64(run, 1), start = lane ? up1 : 0.0;  // (every lane takes part in the shuffle)
                if (some) {
                    const int pick = hit ? __ffsll(hit) - 1 : 63 - __clzll(some);
                    chunk = c0 + pick;
                    pick_before = before + __hiloint2double(__shfl(__double2hiint(start), pick, 64),
                                                            __shfl(__double2loint(start), pick, 64));
                    found = hit != 0;
                }
                before += __hiloint2double(__shfl(__double2hiint(run), 63, 64), __shfl(__double2loint(run), 63, 64));
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
        constexpr int E = kRestChunk / 256;
        const int c0 = s_chunk * kRestChunk + tid * E;
        const double inv_t = 1.0 / (double)d.t, z = s_z;
        const bool whole = s_whole;
        float x[E], q[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = c0 + e < b.cols ? r.x[c0 + e] : -INFINITY;
            q[e] = r.q && c0 + e < b.cols ? fmaxf(r.q[c0 + e], 0.0f) : 0.0f;
        }
        double w[E], sum = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            w[e] = weight(x[e], d.m, inv_t);
            if (!whole) w[e] = r.q ? __builtin_fmax(w[e] - (double)q[e] * z, 0.0) : (uint32_t)(c0 + e) == r.out ? 0.0 : w[e];
            sum += w[e];
        }
        double run = sum;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const double up = shfl_up64(run, off);
            if (lane >= off) run += up;
        }
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
        if (first != 0x7fffffff) atomicMin(&s_first, first);
        if (last >= 0) atomicMax(&s_last, last);
        __syncthreads();
        // (no crossing: the chunk's sum and this one's order differ in their last bits, or u >= 1)
        token = s_first != 0x7fffffff ? (uint32_t)s_first : s_last >= 0 ? (uint32_t)s_last : (uint32_t)d.at;
    }
    const uint32_t* y = b.drafts + (v.row[s] - s);
    for (int i = tid; i < b.out_stride; i += 256)
        b.out[(size_t)s * b.out_stride + i] = i < d.accepted ? y[i] : i == d.accepted ? token : 0xffffffffu;
    if (tid == 0) b.accepted[s] = d.accepted;
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
    const size_t stat_bytes = sizeof(ChunkStat) * (size_t)rows * chunks;
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
        ctx->verify_ws_bytes = need;
    }
    hipEvent_t ev;
    timing_mark_begin(ctx, kClassOther, &ev);
    size_t row0 = 0, draft0 = 0;
    for (int s0 = 0; s0 < n; s0 += kSeqs) {
        const int m = std::min(kSeqs, n - s0);
        VerifyArgs v;
        int r = 0;
        for (int s = 0; s < kSeqs; ++s) {
            v.row[s] = r;
            v.temp[s] = s < m ? vb->temperature[s0 + s] : 0.0f;
            if (s < m) r += vb->draft_len[s0 + s] + 1;
        }
        v.row[kSeqs] = r;
        VerifyBufs b;
        b.logits = d_logits + row0 * cols;
        b.cols = cols;
        b.chunk = chunk;
        b.chunks = chunks;
        b.drafts = vb->d_drafts + draft0;
        b.probs = vb->d_draft_probs ? vb->d_draft_probs + draft0 * cols : nullptr;
        b.u = vb->d_uniforms + row0;
        b.stat = (ChunkStat*)ctx->verify_ws + row0 * chunks;
        b.dec = (Decision*)((char*)ctx->verify_ws + stat_bytes) + s0;
        b.rest = (RestSum*)((char*)ctx->verify_ws + stat_bytes + dec_bytes) + (size_t)s0 * rest_chunks;
        b.rest_chunks = rest_chunks;
        b.out = d_out + (size_t)s0 * out_stride;
        b.out_stride = out_stride;
        b.accepted = d_accepted + s0;
        const bool vec = cols % 4 == 0 && ((uintptr_t)d_logits & 15) == 0;
        auto stats = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(r * chunks), dim3(256), 0, ctx->stream, b, v, m);
        };
        switch (e) {
            case 1: if (vec) stats(verify_stats_kernel<1, true>); else stats(verify_stats_kernel<1, false>); break;
            case 2: if (vec) stats(verify_stats_kernel<2, true>); else stats(verify_stats_kernel<2, false>); break;
            case 4: if (vec) stats(verify_stats_kernel<4, true>); else stats(verify_stats_kernel<4, false>); break;
            default: if (vec) stats(verify_stats_kernel<8, true>); else stats(verify_stats_kernel<8, false>); break;
        }
        ZR_LAUNCH_CHECK(ctx);
        if (vec && ((uintptr_t)vb->d_draft_probs & 15) == 0)
            hipLaunchKernelGGL(verify_rest_kernel<true>, dim3(m * rest_chunks), dim3(256), 0, ctx->stream, b, v);
        else
            hipLaunchKernelGGL(verify_rest_kernel<false>, dim3(m * rest_chunks), dim3(256), 0, ctx->stream, b, v);
        ZR_LAUNCH_CHECK(ctx);
        hipLaunchKernelGGL(verify_emit_kernel, dim3(m), dim3(256), 0, ctx->stream, b, v);
        ZR_LAUNCH_CHECK(ctx);
        row0 += r;
        draft0 += r - m;
    }
    timing_mark_end(ctx, kClassOther, ev);
    return ZR_OK;
}

}  // namespace zr
