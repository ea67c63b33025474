// Attention of sequences that share their leading pages (forked sessions, one
// system prompt for many): every shared page is read once for the query rows
// of all its holders.  No counterpart in the reference, whose sessions own
// their pages; the rows' values are those of forward_pass.rs:2764-2895:
//   o = softmax(q . K^T / sqrt(d)) . V over the row's visible keys.
//
// A segment is a run of pages that the block tables of two or more sequences
// name at the same place.  Its keys precede every new row of its holders, so
// all of their rows see all of them.  Over disjoint key sets i the softmax
// splits into (m_i, l_i, o_i) = (max s, sum 2^(s - m_i), sum 2^(s - m_i) v):
//   M = max m_i,  o = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M).
// One launch takes the segments (units) and every decode tile's own pages
// (tails) and leaves partials; shared_merge_kernel joins those of a row.
//
// A unit is bound by the MFMAs (each page serves up to 128 columns), a tail by
// its pages; the two kinds of workgroup run side by side on a CU, two of 4 waves
// each.  Launch + merge, us, 128-wide heads: 256 sessions behind four prompts of 2040
// rows, 32 / 8 heads, 116 + 8 (519 MB, mostly their own pages; read one by one 2.6
// GB); 48 x 5 rows behind 4011, 16 / 4 heads, 44 + 7 (25 GFLOP executed); 16 behind
// 8000, 32 / 8 heads, 21 + 5.
#include "attn_tile.h"
#include "zr_internal.h"

namespace zr {

struct SharedArgs {
    const float* q;       // [T, q_cols]
    int q_cols;
    const void* pool;     // layer base of the pool
    size_t page_elems;
    int stride;           // block table row stride (the table is a kernel argument)
    const int* units;     // kUnitInts per work unit (zr_internal.h)
    const int4* rec;      // three records per tail, longest first (AttnArgs::rec)
    int n_units, n_tails;
    int unit_groups;      // of 8 workgroups
    int G, kv_heads;
    float scale_log2;     // log2(e) / sqrt(d)
    float* part;          // [items][kv_heads][16][D + 2]
};

// Q^T fragments (B operand) of a column: lane holds Q[col][16 ks + 8 h + j]
// log2(e) / sqrt(d) in three bf16 parts (scores come out in log2 units).
template <int D> struct SharedQ {
    f32x4 x[D / 16][2];
    __device__ __forceinline__ void load(const float* qp) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            x[ks][0] = *(const f32x4*)(qp + 16 * ks);
            x[ks][1] = *(const f32x4*)(qp + 16 * ks + 4);
        }
    }
    __device__ __forceinline__ void split(float scale, int ks, bf16x8 (&q)[3]) const {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[ks][j >> 2][j & 3] * scale;
        split3_bf16x8(y, q);
    }
};

// A unit's page ids, 64 at a time, one per lane: a tile's two come by lane reads,
// so that no table load stands before its copies.  The first 64 lie in the unit's
// record.  Tiles are asked for in order; one past the segment's end repeats its
// last page.
struct SharedPages {
    const int* bt;   // the sequence's table from the unit's first page on
    int last;        // last page of the segment, counted from there
    int base, ids;
    __device__ __forceinline__ void fetch(int lane) {
        ids = bt[min(base + lane, last)];
        // (waited for here, in the rare branch: left pending, the lane reads behind the
        // branch would wait for every copy in flight, each step)
        asm volatile("" : "+v"(ids));
    }
    __device__ __forceinline__ void tile(int rel, int lane, int& pg0, int& pg1) {
        if (2 * rel >= base + 64) {
            base = (2 * rel) & ~63;
            fetch(lane);
        }
        pg0 = __builtin_amdgcn_readlane(ids, 2 * rel - base);
        pg1 = __builtin_amdgcn_readlane(ids, 2 * rel - base + 1);
    }
};

// V rows of keys outside [0, last] enter the product as 0: their weights are 0,
// but 0 x inf is NaN, and rows before a trimmed window hold whatever they held.
// Element j of a fragment is key base + at + 8 (j / 4) + j % 4.
template <int D>
__device__ __forceinline__ void shared_mask_v(bf16x8 (&v)[D / 32], int base, int at, int last) {
    asm volatile("" ::: "memory");  // (keeps the caller's branch: the selects cost every tile otherwise)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int key = base + at + 8 * (j >> 2) + (j & 3);
        if (key < 0 || key > last)
#pragma unroll
            for (int db = 0; db < D / 32; ++db) v[db][j] = (__bf16)0.0f;
    }
}

// The key slices' (m, l, O) of each column meet in LDS (slices 1.. write, slice
// 0 rescales all to the largest m and adds), then the column goes out as one
// split's partial of its 16-column group.
constexpr size_t shared_combine_bytes(int D, int CW, int KW) {
    return (size_t)(KW - 1) * CW * (2 + 16 * (D / 32)) * 64 * 4;
}

template <int D, int CW, int KW>
__device__ __forceinline__ void shared_finish(const SharedArgs& a, f32x16 (&o)[D / 32], float m, float lsum, float* buf,
                                              int slice, int wq, int lane, int kvh, int item0, int nsplits, bool valid) {
    const int h = lane >> 5, col = wq * 32 + (lane & 31);
    lsum = pair_sum(lsum);
    if constexpr (KW > 1) {
        constexpr int W = 2 + 16 * (D / 32);  // floats per column lane
        __syncthreads();                      // the ring is free: every wave has read its last tile
        if (slice > 0) {
            float* c = buf + ((size_t)((slice - 1) * CW + wq) * W) * 64 + lane;
            c[0] = m;
            c[64] = lsum;
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) c[(2 + db * 16 + i) * 64] = o[db][i];
        }
        __syncthreads();
        if (slice > 0) return;
        const float* c = buf + (size_t)wq * W * 64 + lane;
        constexpr size_t step = (size_t)CW * W * 64;
        float mm = m;
#pragma unroll
        for (int k = 0; k < KW - 1; ++k) mm = fmaxf(mm, c[k * step]);
        // (a slice with no tile has m = -inf, l = 0, O = 0: weight 0)
        const float a0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mm);
        lsum *= a0;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] *= a0;
#pragma unroll
        for (int k = 0; k < KW - 1; ++k) {
            const float mk = c[k * step];
            const float ak = mk == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mk - mm);
            lsum += c[k * step + 64] * ak;
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] += c[k * step + (2 + db * 16 + i) * 64] * ak;
        }
        m = mm;
    }
    if (!valid) return;
    float* out = a.part + (((size_t)(item0 + (col >> 4) * nsplits) * a.kv_heads + kvh) * 16 + (col & 15)) * (D + 2);
    if (h == 0) *(float2*)out = make_float2(m, lsum);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            float2* p = (float2*)(out + 2 + db * 32 + 8 * i4 + 4 * h);  // partial rows are 8-byte aligned
            p[0] = make_float2(o[db][4 * i4], o[db][4 * i4 + 1]);
            p[1] = make_float2(o[db][4 * i4 + 2], o[db][4 * i4 + 3]);
        }
}

// bf16 pools.  A workgroup of CW x KW waves owns one kv head of one unit: up to
// 32 CW columns = (row, q head of the kv head) pairs, 32 per column wave, and a
// run of 32-key tiles (two pages) of the segment.  Tiles go to the KW key
// slices in turn; each is copied once into LDS by the CW waves of its slice
// (buffer loads into LDS, the pool's page order, no registers) and serves all
// columns.  Per tile and wave, on v_mfma_f32_32x32x16_bf16 (h = lane / 32):
//   S[key][col] = sum_d K[key][d] Q[col][d]; the lane gets key 8 (i / 4) + 4 h + i % 4, i < 16
//   online softmax per column over the lane's 16 keys and the 16 of lane ^ 32
//   O[d][col] += sum_key V[key][d] P[key][col]: P's fragment is the lane's own scores
// Q and P enter in three bf16 parts, which hold all of an f32's 24 bits (two
// parts, 17 bits, put the result 4e-6 of its norm off: 3.4e-6 from Q, 2.2e-6
// from P; three leave 1e-7), K and V are exact; sums are f32.
//
// NEXT: step t weighs tile t's scores while the MFMAs form those of tile t + 1
// (the matrix pipe and the VALU work side by side on one wave's instructions),
// then adds V^T P of tile t.  K and V have rings of three slots each, K one tile
// ahead, and at D = 128 the third part of Q lies in LDS: 80 KB, two workgroups a
// CU, and no spills (a spilled register's reload waits, in order, for the copies
// issued before it).  Without NEXT two slots and one tile at a time.
constexpr bool unit_q_in_lds(int D, bool next) { return D == 128 && next; }
constexpr size_t unit_lds(int D, int CW, int KW, bool next) {
    return (size_t)(next ? 3 : 2) * KW * 8 * D * 16 + (unit_q_in_lds(D, next) ? (size_t)CW * KW * (D / 16) * 1024 : 0);
}

template <int D, int CW, int KW, bool NEXT>
__device__ __forceinline__ void shared_unit(const SharedArgs& a, const int* __restrict__ block_tables, int wg, bf16x8* buf) {
    constexpr int SLOTS = NEXT ? 3 : 2;
    constexpr int HALF = 4 * D;          // 16 B chunks of a tile's K (or V): 2 pages x 16 rows x D bf16
    constexpr int VM = HALF / 64 / CW;   // copies (1 KiB each) per wave and half tile
    constexpr int RUN = D / 32;          // 1 KiB runs of one head's K (or V) page
    constexpr bool QLDS = unit_q_in_lds(D, NEXT);
    static_assert(VM * 64 * CW == HALF, "tile copy split");
    static_assert(shared_combine_bytes(D, CW, KW) <= (size_t)SLOTS * KW * 2 * HALF * 16, "combine buffer");

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slice = wave / CW, wq = wave - slice * CW;
    const int rank = __builtin_amdgcn_readfirstlane(wg / a.kv_heads);
    const int kvh = wg - rank * a.kv_heads;
    if (rank >= a.n_units) return;
    // everything the copies and the Q loads need comes in one round trip
    const int* unit = a.units + (size_t)rank * kUnitInts;
    const int4 u0 = ((const int4*)unit)[0], u1 = ((const int4*)unit)[1];
    const int ids = unit[kUnitPages + lane];
    const int c = wq * 32 + (lane & 31);
    const int rloc = c / a.G, g = c - rloc * a.G;
    const int grow = unit[kUnitRows + rloc];  // (columns past the unit's rows compute its last row, unused)
    const int seq = __builtin_amdgcn_readfirstlane(u0.x), foff = __builtin_amdgcn_readfirstlane(u0.y);
    const int nrows = __builtin_amdgcn_readfirstlane(u0.z & 0xffff), nsplits = __builtin_amdgcn_readfirstlane(u0.z >> 16);
    const int pb = __builtin_amdgcn_readfirstlane(u0.w), pe = __builtin_amdgcn_readfirstlane(u1.w);
    const int kt0 = __builtin_amdgcn_readfirstlane(u1.x), kt1 = __builtin_amdgcn_readfirstlane(u1.y);
    const int item0 = __builtin_amdgcn_readfirstlane(u1.z);
    if (nrows == 0) return;  // an empty record past a replayed bucket's units
    const int h = lane >> 5;
    const bool valid = rloc < nrows;
    const bool busy = wq * 32 < nrows * a.G;  // the wave has a column
    // (keys before the window lie in the segment's first page, before row foff; those past its end in its last tile)
    const int jlast = (pe - pb) * kPageRows - 1;

    const int p0 = pb + 2 * kt0;  // the unit's first page
    SharedPages pages{block_tables + (size_t)seq * a.stride + p0, pe - 1 - p0, 0, ids};
    // Copies are buffer loads into LDS over one page: its base in the (scalar)
    // buffer descriptor, kept from a tile's K for its V, the lane's 16 B and the
    // wave's run in the vector offset, K or V in the scalar one.
    const uint32_t page_bytes = (uint32_t)(a.page_elems * 2);
    const uint32_t k_off = (uint32_t)kvh * (kPageRows * D * 2), v_off = (uint32_t)a.kv_heads * (kPageRows * D * 2) + k_off;
    auto page_rsrc = [&](int pg) {
        const unsigned char* at = (const unsigned char*)a.pool + (uint64_t)(uint32_t)pg * page_bytes;
        return __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, page_bytes, 0x00020000);
    };
    __amdgpu_buffer_rsrc_t rs0, rs1;  // the two pages of the tile asked for last
    auto tile = [&](int x) {
        int pg0, pg1;
        pages.tile(KW * x + slice, lane, pg0, pg1);
        rs0 = page_rsrc(pg0);
        rs1 = page_rsrc(pg1);
    };
    auto k_slot = [&](int x) { return buf + (size_t)((x % SLOTS) * KW + slice) * 2 * HALF; };
    auto v_slot = [&](int x) { return k_slot(x) + HALF; };
    // the tile's K or V into `to`: the wave takes 1 KiB runs i CW + wq of (page, run)
    auto issue = [&](bf16x8* to, uint32_t off) {
#pragma unroll
        for (int i = 0; i < VM; ++i) {
            const int f = i * CW;
            if constexpr (CW <= RUN) {  // (i, not the wave, tells the page)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(f / RUN ? rs1 : rs0, (lds_void*)(to + (f + wq) * 64), 16,
                                                         lane * 16 + wq * 1024, off + f % RUN * 1024, 0, 0);
            } else {  // CW = 2 RUN: a run a wave
                __builtin_amdgcn_raw_ptr_buffer_load_lds(wq / RUN ? rs1 : rs0, (lds_void*)(to + wq * 64), 16,
                                                         lane * 16 + wq % RUN * 1024, off, 0, 0);
            }
        }
    };
    static_assert(CW <= RUN || CW == 2 * RUN, "a tile's copies by wave");

    f32x16 o[D / 32];
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
    float m = -INFINITY, lsum = 0.0f;

    // step x holds tile kt0 + KW x + slice; the rows' Q goes out behind the first
    // tile's copies
    const int nsteps = (kt1 - kt0 + KW - 1) / KW;
    tile(0);
    issue(k_slot(0), k_off);
    SharedQ<D> qx;
    qx.load(a.q + (size_t)grow * a.q_cols + (size_t)(kvh * a.G + g) * D + 8 * h);
    issue(v_slot(0), v_off);
    if constexpr (NEXT) {  // (V of step x and K of step x + 1 are waited for together)
        tile(1);
        issue(k_slot(1), k_off);
        issue(v_slot(1), v_off);
        tile(2);
        issue(k_slot(2), k_off);
    }
    constexpr int QR = QLDS ? 2 : 3;  // parts of Q in registers
    bf16x8 q[D / 16][QR];
    bf16x8* q_lds = buf + (size_t)SLOTS * KW * 2 * HALF + (size_t)wave * (D / 16) * 64 + lane;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        bf16x8 part[3];
        qx.split(a.scale_log2, ks, part);
#pragma unroll
        for (int i = 0; i < QR; ++i) q[ks][i] = part[i];
        if constexpr (QLDS) q_lds[ks * 64] = part[2];  // (read by this lane alone)
    }

    const int kbase = ((lane >> 4) & 1) * 2 * D + (lane & 15) + h * 16;  // page (l % 32) / 16, row l % 16
    auto q_part = [&](int ks, int i) -> bf16x8 {
        if constexpr (QLDS) {
            if (i == 2) return q_lds[ks * 64];
        }
        return q[ks][i < QR ? i : 0];
    };
    f32x16 s;
    auto first_scores = [&](int x) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const bf16x8 kf = k_slot(x)[kbase + 2 * ks * 16];
#pragma unroll
            for (int i = 0; i < 3; ++i) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q_part(ks, i), s, 0, 0, 0);
        }
    };
    if constexpr (NEXT) {
        ring_barrier<4 * VM>();  // K of step 0: four halves were issued after it
        if (busy) first_scores(0);
    }
    for (int t = 0; t < nsteps; ++t) {
        // V of step t and K of step t + 1 (without NEXT: both of step t) have
        // arrived, and every wave is done with step t - 1
        if constexpr (NEXT) {
            if (t + 1 < nsteps || t == 0) ring_barrier<2 * VM>(); else ring_barrier<0>();
            if (t + 2 < nsteps) {
                issue(v_slot(t + 2), v_off);  // its pages are the ones asked for last
                tile(t + 3);
                issue(k_slot(t + 3), k_off);
            }
        } else {
            ring_barrier<0>();
            if (t + 1 < nsteps) {
                tile(t + 1);
                issue(k_slot(t + 1), k_off);
                issue(v_slot(t + 1), v_off);
            }
        }
        if (!busy) continue;
        const int kt = kt0 + KW * t + slice;
        const bool edge = 32 * kt < foff || 32 * kt + 31 > jlast || kt >= kt1;
        const int last = kt < kt1 ? jlast - foff : -1;  // (a slice without a tile in this step sees no key)
        if constexpr (!NEXT) first_scores(t);
        if (edge) prefill_mask(s, 32 * kt + 4 * h - foff, last);
        // The running max follows a tile's only by jumps of more than 8 (log2 units:
        // P <= 2^8), so O and l are rescaled at the first tile and rarely after.
        float tmax = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) tmax = fmaxf(tmax, s[i]);
        tmax = pair_max(tmax);
        if (__any(tmax > m + 8.0f)) {
            const bool up = tmax > m + 8.0f;  // (m = -inf and no visible key: no move, where m - m would be NaN)
            const float alpha = up ? __builtin_amdgcn_exp2f(m - tmax) : 1.0f;
            if (up) m = tmax;
            lsum *= alpha;
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
        }
        const float mu = m == -INFINITY ? 0.0f : m;
        // The tile's 16 weights a lane, in D / 16 pieces, each behind the three MFMAs of
        // one K fragment of the next tile.  In this order by fences: left to itself
        // the compiler issues the 24 MFMAs, each waiting for the one before, and
        // then the VALU work.  (The last step's next tile is what its slot holds,
        // unused.)
        f32x16 next;
        uint32_t pw[2][3][4];           // P's parts, two weights a word
        constexpr int PIECE = 256 / D;  // weights per piece
        const bf16x8* k_next = k_slot(t + 1) + kbase;
        bf16x8 kf;
        if constexpr (NEXT) {
#pragma unroll
            for (int i = 0; i < 16; ++i) next[i] = 0.0f;
            kf = k_next[0];
        }
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            __builtin_amdgcn_sched_barrier(0);
            bf16x8 q2, ahead;
            if constexpr (NEXT) {
                q2 = q_part(ks, 2);
                ahead = ks + 1 < D / 16 ? k_next[2 * (ks + 1) * 16] : kf;
                next = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q[ks][0], next, 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            float w[PIECE];
#pragma unroll
            for (int e = 0; e < PIECE; ++e) {
                w[e] = __builtin_amdgcn_exp2f(s[ks * PIECE + e] - mu);
                lsum += w[e];
            }
            if constexpr (NEXT) {
                __builtin_amdgcn_sched_barrier(0);
                next = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q[ks][1], next, 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int e = 0; e < PIECE; e += 2) {
                const int at = ks * PIECE + e;
                split3_pair(w[e], w[e + 1], pw[at >> 3], (at & 7) >> 1);
            }
            if constexpr (NEXT) {
                __builtin_amdgcn_sched_barrier(0);
                next = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, q2, next, 0, 0, 0);
                kf = ahead;
            }
        }
        bf16x8 p[2][3];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                p[k][i] = __builtin_bit_cast(bf16x8, make_uint4(pw[k][i][0], pw[k][i][1], pw[k][i][2], pw[k][i][3]));
                // (P is complete here: its work must not sink past the branch below)
                asm volatile("" ::"v"(p[k][i]));
            }
        __builtin_amdgcn_sched_barrier(0);
        // V^T P by 16 keys: a fragment's registers take the other 16 keys' once its three MFMAs are out
        const bf16x4* sv = (const bf16x4*)v_slot(t) + (h * 16 + (lane & 15)) * 2 + ((lane >> 4) & 1);
        auto v_frag = [&](int ks2, int db) {
            const bf16x4* at = sv + ks2 * 4 * D + db * 128;  // page ks2's V block, in 8-byte units
            return __builtin_shufflevector(at[0], at[64], 0, 1, 2, 3, 4, 5, 6, 7);
        };
        bf16x8 vf[D / 32];
#pragma unroll
        for (int db = 0; db < D / 32; ++db) vf[db] = v_frag(0, db);
        if (edge) shared_mask_v<D>(vf, 32 * kt - foff, 4 * h, last);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[db], p[0][i], o[db], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            vf[db] = v_frag(1, db);
        }
        if (edge) shared_mask_v<D>(vf, 32 * kt - foff, 16 + 4 * h, last);
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int i = 0; i < 3; ++i)
                o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[db], p[1][i], o[db], 0, 0, 0);
        if constexpr (NEXT) s = next;
    }
    // (copies issued for steps that do not run land before the combine's barrier)
    ring_barrier<0>();
    shared_finish<D, CW, KW>(a, o, m, lsum, (float*)buf, slice, wq, lane, kvh, item0, nsplits, valid);
}

// f32 pools: K, V, Q and P each enter the MFMA in three bf16 parts; of the nine
// products of a pair the six above 2^-24 of the result are formed (two parts and
// three products are 8e-6 of the result's norm off).  A tile is split once
// per workgroup: each wave loads its share of the next tile's f32 runs into
// registers a step ahead, splits them and stores three planes in the LDS order
// of a bf16 tile, two slots deep, one barrier per step.
constexpr size_t unit_f32_lds(int D) { return (size_t)2 * 3 * 8 * D * 16; }

template <int D>
__device__ __forceinline__ void shared_unit_f32(const SharedArgs& a, const int* __restrict__ block_tables, int wg,
                                                bf16x8* buf) {
    constexpr int CW = 4, KW = 1;
    constexpr int CHUNKS = 8 * D;         // 16 B chunks per plane of a tile
    constexpr int VM = CHUNKS / 64 / CW;  // 512-element runs per wave and tile
    constexpr int RUN = D / 32;
    static_assert(VM * 64 * CW == CHUNKS, "tile copy split");
    auto lds = [&](int slot, int part) { return buf + (size_t)(slot * 3 + part) * CHUNKS; };

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slice = wave / CW, wq = wave - slice * CW;
    const int rank = __builtin_amdgcn_readfirstlane(wg / a.kv_heads);
    const int kvh = wg - rank * a.kv_heads;
    if (rank >= a.n_units) return;
    // everything the copies and the Q loads need comes in one round trip
    const int* unit = a.units + (size_t)rank * kUnitInts;
    const int4 u0 = ((const int4*)unit)[0], u1 = ((const int4*)unit)[1];
    const int ids = unit[kUnitPages + lane];
    const int c = wq * 32 + (lane & 31);
    const int rloc = c / a.G, g = c - rloc * a.G;
    const int grow = unit[kUnitRows + rloc];  // (columns past the unit's rows compute its last row, unused)
    const int seq = __builtin_amdgcn_readfirstlane(u0.x), foff = __builtin_amdgcn_readfirstlane(u0.y);
    const int nrows = __builtin_amdgcn_readfirstlane(u0.z & 0xffff), nsplits = __builtin_amdgcn_readfirstlane(u0.z >> 16);
    const int pb = __builtin_amdgcn_readfirstlane(u0.w), pe = __builtin_amdgcn_readfirstlane(u1.w);
    const int kt0 = __builtin_amdgcn_readfirstlane(u1.x), kt1 = __builtin_amdgcn_readfirstlane(u1.y);
    const int item0 = __builtin_amdgcn_readfirstlane(u1.z);
    if (nrows == 0) return;
    const int h = lane >> 5;
    const bool valid = rloc < nrows;
    const bool busy = wq * 32 < nrows * a.G;
    const int jlast = (pe - pb) * kPageRows - 1;

    const int p0 = pb + 2 * kt0;
    SharedPages pages{block_tables + (size_t)seq * a.stride + p0, pe - 1 - p0, 0, ids};
    const size_t kv_tile = (size_t)kPageRows * D;
    const size_t v_block = (size_t)a.kv_heads * kv_tile;
    const float* pool = (const float*)a.pool + (size_t)kvh * kv_tile + 4 * lane;
    f32x4 raw[VM][2];
    auto load_raw = [&](int pg0, int pg1) {
#pragma unroll
        for (int i = 0; i < VM; ++i) {
            const int f = i * CW + wq;
            const int pp = f / (2 * RUN), kv = (f / RUN) & 1, run = f % RUN;
            const f32x4* src =
                (const f32x4*)(pool + (size_t)(pp ? pg1 : pg0) * a.page_elems + (kv ? v_block : 0) + (size_t)run * 512);
            raw[i][0] = src[0];
            raw[i][1] = src[kWave];
        }
    };
    auto store_split = [&](int slot) {
#pragma unroll
        for (int i = 0; i < VM; ++i) {
            const int f = i * CW + wq;
            const float x[8] = {raw[i][0][0], raw[i][0][1], raw[i][0][2], raw[i][0][3],
                                raw[i][1][0], raw[i][1][1], raw[i][1][2], raw[i][1][3]};
            bf16x8 p[3];
            split3_bf16x8(x, p);
#pragma unroll
            for (int k = 0; k < 3; ++k) lds(slot, k)[f * 64 + lane] = p[k];
        }
    };

    f32x16 o[D / 32];
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
    float m = -INFINITY, lsum = 0.0f;
    const int nsteps = (kt1 - kt0 + KW - 1) / KW;
    int pg0, pg1;
    pages.tile(slice, lane, pg0, pg1);
    load_raw(pg0, pg1);
    SharedQ<D> qx;
    qx.load(a.q + (size_t)grow * a.q_cols + (size_t)(kvh * a.G + g) * D + 8 * h);
    store_split(0);
    bf16x8 q[D / 16][3];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qx.split(a.scale_log2, ks, q[ks]);
    pages.tile(KW + slice, lane, pg0, pg1);
    load_raw(pg0, pg1);

    auto v_frags = [&](const bf16x8* plane, bf16x8 (&v)[2][D / 32]) {
        const bf16x4* sv = (const bf16x4*)plane;
#pragma unroll
        for (int ks2 = 0; ks2 < 2; ++ks2) {
            const int vbase = (2 * ks2 + 1) * 4 * D;
#pragma unroll
            for (int db = 0; db < D / 32; ++db) {
                const int u = ((db * 4 + h) * 16 + (lane & 15)) * 2 + ((lane >> 4) & 1);
                const bf16x4 v0 = sv[vbase + u], v1 = sv[vbase + u + 2 * 16 * 2];
                v[ks2][db] = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        }
    };

    auto mask_v = [&](bf16x8 (&v)[2][D / 32], int kt) {
        shared_mask_v<D>(v[0], 32 * kt - foff, 4 * h, jlast - foff);
        shared_mask_v<D>(v[1], 32 * kt - foff, 16 + 4 * h, jlast - foff);
    };
    for (int t = 0; t < nsteps; ++t) {
        ring_barrier<63>();  // the slot is written (LDS only: the next tile's loads stay in flight)
        const int kt = kt0 + KW * t + slice;
        if (busy && kt < kt1) {
            const bf16x8* st[3] = {lds(t & 1, 0), lds(t & 1, 1), lds(t & 1, 2)};
            const int kbase = ((lane >> 4) & 1) * 2 * (2 * D) + (lane & 15);
            f32x16 s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                bf16x8 k[3];
#pragma unroll
                for (int i = 0; i < 3; ++i) k[i] = st[i][kbase + (2 * ks + h) * 16];
#pragma unroll
                for (int i = 0; i < 3; ++i)
#pragma unroll
                    for (int j = 0; j < 3 - i; ++j)
                        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[j], q[ks][i], s, 0, 0, 0);
            }
            const bool edge = 32 * kt < foff || 32 * kt + 31 > jlast;
            bf16x8 vf[2][D / 32];
            v_frags(st[0], vf);
            __builtin_amdgcn_sched_barrier(0);  // the V reads go out before the softmax
            if (edge) {
                prefill_mask(s, 32 * kt + 4 * h - foff, jlast - foff);
                mask_v(vf, kt);
            }
            float pr[16];
            prefill_softmax<D>(s, o, m, lsum, pr);
            bf16x8 p[2][3];
            split3_bf16x8(pr, p[0]);
            split3_bf16x8(pr + 8, p[1]);
#pragma unroll
            for (int j = 0; j < 3; ++j) {  // part j of V with the parts of P that count
#pragma unroll
                for (int ks2 = 0; ks2 < 2; ++ks2)
#pragma unroll
                    for (int i = 0; i < 3 - j; ++i)
#pragma unroll
                        for (int db = 0; db < D / 32; ++db)
                            o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[ks2][db], p[ks2][i], o[db], 0, 0, 0);
                if (j < 2) {
                    v_frags(st[j + 1], vf);
                    if (edge) mask_v(vf, kt);
                }
            }
        }
        if (t + 1 < nsteps) {
            store_split((t + 1) & 1);  // last read in step t - 1, a barrier ago
            if (t + 2 < nsteps) {
                pages.tile(KW * (t + 2) + slice, lane, pg0, pg1);
                load_raw(pg0, pg1);
            }
        }
    }
    shared_finish<D, CW, KW>(a, o, m, lsum, (float*)buf, slice, wq, lane, kvh, item0, nsplits, valid);
}

// A tail: one wave per kv head of one split of a decode tile, 16 columns = (query,
// q head of the kv head) pairs of one sequence, its own pages two at a time
// through a ring of RING page sets in registers (the first four ids in the
// record); the partial goes out.  Per page pair (lane l, column l % 16, quad
// l / 16), on v_mfma_f32_16x16x32_bf16: S^T = K Q^T, an online softmax step over
// 32 keys, O^T += V^T P^T with P^T the lane's own scores.  Q and P (f32 pools: K
// and V) in three bf16 parts as in the units; bound by the pages.
template <int D>
__device__ __forceinline__ f32x4 tail_qk(const PageRegs<uint16_t, D>& pg, const bf16x8* q, int lane) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < D / 32; ++kb)
#pragma unroll
        for (int i = 0; i < 3; ++i)
            s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pg.k[kb], q[(i * (D / 32) + kb) * 64 + lane], s, 0, 0, 0);
    return s;
}

template <int D>
__device__ __forceinline__ f32x4 tail_qk(const PageRegs<float, D>& pg, const bf16x8* q, int lane) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < D / 32; ++kb) {
        float kf[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) kf[j] = pg.k[kb][j >> 2][j & 3];
        bf16x8 k[3];
        split3_bf16x8(kf, k);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const bf16x8 qi = q[(i * (D / 32) + kb) * 64 + lane];
#pragma unroll
            for (int j = 0; j < 3 - i; ++j) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[j], qi, s, 0, 0, 0);
        }
    }
    return s;
}

template <int D>
__device__ __forceinline__ void tail_pv(const PageRegs<uint16_t, D>& pa, const PageRegs<uint16_t, D>& pb,
                                        const bf16x8 (&p)[3], f32x4* o) {
#pragma unroll
    for (int vb = 0; vb < D / 32; ++vb) {
        const bf16x8 v0 = __builtin_shufflevector(pa.v[vb], pb.v[vb], 0, 1, 2, 3, 8, 9, 10, 11);
        const bf16x8 v1 = __builtin_shufflevector(pa.v[vb], pb.v[vb], 4, 5, 6, 7, 12, 13, 14, 15);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            o[2 * vb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, p[i], o[2 * vb], 0, 0, 0);
            o[2 * vb + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, p[i], o[2 * vb + 1], 0, 0, 0);
        }
    }
}

template <int D>
__device__ __forceinline__ void tail_pv(const PageRegs<float, D>& pa, const PageRegs<float, D>& pb,
                                        const bf16x8 (&p)[3], f32x4* o) {
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
        const f32x4 va = pa.v[db >> 1][db & 1], vb = pb.v[db >> 1][db & 1];
        const float vf[8] = {va[0], va[1], va[2], va[3], vb[0], vb[1], vb[2], vb[3]};
        bf16x8 v[3];
        split3_bf16x8(vf, v);
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int j = 0; j < 3 - i; ++j) o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[j], p[i], o[db], 0, 0, 0);
    }
}

constexpr size_t tail_lds(int D) { return (size_t)4 * 3 * (D / 32) * 64 * 16; }

template <typename KV, int D, int RING>
__device__ __forceinline__ void shared_tail(const SharedArgs& a, const int* __restrict__ block_tables, int group,
                                            bf16x8* buf) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Workgroups go to the 8 XCDs round-robin; on each, wave n of the tails takes
    // kv head n % kv_heads of every eighth record, so that all of a tail's pages
    // go through one XCD.
    const int n = group * 4 + wave;
    const int kvh = n % a.kv_heads;
    const int rank = (n / a.kv_heads) * 8 + (blockIdx.x & 7);
    if (rank >= a.n_tails) return;  // (no barrier in a tail)
    const int4 r0 = a.rec[3 * rank], r1 = a.rec[3 * rank + 1], r2 = a.rec[3 * rank + 2];
    const int seq = r0.x, row0 = r0.y, nq = r0.z, page_b = r0.w, page_e = r1.x, foff = r1.z;
    if (nq == 0) return;  // an empty record past a replayed bucket's items
    const int item = (int)((unsigned)r1.w & (kAttnSingle - 1));
    const int c = lane & 15, q4 = lane >> 4;
    const int qi = c / a.G, g = c - qi * a.G;
    const bool valid = qi < nq;                  // (16 is a multiple of G)
    const int jmax = r1.y + (valid ? qi : 0);    // last visible key of the column
    const KV* pool = (const KV*)a.pool;
    const int* bt = block_tables + (size_t)seq * a.stride;
    const size_t kv_tile = (size_t)kPageRows * D;
    const size_t v_block = (size_t)a.kv_heads * kv_tile;
    PageRegs<KV, D> ring[RING];
    auto load_page = [&](PageRegs<KV, D>& r, int page) {
        const KV* base = pool + (size_t)page * a.page_elems + (size_t)kvh * kv_tile;
        r.load(base, base + v_block, lane);
    };
    // the ids of 64 pages at a time, one per lane, so that no table load stands
    // before a page's (past the split's end: its last page again)
    int base = page_b, ids = bt[min(page_b + lane, page_e - 1)];
    auto load_next = [&](PageRegs<KV, D>& r, int p) {
        if (p >= base + 64) {
            base += 64;
            ids = bt[min(base + lane, page_e - 1)];
            asm volatile("" : "+v"(ids));  // waited for in this branch (SharedPages::fetch)
        }
        load_page(r, __builtin_amdgcn_readlane(ids, p - base));
    };
    f32x4 qx[D / 32][2];
    const float* qp = a.q + (size_t)(row0 + (valid ? qi : 0)) * a.q_cols + (size_t)(kvh * a.G + g) * D + q4 * 8;
#pragma unroll
    for (int kb = 0; kb < D / 32; ++kb) {
        qx[kb][0] = *(const f32x4*)(qp + kb * 32);
        qx[kb][1] = *(const f32x4*)(qp + kb * 32 + 4);
    }
    static_assert(RING % 2 == 0 && RING >= 4 && RING - 2 <= 4, "ring of page pairs; the record holds 4 pages");
    const int first_pages[4] = {r2.x, r2.y, r2.z, r2.w};
#pragma unroll
    for (int r = 0; r < RING - 2; ++r) load_page(ring[r], first_pages[r]);
    bf16x8* qs = buf + (size_t)wave * 3 * (D / 32) * 64;
#pragma unroll
    for (int kb = 0; kb < D / 32; ++kb) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = qx[kb][j >> 2][j & 3] * a.scale_log2;
        bf16x8 q3[3];
        split3_bf16x8(x, q3);
#pragma unroll
        for (int i = 0; i < 3; ++i) qs[(i * (D / 32) + kb) * 64 + lane] = q3[i];
    }
    f32x4 o[D / 16];
#pragma unroll
    for (int db = 0; db < D / 16; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, lsum = 0.0f;
    auto step = [&](const PageRegs<KV, D>& pa, const PageRegs<KV, D>& pb, int p, bool has_b) {
        const f32x4 sa = tail_qk<D>(pa, qs, lane);
        const f32x4 sb = tail_qk<D>(pb, qs, lane);
        float sc[8], pmax = -INFINITY;
        const int j0 = p * kPageRows + q4 * 4 - foff;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int ja = j0 + i, jb = ja + kPageRows;
            sc[i] = ja >= 0 && ja <= jmax ? sa[i] : -INFINITY;
            sc[4 + i] = has_b && jb <= jmax ? sb[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) pmax = fmaxf(pmax, sc[i]);
        pmax = quad_max(pmax);
        const float mn = fmaxf(m, pmax);
        const float mu = mn == -INFINITY ? 0.0f : mn;  // no visible key so far
        const float alpha = __builtin_amdgcn_exp2f(m - mu);
        float pr[8], ps = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            pr[i] = __builtin_amdgcn_exp2f(sc[i] - mu);
            ps += pr[i];
        }
        lsum = lsum * alpha + ps;
        m = mn;
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[db][i] *= alpha;
        bf16x8 p3[3];
        split3_bf16x8(pr, p3);
        tail_pv<D>(pa, pb, p3, o);
    };
    for (int p = page_b; p < page_e; p += RING) {
#pragma unroll
        for (int r = 0; r < RING; r += 2) {
            const int pp = p + r;
            if (pp >= page_e) break;
            load_next(ring[(r + RING - 2) % RING], pp + RING - 2);
            load_next(ring[(r + RING - 1) % RING], pp + RING - 1);
            const bool has_b = pp + 1 < page_e;
            step(ring[r], has_b ? ring[r + 1] : ring[r], pp, has_b);
        }
    }
    lsum += __shfl_xor(lsum, 16, 64);
    lsum += __shfl_xor(lsum, 32, 64);
    if (!valid) return;
    float* out = a.part + (((size_t)item * a.kv_heads + kvh) * 16 + c) * (D + 2);
    if (q4 == 0) *(float2*)out = make_float2(m, lsum);
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
        float2* x = (float2*)(out + 2 + db * 16 + q4 * 4);
        x[0] = make_float2(o[db][0], o[db][1]);
        x[1] = make_float2(o[db][2], o[db][3]);
    }
}

// Units first: they run longest, and as many of them as CUs get one each (in turn
// with the tails, two units shared one CU and two tails another).  Tails go
// in groups of 8 workgroups, one per XCD.
__device__ __forceinline__ bool shared_split(const SharedArgs& a, int& unit_wg, int& tail_group) {
    unit_wg = blockIdx.x;
    tail_group = (int)(blockIdx.x >> 3) - a.unit_groups;
    return tail_group < 0;
}

template <int D, int CW, int KW, bool NEXT, int RING>
__global__ __launch_bounds__(256, 2) void shared_attention_kernel(SharedArgs a, const int* __restrict__ block_tables) {
    constexpr size_t unit = unit_lds(D, CW, KW, NEXT), bytes = unit > tail_lds(D) ? unit : tail_lds(D);
    __shared__ bf16x8 buf[bytes / 16];
    int unit_wg, tail_group;
    if (shared_split(a, unit_wg, tail_group))
        shared_unit<D, CW, KW, NEXT>(a, block_tables, unit_wg, buf);
    else
        shared_tail<uint16_t, D, RING>(a, block_tables, tail_group, buf);
}

template <int D, int RING>
__global__ __launch_bounds__(256, 1) void shared_attention_f32_kernel(SharedArgs a, const int* __restrict__ block_tables) {
    constexpr size_t bytes = unit_f32_lds(D) > tail_lds(D) ? unit_f32_lds(D) : tail_lds(D);
    __shared__ bf16x8 buf[bytes / 16];
    int unit_wg, tail_group;
    if (shared_split(a, unit_wg, tail_group))
        shared_unit_f32<D>(a, block_tables, unit_wg, buf);
    else
        shared_tail<float, D, RING>(a, block_tables, tail_group, buf);
}

// Joins a row's partials.  16 lanes per part: lane j of a part holds its dims
// j D / 16 and on.  W waves take a (row, q head), so that 4 W parts come at once
// (AHEAD of those in flight): one wave where rows are many or their parts few,
// four where a long prefix left many parts to few rows.  A part group sums its
// parts p = group mod 4 W in order, then the groups meet in order: the sums do
// not depend on timing.
// rec: {row, first source, sources, parts}; src: {first item, parts, first column, 0}.
template <int D, int W>
__global__ __launch_bounds__(256) void shared_merge_kernel(const float* __restrict__ part, const int4* __restrict__ rec,
                                                           const int4* __restrict__ src, int jobs, int G, int kv_heads,
                                                           int q_cols, float* out, uint16_t* out_bf16,
                                                           size_t lo_offset) {
    constexpr int V = D / 16, V2 = V / 2, GROUPS = 4 * W, AHEAD = W == 1 ? 4 : 2;
    __shared__ float sm[4][4], sl[4][4], so[4][4][D];  // [wave][group of the wave]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sub = lane >> 4, d0 = (lane & 15) * V;
    const int job = blockIdx.x * (4 / W) + (W == 1 ? wave : 0);
    const int group = W == 1 ? sub : wave * 4 + sub;
    const int heads = kv_heads * G;
    const int ri = job / heads, head = job - ri * heads, kvh = head / G, g = head - kvh * G;
    const int4 r = job < jobs ? rec[ri] : make_int4(0, 0, 0, 0);  // (empty too: past a replayed bucket's rows)
    const size_t pstride = (size_t)kv_heads * 16 * (D + 2);
    float M = -INFINITY, L = 0.0f, acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
    int si = r.y, start = 0;      // the source holding part p, and its first part
    int4 s = r.z > 0 ? src[si] : make_int4(0, 0, 0, 0);
    for (int p0 = group; p0 < r.w; p0 += GROUPS * AHEAD) {
        float2 ml[AHEAD], x[AHEAD][V2];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int p = p0 + GROUPS * u;
            ml[u] = make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int j = 0; j < V2; ++j) x[u][j] = make_float2(0.0f, 0.0f);
            if (p < r.w) {
                while (p - start >= s.y) {
                    start += s.y;
                    s = src[++si];
                }
                const float* b =
                    part + (((size_t)s.x * kv_heads + kvh) * 16 + s.z + g) * (D + 2) + (size_t)(p - start) * pstride;
                ml[u] = *(const float2*)b;
#pragma unroll
                for (int j = 0; j < V2; ++j) x[u][j] = *(const float2*)(b + 2 + d0 + 2 * j);
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const float Mn = fmaxf(M, ml[u].x);
            if (Mn == -INFINITY) continue;  // no visible key so far
            const float keep = exp2f(M - Mn), w = exp2f(ml[u].x - Mn);
            M = Mn;
            L = L * keep + ml[u].y * w;
#pragma unroll
            for (int j = 0; j < V2; ++j) {
                acc[2 * j] = fmaf(x[u][j].x, w, acc[2 * j] * keep);
                acc[2 * j + 1] = fmaf(x[u][j].y, w, acc[2 * j + 1] * keep);
            }
        }
    }
    if ((lane & 15) == 0) {
        sm[wave][sub] = M;
        sl[wave][sub] = L;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) so[wave][sub][d0 + j] = acc[j];
    __syncthreads();
    // (W == 1: each wave its own job; W == 4: the workgroup's D threads the one)
    const int nt = W == 1 ? 64 : 256, at = W == 1 ? lane : tid, w0 = W == 1 ? wave : 0;
    if (r.z == 0) return;
    float mm = -INFINITY;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) mm = fmaxf(mm, sm[w0 + i / 4][i & 3]);
    for (int d = at; d < D; d += nt) {
        float l = 0.0f, o = 0.0f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const float mi = sm[w0 + i / 4][i & 3];
            const float w = mi == -INFINITY ? 0.0f : exp2f(mi - mm);
            l = fmaf(sl[w0 + i / 4][i & 3], w, l);
            o = fmaf(so[w0 + i / 4][i & 3][d], w, o);
        }
        o /= l;
        const int col = head * D + d;
        if (out_bf16) {
            uint16_t hi, lo;
            split_bf16(o, hi, lo);
            const size_t idx = a_pack_index(r.x, col, q_cols);
            out_bf16[idx] = hi;
            if (lo_offset) out_bf16[lo_offset + idx] = lo;
        } else {
            out[(size_t)r.x * q_cols + col] = o;
        }
    }
}

template <int D>
static void launch_shared(zr_context* ctx, StagedMeta* st, const SharedArgs& a, int groups) {
    const dim3 grid(8 * groups), block(256);
    constexpr int RING = D == 64 ? 6 : 4;
    if (ctx->desc.kv_dtype == ZR_DTYPE_F32)
        hipLaunchKernelGGL((shared_attention_f32_kernel<D, 4>), grid, block, 0, ctx->stream, a, st->block_tables);
    else if (st->unit_cols == 128)
        hipLaunchKernelGGL((shared_attention_kernel<D, 4, 1, true, RING>), grid, block, 0, ctx->stream, a, st->block_tables);
    else if (st->unit_cols == 64)
        hipLaunchKernelGGL((shared_attention_kernel<D, 2, 2, D == 64, RING>), grid, block, 0, ctx->stream, a, st->block_tables);
    else
        hipLaunchKernelGGL((shared_attention_kernel<D, 1, 4, false, RING>), grid, block, 0, ctx->stream, a, st->block_tables);
}

zr_status launch_shared_attention(zr_context* ctx, StagedMeta* st, int layer, const float* q) {
    const size_t esz = ctx->desc.kv_dtype == ZR_DTYPE_BF16 ? 2 : 4;
    SharedArgs a;
    a.q = q;
    a.q_cols = ctx->q_cols;
    a.page_elems = (size_t)2 * ctx->kv_cols * kPageRows;
    a.pool = (const unsigned char*)ctx->kv_pool + (size_t)layer * ctx->n_pages * a.page_elems * esz;
    a.stride = st->stride;
    a.units = st->sunits;
    a.rec = st->attn_rec;
    a.n_units = st->grid_units;
    a.n_tails = st->grid_items;
    a.kv_heads = ctx->local_kv_heads;
    a.unit_groups = (a.n_units * a.kv_heads + 7) / 8;
    const int groups = a.unit_groups + ((a.n_tails + 7) / 8 * a.kv_heads + 3) / 4;
    a.G = ctx->q_per_kv;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)ctx->head_dim);
    a.part = ctx->attn_part;
    hipEvent_t ev;
    timing_mark_begin(ctx, kClassAttention, &ev);
    if (ctx->head_dim == 64) launch_shared<64>(ctx, st, a, groups); else launch_shared<128>(ctx, st, a, groups);
    ZR_LAUNCH_CHECK(ctx);
    timing_mark_end(ctx, kClassAttention, ev);
    return ZR_OK;
}

zr_status launch_shared_merge(zr_context* ctx, StagedMeta* st, float* out, uint16_t* out_bf16) {
    if (st->grid_smerge == 0) return ZR_OK;
    const size_t lo = (ctx->desc.flags & ZR_FLAG_SPLIT_ACTIVATIONS) ? a_plane(st->total_q, ctx->q_cols) : 0;
    const int jobs = st->grid_smerge * ctx->local_q_heads;
    const bool wide = st->merge_wide;
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(wide ? jobs : (jobs + 3) / 4), dim3(256), 0, ctx->stream, ctx->attn_part,
                           st->smerge, st->ssrc, jobs, ctx->q_per_kv, ctx->local_kv_heads, ctx->q_cols, out, out_bf16,
                           lo);
    };
    hipEvent_t ev;
    timing_mark_begin(ctx, kClassOther, &ev);
    if (ctx->head_dim == 64) {
        if (wide) launch(shared_merge_kernel<64, 4>); else launch(shared_merge_kernel<64, 1>);
    } else {
        if (wide) launch(shared_merge_kernel<128, 4>); else launch(shared_merge_kernel<128, 1>);
    }
    ZR_LAUNCH_CHECK(ctx);
    timing_mark_end(ctx, kClassOther, ev);
    return ZR_OK;
}

// ------------------------------------------------------------------ staging
// Walks the trie of block tables: `members` (sequences, all with the same pages
// before page `d`) share pages from `begin` on while their next pages agree.
// What a run saves is (members - 1) reads of its pages; a shorter one than
// kMinRun, or one that saves less than kMinSaved, is left to the runs below
// it (which then start at `begin`) and to the sequences themselves.
namespace {

constexpr int kMinRun = 4, kMinSaved = 8;  // pages

struct Walk {
    const zr_microbatch* mb;
    const std::vector<int>* limit;  // full pages before each sequence's new rows
    std::vector<SharedSegment>* out;
    std::vector<int>* cover;

    const int* table(int s) const { return mb->block_tables + (size_t)s * mb->block_table_stride; }

    void descend(std::vector<int> members, int begin, int d) {
        for (;;) {
            if (members.size() < 2) return;
            // pages that every member names
            const int* first = table(members[0]);
            int end = (*limit)[members[0]];
            for (size_t i = 1; i < members.size(); ++i) {
                const int* t = table(members[i]);
                end = std::min(end, (*limit)[members[i]]);
                int e = d;
                while (e < end && t[e] == first[e]) ++e;
                end = e;
            }
            const int run = end - begin;
            if (run >= kMinRun && (long)(members.size() - 1) * run >= kMinSaved) {
                out->push_back({members[0], begin, end, members});
                for (int s : members) (*cover)[s] = end;
                begin = end;
            }
            // the members that go on, by their next page
            std::vector<int> on;
            for (int s : members)
                if ((*limit)[s] > end) on.push_back(s);
            std::stable_sort(on.begin(), on.end(), [&](int x, int y) { return table(x)[end] < table(y)[end]; });
            std::vector<std::vector<int>> parts;
            for (size_t i = 0; i < on.size();) {
                size_t j = i + 1;
                while (j < on.size() && table(on[j])[end] == table(on[i])[end]) ++j;
                if (j - i >= 2) parts.emplace_back(on.begin() + i, on.begin() + j);
                i = j;
            }
            if (parts.empty()) return;
            for (size_t i = 1; i < parts.size(); ++i) descend(parts[i], begin, end + 1);
            members.swap(parts[0]);
            d = end + 1;
        }
    }
};

}  // namespace

void shared_segments(const zr_microbatch* mb, const std::vector<char>& takes, std::vector<SharedSegment>* out,
                     std::vector<int>* cover) {
    const int S = mb->num_seqs, stride = mb->block_table_stride;
    out->clear();
    cover->assign(S, 0);
    // sequences by their first page and the row their window starts at in it
    std::vector<int> order, limit(S, 0);
    for (int s = 0; s < S; ++s) {
        limit[s] = (mb->first_offset[s] + mb->kv_before[s]) / kPageRows;
        if (takes[s] && limit[s] > 0) order.push_back(s);
    }
    auto key = [&](int s) { return std::make_pair(mb->block_tables[(size_t)s * stride], mb->first_offset[s]); };
    std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return key(x) < key(y); });
    Walk w{mb, &limit, out, cover};
    for (size_t i = 0; i < order.size();) {
        size_t j = i + 1;
        while (j < order.size() && key(order[j]) == key(order[i])) ++j;
        if (j - i >= 2) w.descend(std::vector<int>(order.begin() + i, order.begin() + j), 0, 1);
        i = j;
    }
}

}  // namespace zr
