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
// Segments run here, the pages after them in paged_attention_kernel's tiles,
// and shared_merge_kernel joins the partials of a row.
#include "attn_tile.h"
#include "zr_internal.h"

namespace zr {

struct SharedArgs {
    const float* q;       // [T, q_cols]
    int q_cols;
    const void* pool;     // layer base of the pool
    size_t page_elems;
    int stride;           // block table row stride
    const int* first_offset;
    const int4* units;    // two records per work unit: {seq, first of its rows in `rows`, rows | splits << 16, first page},
                          // {first key tile, end key tile, partial item, end page}
    const int* rows;      // query rows of the microbatch
    int n_units;
    int G, kv_heads;
    float scale_log2;     // log2(e) / sqrt(d)
    float* part;          // [items][kv_heads][16][D + 2]
};

// Q^T fragments (B operand) of a column: lane holds Q[col][16 ks + 8 h + j]
// log2(e) / sqrt(d) in three bf16 parts (scores come out in log2 units).
template <int D>
__device__ __forceinline__ void shared_load_q(const float* qp, float scale, bool valid, bf16x8 (&q)[D / 16][3]) {
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        const f32x4 x0 = valid ? *(const f32x4*)(qp + 16 * ks) : zero;
        const f32x4 x1 = valid ? *(const f32x4*)(qp + 16 * ks + 4) : zero;
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = x0[j] * scale;
            x[4 + j] = x1[j] * scale;
        }
        split3_bf16x8(x, q[ks]);
    }
}

// V rows of keys outside [0, last] enter the product as 0: their weights are 0,
// but 0 x inf is NaN, and rows before a trimmed window hold whatever they held.
// Element j of k-step ks2 is key base + 16 ks2 + 8 (j / 4) + 4 h + j % 4.
template <int D>
__device__ __forceinline__ void shared_mask_v(bf16x8 (&v)[2][D / 32], int base, int h, int last) {
#pragma unroll
    for (int ks2 = 0; ks2 < 2; ++ks2)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = base + 16 * ks2 + 8 * (j >> 2) + 4 * h + (j & 3);
            if (key < 0 || key > last)
#pragma unroll
                for (int db = 0; db < D / 32; ++db) v[ks2][db][j] = (__bf16)0.0f;
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
// slices in turn; each is copied once into an LDS ring by the CW waves of its
// slice (buffer loads into LDS, the pool's page order, no registers) and serves
// all columns.  Per tile and wave, on v_mfma_f32_32x32x16_bf16 (h = lane / 32):
//   S[key][col] = sum_d K[key][d] Q[col][d]; the lane gets key 8 (i / 4) + 4 h + i % 4, i < 16
//   online softmax per column over the lane's 16 keys and the 16 of lane ^ 32
//   O[d][col] += sum_key V[key][d] P[key][col]: P's fragment is the lane's own scores
// Q and P enter in three bf16 parts, which hold all of an f32's 24 bits (two
// parts, 17 bits, put the result 4e-6 of its norm off: 3.4e-6 from Q, 2.2e-6
// from P; three leave 1e-7), K and V are exact; sums are f32.
template <int D, int CW, int KW, int STAGES>
__global__ __launch_bounds__(64 * CW * KW, CW * KW / 4) void shared_prefix_kernel(SharedArgs a,
                                                                              const int* __restrict__ block_tables) {
    constexpr int CHUNKS = 8 * D;        // 16 B chunks per tile: 2 pages x (K, V) x 16 rows x D bf16
    constexpr int VM = CHUNKS / 64 / CW; // copies (1 KiB each) per wave and tile
    constexpr int RUN = D / 32;          // 1 KiB runs of one head's K (or V) page
    static_assert(VM * 64 * CW == CHUNKS, "tile copy split");
    __shared__ bf16x8 lds[STAGES][KW][CHUNKS];
    static_assert(shared_combine_bytes(D, CW, KW) <= sizeof(lds), "combine buffer");

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slice = wave / CW, wq = wave - slice * CW;
    const int rank = __builtin_amdgcn_readfirstlane(blockIdx.x / a.kv_heads);
    const int kvh = blockIdx.x - rank * a.kv_heads;
    const int4 u0 = a.units[2 * rank], u1 = a.units[2 * rank + 1];
    const int seq = __builtin_amdgcn_readfirstlane(u0.x), row0 = __builtin_amdgcn_readfirstlane(u0.y);
    const int nrows = __builtin_amdgcn_readfirstlane(u0.z & 0xffff), nsplits = __builtin_amdgcn_readfirstlane(u0.z >> 16);
    const int pb = __builtin_amdgcn_readfirstlane(u0.w), pe = __builtin_amdgcn_readfirstlane(u1.w);
    const int kt0 = __builtin_amdgcn_readfirstlane(u1.x), kt1 = __builtin_amdgcn_readfirstlane(u1.y);
    const int item0 = __builtin_amdgcn_readfirstlane(u1.z);
    if (nrows == 0) return;  // an empty record past a replayed bucket's units
    const int h = lane >> 5;
    const int c = wq * 32 + (lane & 31);
    const int rloc = c / a.G, g = c - rloc * a.G;
    const bool valid = rloc < nrows;
    const bool busy = wq * 32 < nrows * a.G;  // the wave has a column
    // keys of the segment's first page before the window, and of its last tile past its end
    const int foff = pb == 0 ? __builtin_amdgcn_readfirstlane(a.first_offset[seq]) : 0;
    const int jlast = (pe - pb) * kPageRows - 1;

    const uint16_t* pool = (const uint16_t*)a.pool;
    const int* bt = block_tables + (size_t)seq * a.stride;
    const size_t kv_tile = (size_t)kPageRows * D;
    const size_t v_block = (size_t)a.kv_heads * kv_tile;
    // pool pages of tile kt (a tile past the segment's end repeats its last page)
    auto tile_pages = [&](int kt, int& pg0, int& pg1) {
        pg0 = __builtin_amdgcn_readfirstlane(bt[min(pb + 2 * kt, pe - 1)]);
        pg1 = __builtin_amdgcn_readfirstlane(bt[min(pb + 2 * kt + 1, pe - 1)]);
    };
    const uint32_t page_bytes = (uint32_t)(a.page_elems * 2);
    const int voff = lane * 16;
    auto issue = [&](int slot, int pg0, int pg1) {
        const __amdgpu_buffer_rsrc_t r0 =
            __builtin_amdgcn_make_buffer_rsrc((void*)(pool + (size_t)pg0 * a.page_elems), 0, page_bytes, 0x00020000);
        const __amdgpu_buffer_rsrc_t r1 =
            __builtin_amdgcn_make_buffer_rsrc((void*)(pool + (size_t)pg1 * a.page_elems), 0, page_bytes, 0x00020000);
#pragma unroll
        for (int i = 0; i < VM; ++i) {
            const int f = i * CW + wq;  // (page, K or V, 1 KiB run)
            const int pp = f / (2 * RUN), kv = (f / RUN) & 1, run = f % RUN;
            const int soff = (int)(((kv ? v_block : 0) + (size_t)kvh * kv_tile) * 2) + run * 1024;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(pp ? r1 : r0, (lds_void*)&lds[slot][slice][f * 64], 16, voff, soff,
                                                     0, 0);
        }
    };

    f32x16 o[D / 32];
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
    float m = -INFINITY, lsum = 0.0f;

    // step p holds tile kt0 + KW p + slice
    const int nsteps = (kt1 - kt0 + KW - 1) / KW;
    int npg0 = 0, npg1 = 0;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
        if (s < nsteps) {
            tile_pages(kt0 + KW * s + slice, npg0, npg1);
            issue(s, npg0, npg1);
        }
    tile_pages(kt0 + KW * (STAGES - 1) + slice, npg0, npg1);
    const int grow = a.rows[row0 + (valid ? rloc : 0)];
    bf16x8 q[D / 16][3];
    shared_load_q<D>(a.q + (size_t)grow * a.q_cols + (size_t)(kvh * a.G + g) * D + 8 * h, a.scale_log2, valid, q);

    for (int t = 0; t < nsteps; ++t) {
        ring_wait<VM, STAGES - 2>(min(STAGES - 2, nsteps - 1 - t));
        if (t + STAGES - 1 < nsteps) issue((t + STAGES - 1) % STAGES, npg0, npg1);
        const int kt = kt0 + KW * t + slice;
        if (busy && kt < kt1) {
            const bf16x8* st = lds[t % STAGES][slice];
            const int kbase = ((lane >> 4) & 1) * 2 * (2 * D) + (lane & 15);  // page (l % 32) / 16, row l % 16
            bf16x8 kf[D / 16];
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) kf[ks] = st[kbase + (2 * ks + h) * 16];
            __builtin_amdgcn_sched_barrier(0);  // the K reads stay ahead of the MFMAs
            f32x16 s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks], q[ks][i], s, 0, 0, 0);
            }
            bf16x8 vf[2][D / 32];
            const bf16x4* sv = (const bf16x4*)st;
#pragma unroll
            for (int ks2 = 0; ks2 < 2; ++ks2) {
                const int vbase = (2 * ks2 + 1) * 4 * D;  // 8-byte units of page ks2's V block
#pragma unroll
                for (int db = 0; db < D / 32; ++db) {
                    const int u = ((db * 4 + h) * 16 + (lane & 15)) * 2 + ((lane >> 4) & 1);
                    const bf16x4 v0 = sv[vbase + u], v1 = sv[vbase + u + 2 * 16 * 2];
                    vf[ks2][db] = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // the V reads go out before the softmax
            if (32 * kt < foff || 32 * kt + 31 > jlast) {
                prefill_mask(s, 32 * kt + 4 * h - foff, jlast - foff);
                shared_mask_v<D>(vf, 32 * kt - foff, h, jlast - foff);
            }
            float pr[16];
            prefill_softmax<D>(s, o, m, lsum, pr);
#pragma unroll
            for (int ks2 = 0; ks2 < 2; ++ks2) {
                bf16x8 p[3];
                split3_bf16x8(pr + 8 * ks2, p);
#pragma unroll
                for (int i = 0; i < 3; ++i)
#pragma unroll
                    for (int db = 0; db < D / 32; ++db)
                        o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[ks2][db], p[i], o[db], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (t + STAGES - 1 < nsteps) tile_pages(kt0 + KW * (t + STAGES) + slice, npg0, npg1);
    }
    shared_finish<D, CW, KW>(a, o, m, lsum, (float*)&lds[0][0][0], slice, wq, lane, kvh, item0, nsplits, valid);
}

// f32 pools: K, V, Q and P each enter the MFMA in three bf16 parts; of the nine
// products of a pair the six above 2^-24 of the result are formed (two parts and
// three products are 8e-6 of the result's norm off).  A tile is split once
// per workgroup: each wave loads its share of the next tile's f32 runs into
// registers a step ahead, splits them and stores three planes in the LDS order
// of a bf16 tile, two slots deep, one barrier per step.  At D = 128 the planes
// and the registers hold one key slice: its waves are alone on their SIMDs.
template <int D, int CW, int KW>
__global__ __launch_bounds__(64 * CW * KW, CW * KW / 4) void shared_prefix_f32_kernel(SharedArgs a,
                                                                                  const int* __restrict__ block_tables) {
    constexpr int CHUNKS = 8 * D;         // 16 B chunks per plane of a tile
    constexpr int VM = CHUNKS / 64 / CW;  // 512-element runs per wave and tile
    constexpr int RUN = D / 32;
    static_assert(VM * 64 * CW == CHUNKS, "tile copy split");
    __shared__ bf16x8 lds[2][KW][3][CHUNKS];  // [slot][slice][part]
    static_assert(shared_combine_bytes(D, CW, KW) <= sizeof(lds), "combine buffer");

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slice = wave / CW, wq = wave - slice * CW;
    const int rank = __builtin_amdgcn_readfirstlane(blockIdx.x / a.kv_heads);
    const int kvh = blockIdx.x - rank * a.kv_heads;
    const int4 u0 = a.units[2 * rank], u1 = a.units[2 * rank + 1];
    const int seq = __builtin_amdgcn_readfirstlane(u0.x), row0 = __builtin_amdgcn_readfirstlane(u0.y);
    const int nrows = __builtin_amdgcn_readfirstlane(u0.z & 0xffff), nsplits = __builtin_amdgcn_readfirstlane(u0.z >> 16);
    const int pb = __builtin_amdgcn_readfirstlane(u0.w), pe = __builtin_amdgcn_readfirstlane(u1.w);
    const int kt0 = __builtin_amdgcn_readfirstlane(u1.x), kt1 = __builtin_amdgcn_readfirstlane(u1.y);
    const int item0 = __builtin_amdgcn_readfirstlane(u1.z);
    if (nrows == 0) return;
    const int h = lane >> 5;
    const int c = wq * 32 + (lane & 31);
    const int rloc = c / a.G, g = c - rloc * a.G;
    const bool valid = rloc < nrows;
    const bool busy = wq * 32 < nrows * a.G;
    const int foff = pb == 0 ? __builtin_amdgcn_readfirstlane(a.first_offset[seq]) : 0;
    const int jlast = (pe - pb) * kPageRows - 1;

    const int* bt = block_tables + (size_t)seq * a.stride;
    const size_t kv_tile = (size_t)kPageRows * D;
    const size_t v_block = (size_t)a.kv_heads * kv_tile;
    const float* pool = (const float*)a.pool + (size_t)kvh * kv_tile + 4 * lane;
    auto tile_pages = [&](int kt, int& pg0, int& pg1) {
        pg0 = __builtin_amdgcn_readfirstlane(bt[min(pb + 2 * kt, pe - 1)]);
        pg1 = __builtin_amdgcn_readfirstlane(bt[min(pb + 2 * kt + 1, pe - 1)]);
    };
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
            for (int k = 0; k < 3; ++k) lds[slot][slice][k][f * 64 + lane] = p[k];
        }
    };

    f32x16 o[D / 32];
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
    float m = -INFINITY, lsum = 0.0f;
    const int nsteps = (kt1 - kt0 + KW - 1) / KW;
    int pg0, pg1, npg0, npg1;
    tile_pages(kt0 + slice, pg0, pg1);
    tile_pages(kt0 + KW + slice, npg0, npg1);
    load_raw(pg0, pg1);
    const int grow = a.rows[row0 + (valid ? rloc : 0)];
    bf16x8 q[D / 16][3];
    shared_load_q<D>(a.q + (size_t)grow * a.q_cols + (size_t)(kvh * a.G + g) * D + 8 * h, a.scale_log2, valid, q);
    store_split(0);
    load_raw(npg0, npg1);
    tile_pages(kt0 + 2 * KW + slice, npg0, npg1);

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

    for (int t = 0; t < nsteps; ++t) {
        ring_barrier<63>();  // the slot is written (LDS only: the next tile's loads stay in flight)
        const int kt = kt0 + KW * t + slice;
        if (busy && kt < kt1) {
            const bf16x8(&st)[3][CHUNKS] = lds[t & 1][slice];
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
                shared_mask_v<D>(vf, 32 * kt - foff, h, jlast - foff);
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
                    if (edge) shared_mask_v<D>(vf, 32 * kt - foff, h, jlast - foff);
                }
            }
        }
        if (t + 1 < nsteps) {
            store_split((t + 1) & 1);  // last read in step t - 1, a barrier ago
            if (t + 2 < nsteps) {
                load_raw(npg0, npg1);
                tile_pages(kt0 + KW * (t + 3) + slice, npg0, npg1);
            }
        }
    }
    shared_finish<D, CW, KW>(a, o, m, lsum, (float*)&lds[0][0][0][0], slice, wq, lane, kvh, item0, nsplits, valid);
}

// Joins a row's partials.  A wave per (row, q head): lane s takes part s's
// (m, l) (64 at a time), then every lane its D / 64 dims of every part.  Parts
// are summed in the order of the row's sources (segments, then its own pages).
// rec: {row, first source, sources, 0}; src: {first item, parts, first column, 0}.
template <int D>
__global__ __launch_bounds__(256) void shared_merge_kernel(const float* __restrict__ part, const int4* __restrict__ rec,
                                                           const int4* __restrict__ src, int n_rows, int G, int kv_heads,
                                                           int q_cols, float* out, uint16_t* out_bf16,
                                                           size_t lo_offset) {
    const int lane = threadIdx.x & 63;
    const int heads = kv_heads * G;
    const int job = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (job >= n_rows * heads) return;
    const int ri = job / heads, head = job - ri * heads, kvh = head / G, g = head - kvh * G;
    const int4 r = rec[ri];
    if (r.z == 0) return;  // an empty record past a replayed bucket's rows
    constexpr int V = D / 64;
    float M = -INFINITY, L = 0.0f, acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
    const size_t pstride = (size_t)kv_heads * 16 * (D + 2);
    for (int si = 0; si < r.z; ++si) {
        const int4 s = src[r.y + si];
        const float* base = part + (((size_t)s.x * kv_heads + kvh) * 16 + s.z + g) * (D + 2);
        for (int p0 = 0; p0 < s.y; p0 += 64) {
            const int np = min(64, s.y - p0);
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (lane < np) ml = *(const float2*)(base + (size_t)(p0 + lane) * pstride);
            float mx = ml.x;
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
            const float Mn = fmaxf(M, mx);
            if (Mn == -INFINITY) continue;  // no visible key so far
            const float keep = exp2f(M - Mn);
            const float w = exp2f(ml.x - Mn);  // 0 for a part with no visible key
            float ls = ml.y * w;
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) ls += __shfl_xor(ls, off, 64);
            L = L * keep + ls;
            M = Mn;
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] *= keep;
            const float* pv = base + (size_t)p0 * pstride + 2 + lane * V;
#pragma unroll 8
            for (int p = 0; p < np; ++p) {
                const float wp = __shfl(w, p, 64);
                if constexpr (V == 2) {
                    const float2 x = *(const float2*)(pv + (size_t)p * pstride);
                    acc[0] = fmaf(x.x, wp, acc[0]);
                    acc[1] = fmaf(x.y, wp, acc[1]);
                } else {
                    acc[0] = fmaf(pv[(size_t)p * pstride], wp, acc[0]);
                }
            }
        }
    }
    const float inv = 1.0f / L;
    const int col = head * D + lane * V;
    if (out_bf16) {
        const size_t o = a_pack_index(r.x, col, q_cols);  // V consecutive columns are one run of the packed operand
#pragma unroll
        for (int j = 0; j < V; ++j) {
            uint16_t hi, lo;
            split_bf16(acc[j] * inv, hi, lo);
            out_bf16[o + j] = hi;
            if (lo_offset) out_bf16[lo_offset + o + j] = lo;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) out[(size_t)r.x * q_cols + col + j] = acc[j] * inv;
    }
}

template <int D>
static void launch_units(zr_context* ctx, StagedMeta* st, const SharedArgs& a) {
    const dim3 grid(st->n_sunits * ctx->local_kv_heads);
    constexpr int KW = D == 64 ? 2 : 1;
    if (ctx->desc.kv_dtype == ZR_DTYPE_BF16)
        hipLaunchKernelGGL((shared_prefix_kernel<D, 4, 2, 3>), grid, dim3(512), 0, ctx->stream, a, st->block_tables);
    else
        hipLaunchKernelGGL((shared_prefix_f32_kernel<D, 4, KW>), grid, dim3(256 * KW), 0, ctx->stream, a,
                           st->block_tables);
}

zr_status launch_shared_prefix(zr_context* ctx, StagedMeta* st, int layer, const float* q) {
    if (st->n_sunits == 0) return ZR_OK;
    const size_t esz = ctx->desc.kv_dtype == ZR_DTYPE_BF16 ? 2 : 4;
    SharedArgs a;
    a.q = q;
    a.q_cols = ctx->q_cols;
    a.page_elems = (size_t)2 * ctx->kv_cols * kPageRows;
    a.pool = (const unsigned char*)ctx->kv_pool + (size_t)layer * ctx->n_pages * a.page_elems * esz;
    a.stride = st->stride;
    a.first_offset = st->first_offset;
    a.units = st->sunits;
    a.rows = st->srows;
    a.n_units = st->n_sunits;
    a.G = ctx->q_per_kv;
    a.kv_heads = ctx->local_kv_heads;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)ctx->head_dim);
    a.part = ctx->attn_part;
    hipEvent_t ev;
    timing_mark_begin(ctx, kClassAttention, &ev);
    if (ctx->head_dim == 64) launch_units<64>(ctx, st, a); else launch_units<128>(ctx, st, a);
    ZR_LAUNCH_CHECK(ctx);
    timing_mark_end(ctx, kClassAttention, ev);
    return ZR_OK;
}

zr_status launch_shared_merge(zr_context* ctx, StagedMeta* st, float* out, uint16_t* out_bf16) {
    if (st->n_smerge == 0) return ZR_OK;
    const size_t lo = (ctx->desc.flags & ZR_FLAG_SPLIT_ACTIVATIONS) ? a_plane(st->total_q, ctx->q_cols) : 0;
    const dim3 grid((st->n_smerge * ctx->local_q_heads + 3) / 4);
    hipEvent_t ev;
    timing_mark_begin(ctx, kClassOther, &ev);
    if (ctx->head_dim == 64)
        hipLaunchKernelGGL((shared_merge_kernel<64>), grid, dim3(256), 0, ctx->stream, ctx->attn_part, st->smerge,
                           st->ssrc, st->n_smerge, ctx->q_per_kv, ctx->local_kv_heads, ctx->q_cols, out, out_bf16, lo);
    else
        hipLaunchKernelGGL((shared_merge_kernel<128>), grid, dim3(256), 0, ctx->stream, ctx->attn_part, st->smerge,
                           st->ssrc, st->n_smerge, ctx->q_per_kv, ctx->local_kv_heads, ctx->q_cols, out, out_bf16, lo);
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
