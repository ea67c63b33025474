// What the attention kernels share: a page's registers, operands in bf16 parts, and
// steps on one tile of scores (v_mfma_f32_32x32x16_bf16: a lane holds 16 scores of
// one column, lane l ^ 32 the other 16).
#pragma once

#include "zr_internal.h"

namespace zr {

// Every page of the pool is read once per launch (one workgroup per kv head
// and page run), so the loads carry the nontemporal hint: the lines are
// streamed through L2 with low retention instead of displacing what the other
// waves on the XCD still read (256-session Llama-3-8B step: attention 9.55-9.78
// -> 8.81-8.99 ms per step; 32-session TinyLlama step unchanged).
template <typename KV, int D> struct PageRegs;

// bf16 pool: K fragment per 32 dims = 8 bf16 (16 B); V per 32 dims = 8 bf16
// (16 B): tokens 4 q4 .. 4 q4 + 3 of dims 32 vb + c, then of 32 vb + 16 + c.
// Both are one 1 KiB contiguous wave load.
template <int D> struct PageRegs<uint16_t, D> {
    bf16x8 k[D / 32];
    bf16x8 v[D / 32];
    __device__ inline void load(const uint16_t* kp, const uint16_t* vp, int lane) {
#pragma unroll
        for (int kb = 0; kb < D / 32; ++kb)
            k[kb] = __builtin_nontemporal_load((const bf16x8*)(kp + ((size_t)kb * kWave + lane) * 8));
#pragma unroll
        for (int vb = 0; vb < D / 32; ++vb)
            v[vb] = __builtin_nontemporal_load((const bf16x8*)(vp + ((size_t)vb * kWave + lane) * 8));
    }
};

// f32 pool (page_order): the same 8 values per lane and 32 dims, as two
// 16 B halves that each come from one contiguous 1 KiB wave run (K: dims
// 8 g + [0, 4) then + [4, 8); V: dim d then d + 16, 4 tokens each).
template <int D> struct PageRegs<float, D> {
    f32x4 k[D / 32][2];
    f32x4 v[D / 32][2];
    __device__ inline void load(const float* kp, const float* vp, int lane) {
#pragma unroll
        for (int kb = 0; kb < D / 32; ++kb) {
            const f32x4* src = (const f32x4*)(kp + (size_t)kb * kWave * 8) + lane;
            k[kb][0] = __builtin_nontemporal_load(src);
            k[kb][1] = __builtin_nontemporal_load(src + kWave);
        }
#pragma unroll
        for (int vb = 0; vb < D / 32; ++vb) {
            const f32x4* src = (const f32x4*)(vp + (size_t)vb * kWave * 8) + lane;
            v[vb][0] = __builtin_nontemporal_load(src);
            v[vb][1] = __builtin_nontemporal_load(src + kWave);
        }
    }
};

// x[0..7] as bf16 hi + lo fragments, two values per v_cvt_pk_bf16_f32 (the
// same bits as split_bf16)
__device__ inline void split_bf16x8(const float* x, bf16x8& hi, bf16x8& lo) {
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;
    typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f32x2 v = {x[2 * j], x[2 * j + 1]};
        const bf16x2 h = __builtin_convertvector(v, bf16x2);
        const bf16x2 l = __builtin_convertvector(v - __builtin_convertvector(h, f32x2), bf16x2);
        hi[2 * j] = h[0];
        hi[2 * j + 1] = h[1];
        lo[2 * j] = l[0];
        lo[2 * j + 1] = l[1];
    }
}

// x[0..7] as three bf16 fragments whose sum is x to its last f32 bit (8 bits
// each; a remainder is exact in f32, so only the third part is rounded away
// from x, below 2^-25 of it)
__device__ inline void split3_bf16x8(const float* x, bf16x8 (&p)[3]) {
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;
    typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f32x2 v = {x[2 * j], x[2 * j + 1]};
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const bf16x2 h = __builtin_convertvector(v, bf16x2);
            if (k < 2) v -= __builtin_convertvector(h, f32x2);
            p[k][2 * j] = h[0];
            p[k][2 * j + 1] = h[1];
        }
    }
}

// ... of two values, as word `at` of the parts
__device__ inline void split3_pair(float a, float b, uint32_t (&p)[3][4], int at) {
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;
    typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
    f32x2 v = {a, b};
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const bf16x2 h = __builtin_convertvector(v, bf16x2);
        if (k < 2) v -= __builtin_convertvector(h, f32x2);
        p[k][at] = __builtin_bit_cast(uint32_t, h);
    }
}

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;

__device__ inline float pair_max(float x) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ inline float pair_sum(float x) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Scores of keys a column does not see: element i is logical key jbase + 8 (i / 4) + i % 4.
__device__ __forceinline__ void prefill_mask(f32x16& s, int jbase, int jmax) {
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int j = jbase + 8 * (i >> 2) + (i & 3);
        if (j < 0 || j > jmax) s[i] = -INFINITY;
    }
}

// One online softmax step over a tile's scores: pr = 2^(s - m), l and O
// rescaled where m moves.
template <int D>
__device__ __forceinline__ void prefill_softmax(const f32x16& s, f32x16 (&o)[D / 32], float& m, float& lsum,
                                                float (&pr)[16]) {
    float tmax = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) tmax = fmaxf(tmax, s[i]);
    tmax = pair_max(tmax);
    // Lazy rescale: a column keeps its running max m until a tile's max
    // exceeds it by more than 8 (log2 units), so P <= 2^8 and O and l are
    // rescaled only when some column of the wave moves that far (the first
    // tile with a visible key, then rarely).  The result is the same
    // softmax: O and l share the scale.
    if (__any(tmax > m + 8.0f)) {
        // only the lanes whose max moves rescale (alpha 0 while m = -inf);
        // the others keep alpha = 1 exactly, also a column with no visible
        // key yet (m = -inf, where m - m would be NaN)
        const bool up = tmax > m + 8.0f;
        const float alpha = up ? __builtin_amdgcn_exp2f(m - tmax) : 1.0f;
        if (up) m = tmax;
        lsum *= alpha;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
    }
    const float m_use = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        pr[i] = __builtin_amdgcn_exp2f(s[i] - m_use);
        lsum += pr[i];
    }
}

// max over the lanes {l, l^16, l^32, l^48} (the four quads holding one column),
// with gfx950's VALU lane swaps.
__device__ inline float quad_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

}  // namespace zr
