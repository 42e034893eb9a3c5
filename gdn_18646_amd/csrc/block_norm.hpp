// What the block-norm kernels (block_norm.hip, block_norm_bwd.hip) share: the
// parameter block, eight-element loads and stores, gate activations, row sums
// and the launch's choice of lanes per row.
//
// A row of D elements is held by LPR lanes, NV vectors of 8 elements each:
// lane l's vector u is columns 8 (l + LPR u) .. + 7, so 16 neighbouring lanes
// hold 128 adjacent columns.  Rows are read once and stay in registers between
// their sums and what is written from them.
//
// Where 16-byte accesses do not fit (VEC false: D no multiple of 8, or rows at
// odd addresses) the lane with the row's end loads its last 8 columns, some of
// which belong to the lane before it; the sums take each from its own lane.  That
// way every load is whole and all are under way at once; loading the end element
// by element made that wave wait for each tensor in turn (backward, bf16,
// 16384 x 1001, 512 workgroups: 199 us against 115).
#pragma once

#include "gdn_common.hpp"

namespace gdn_block {

struct NormParams {
    const void *y, *residual, *gate, *post_gamma, *gamma, *scale;  // residual .. scale: null where there is none
    long long ldy, ldr, ldg;
    unsigned rows_per_gate;  // row r takes gate row r / rows_per_gate
    float rs, eps;
    int act;
    void *h, *n;  // null: not written
    long long ldh, ldn;
    uint8_t *codes, *scales;  // null: not quantised
    long long ldc, lds;
    float *rstd_y, *rstd_h;
    int R, D;
    float inv_D;
};

struct NormBwdParams {
    const void *dh, *dn, *y, *residual, *gate, *post_gamma, *gamma, *scale;
    long long lddh, lddn, ldy, ldr, ldg;
    unsigned rows_per_gate;
    float rs;
    int act;
    const float *rstd_y, *rstd_h;
    void *dresidual, *dy, *dgate;  // contiguous; dgate: a row each (per-token gate) or null
    float* part;                   // [groups * chunks][2][D] column sums
    int R, D;
    int group_rows, chunks;  // rows of a gate group, workgroups a group
    float inv_D;
    int shared;              // rows share gate rows: the column sums leave the gate to the second launch
};

}  // namespace gdn_block

namespace {

using namespace gdn;
using gdn_block::NormBwdParams;
using gdn_block::NormParams;

// The first of the 8 columns that the lane of columns c .. c + 7 holds, without VEC.
__device__ __forceinline__ int vector_at(int c, int D) { return max(min(c, D - 8), 0); }
// Whether the lane's element e is one of its own columns c .. c + 7, and inside the row.
template <bool VEC>
__device__ __forceinline__ bool own(int c, int e, int D) {
    const int at = vector_at(c, D);
    return VEC ? c < D : e >= c - at && at + e < D;
}

// Eight elements of a row as they lie in memory.
template <class T>
struct Oct {
    u32x4 w[sizeof(T) / 2];

    // The lane's 8 columns (vector_at(c, D) .. + 7) of the row at element `row`.
    // Lanes past the end read some of the row's; the callers drop them, and the
    // repeated elements of a row of fewer than 8.
    template <bool VEC>
    __device__ __forceinline__ static Oct load(const void* base, long long row, int c, int D) {
        const T* p = static_cast<const T*>(base) + row;
        Oct o;
        if constexpr (VEC) {
            const u32x4* q = reinterpret_cast<const u32x4*>(p + (c < D ? c : 0));
#pragma unroll
            for (unsigned i = 0; i < sizeof(T) / 2; ++i) o.w[i] = q[i];
        } else if (D >= 8) {
            __builtin_memcpy(o.w, p + vector_at(c, D), 8 * sizeof(T));  // 16-byte loads at any address
        } else {
            T e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = p[min(i, D - 1)];
            __builtin_memcpy(o.w, e, 8 * sizeof(T));
        }
        return o;
    }
    __device__ __forceinline__ void get(float* f) const {
        if constexpr (sizeof(T) == 2) {
            unpack8(w[0], f);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i / 4][i % 4]);
        }
    }
};

// WHOLE (without VEC): the lane with the row's end stores all its 8 columns, so
// two lanes write the same values to some (backward, bf16, 16000 x 500: 41 us, 51
// without).  The forward pass, whose h may take the residual's place, lets each
// column's own lane write it, as the other may be in a wave that has yet to read
// it (no slower there).
template <class T, bool VEC, bool WHOLE>
__device__ __forceinline__ void store8(void* base, long long row, int c, int D, const float* f) {
    T* p = static_cast<T*>(base) + row;
    u32x4 w[sizeof(T) / 2];
    if constexpr (sizeof(T) == 2) {
        w[0] = u32x4{pack2_bf16(f[0], f[1]), pack2_bf16(f[2], f[3]), pack2_bf16(f[4], f[5]), pack2_bf16(f[6], f[7])};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i / 4][i % 4] = __float_as_uint(f[i]);
    }
    if (c >= D) return;
    if constexpr (VEC) {
        u32x4* q = reinterpret_cast<u32x4*>(p + c);
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) / 2; ++i) q[i] = w[i];
    } else if (WHOLE ? D >= 8 : c + 8 <= D) {
        __builtin_memcpy(p + vector_at(c, D), w, 8 * sizeof(T));
    } else {
        const int at = vector_at(c, D);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + i >= c && at + i < D) p[at + i] = static_cast<T>(f[i]);
    }
}

// The values of columns vector_at .. + 7 moved down by `shift` to those of c .. c + 7, zeros past the row's end.
__device__ __forceinline__ void to_natural(float* f, int shift, int D) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < D ? f[e] : 0.f;
#pragma unroll
    for (int o = 4; o; o >>= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = shift & o ? (e + o < 8 ? f[e + o] : 0.f) : f[e];
    if (shift >= 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.f;
    }
}

// act(g) of eight gates and, with DERIV, its derivative, on the hardware's exp2
// and reciprocal (about 1 ulp each).
__device__ __forceinline__ float fast_sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}
// Around 0, where 1 - 2 / (1 + e^2x) cancels, the Taylor series to x^11 (its next
// term is 6e-8 of x at 0.4).
__device__ __forceinline__ float fast_tanh(float x) {
    const float far = fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.8853900817779268f * x)), 1.f);
    const float s = x * x;
    float p = fmaf(s, -8.8632355e-3f, 2.1869488e-2f);
    p = fmaf(s, p, -5.3968254e-2f);
    p = fmaf(s, p, 1.3333333e-1f);
    p = fmaf(s, p, -3.3333333e-1f);
    return s < 0.16f ? fmaf(x * s, p, x) : far;
}
template <bool DERIV>
__device__ __forceinline__ void act8(const float* g, int act, float* a, float* d) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        a[e] = g[e];
        if (DERIV) d[e] = 1.f;
    }
    if (act == GDN_ACT_NONE) return;
    if (act == GDN_ACT_TANH) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            a[e] = fast_tanh(g[e]);
            if (DERIV) d[e] = fmaf(-a[e], a[e], 1.f);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float s = fast_sigmoid(g[e]);
        const float ds = s * (1.f - s);
        a[e] = act == GDN_ACT_SILU ? g[e] * s : s;
        if (DERIV) d[e] = act == GDN_ACT_SILU ? fmaf(g[e], ds, s) : ds;
    }
}

// Sum over the LPR lanes of a row, the same in each of them, in a fixed order.
// `slot`: the call's own LDS words (a row's calls and the next row's use
// different ones, so one barrier a call is enough).
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* slot) {
    if constexpr (LPR <= 32) {
        v = sum8(v);
        v += dpp_f<0x140>(v);  // row_mirror: the 16-lane row's sum
        if constexpr (LPR == 32) v += __shfl_xor(v, 16);
        return v;
    } else {
        v = wave_sum_dpp(v);
        if constexpr (LPR == 64) return v;
        constexpr int W = LPR / 64;
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) s += slot[i];
        return s;
    }
}

// Lanes a row and vectors a lane for rows of D: f(LPR, NV).  Up to 512 columns a
// part of a wave or a wave, above that a workgroup, one vector a lane as far as
// that goes (the backward pass, which holds three times as much, has two a lane
// from 4096 columns on, sixteen waves having too few registers).
template <bool BWD, class F>
int with_row_shape(int D, bool vec, F&& f) {
    using std::integral_constant;
    const auto shape = [&](auto v) {
        if (D <= 128) return f(integral_constant<int, 16>{}, integral_constant<int, 1>{}, v);
        if (D <= 256) return f(integral_constant<int, 32>{}, integral_constant<int, 1>{}, v);
        if (D <= 512) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{}, v);
        if (D <= 1024) return f(integral_constant<int, 128>{}, integral_constant<int, 1>{}, v);
        if (D <= 2048) return f(integral_constant<int, 256>{}, integral_constant<int, 1>{}, v);
        if (D <= 4096) return f(integral_constant<int, 512>{}, integral_constant<int, 1>{}, v);
        if constexpr (BWD) {
            if (D <= 8192) return f(integral_constant<int, 512>{}, integral_constant<int, 2>{}, v);
        } else {
            if (D <= 8192) return f(integral_constant<int, 1024>{}, integral_constant<int, 1>{}, v);
        }
        return f(integral_constant<int, 1024>{}, integral_constant<int, 2>{}, v);
    };
    return vec ? shape(std::true_type{}) : shape(std::false_type{});
}
// Rows a workgroup holds at a time.
constexpr int slots_of(int lpr) { return lpr <= 64 ? 256 / lpr : 1; }

constexpr int kMostColumns = 16384;

// The element types of a call: f(TY, TR, TP) of y, gate and n; of the residual
// stream; of the parameters.
inline bool types_ok(int ty, int tr, int tp) {
    return (ty == GDN_BF16 && tr == GDN_BF16 && tp == GDN_BF16) || (ty == GDN_BF16 && tr == GDN_BF16 && tp == GDN_F32) ||
           (ty == GDN_BF16 && tr == GDN_F32 && tp == GDN_F32) || (ty == GDN_F32 && tr == GDN_F32 && tp == GDN_F32);
}
template <class F>
int with_types(int ty, int tr, int tp, F&& f) {
    if (ty == GDN_F32) return f(0.f, 0.f, 0.f);
    if (tr == GDN_F32) return f(bf16(), 0.f, 0.f);
    if (tp == GDN_F32) return f(bf16(), bf16(), 0.f);
    return f(bf16(), bf16(), bf16());
}

// (mean + eps)^-1/2 of a sum of squares, 1 ulp.  The hardware's takes subnormal
// numbers, rows of under 1e-19 without eps, for zero.
__device__ __forceinline__ float rstd_of(float sum, float inv_D, float eps) {
    const float v = fmaf(sum, inv_D, eps);
    const bool tiny = v < 0x1p-126f;
    return __builtin_amdgcn_rsqf(tiny ? v * 0x1p32f : v) * (tiny ? 0x1p16f : 1.f);
}

inline size_t type_bytes(int t) { return t == GDN_F32 ? 4 : 2; }

// Whether rows of type t at p with stride ld take 16-byte accesses (rows of a
// null pointer do).
inline bool vec_rows(const void* p, long long ld, int t) {
    return !p || (gdn_host::aligned(p, 16) && ld * static_cast<long long>(type_bytes(t)) % 16 == 0);
}

}  // namespace
