// What the block-norm kernels (block_norm.hip, block_norm_bwd.hip) share: the
// parameter block, eight-element loads and stores, gate activations, row sums
// and the launch's choice of lanes per row.
//
// A row of D elements is held by LPR lanes, NV vectors of 8 elements each:
// lane l's vector u is columns 8 (l + LPR u) .. + 7, so 16 neighbouring lanes
// hold 128 adjacent columns.  Rows are read once and stay in registers between
// their sums and what is written from them.
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
    int shared;              // rows share gate rows: the column sums leave the gate to the second launch
};

}  // namespace gdn_block

namespace {

using namespace gdn;
using gdn_block::NormBwdParams;
using gdn_block::NormParams;

// Eight elements of a row as they lie in memory.
template <class T>
struct Oct {
    u32x4 w[sizeof(T) / 2];

    // Columns c .. c + 7 of the row at `row` of D columns; columns past the end
    // repeat one inside it (the callers drop them).  VEC: rows and D allow
    // 16-byte loads.
    template <bool VEC>
    __device__ __forceinline__ static Oct load(const void* base, long long row, int c, int D) {
        const T* p = static_cast<const T*>(base) + row;
        Oct o;
        if constexpr (VEC) {
            const u32x4* q = reinterpret_cast<const u32x4*>(p + (c < D ? c : 0));
#pragma unroll
            for (unsigned i = 0; i < sizeof(T) / 2; ++i) o.w[i] = q[i];
        } else {
            T e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = p[min(c + i, D - 1)];
#pragma unroll
            for (unsigned i = 0; i < sizeof(T) / 2; ++i) o.w[i] = reinterpret_cast<const u32x4*>(e)[i];
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

template <class T, bool VEC>
__device__ __forceinline__ void store8(void* base, long long row, int c, int D, const float* f) {
    T* p = static_cast<T*>(base) + row;
    if constexpr (VEC) {
        if (c >= D) return;
        u32x4* q = reinterpret_cast<u32x4*>(p + c);
        if constexpr (sizeof(T) == 2) {
            q[0] = u32x4{pack2_bf16(f[0], f[1]), pack2_bf16(f[2], f[3]), pack2_bf16(f[4], f[5]), pack2_bf16(f[6], f[7])};
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                q[i] = u32x4{__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                             __float_as_uint(f[4 * i + 3])};
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < D) p[c + i] = static_cast<T>(f[i]);
    }
}

// act(g) and its derivative.
__device__ __forceinline__ float act_f(float g, int act) {
    switch (act) {
        case GDN_ACT_SIGMOID: return sigmoid_f(g);
        case GDN_ACT_SILU: return g * sigmoid_f(g);
        case GDN_ACT_TANH: return tanhf(g);
        default: return g;
    }
}
__device__ __forceinline__ float act_grad_f(float g, int act) {
    switch (act) {
        case GDN_ACT_SIGMOID: {
            const float s = sigmoid_f(g);
            return s * (1.f - s);
        }
        case GDN_ACT_SILU: {
            const float s = sigmoid_f(g);
            return s * (1.f + g * (1.f - s));
        }
        case GDN_ACT_TANH: {
            const float t = tanhf(g);
            return 1.f - t * t;
        }
        default: return 1.f;
    }
}

// Sum over the LPR lanes of a row, the same in each of them, in a fixed order.
// `slot`: the call's own LDS words (a kernel's calls use different ones, so one
// barrier a call is enough within a row).
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

// Lanes a row and vectors a lane for rows of D: f(LPR, NV).  Up to 512 columns
// a part of a wave or a wave with one vector, up to 2048 a wave, above that a
// workgroup with two vectors a lane.  Rows that 16-byte accesses do not fit run
// on two of these forms.
template <class F>
int with_row_shape(int D, bool vec, F&& f) {
    using std::integral_constant;
    if (!vec) {
        if (D <= 2048) return f(integral_constant<int, 64>{}, integral_constant<int, 4>{}, std::false_type{});
        return f(integral_constant<int, 1024>{}, integral_constant<int, 2>{}, std::false_type{});
    }
    if (D <= 128) return f(integral_constant<int, 16>{}, integral_constant<int, 1>{}, std::true_type{});
    if (D <= 256) return f(integral_constant<int, 32>{}, integral_constant<int, 1>{}, std::true_type{});
    if (D <= 512) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{}, std::true_type{});
    if (D <= 2048) return f(integral_constant<int, 64>{}, integral_constant<int, 4>{}, std::true_type{});
    if (D <= 4096) return f(integral_constant<int, 256>{}, integral_constant<int, 2>{}, std::true_type{});
    if (D <= 8192) return f(integral_constant<int, 512>{}, integral_constant<int, 2>{}, std::true_type{});
    return f(integral_constant<int, 1024>{}, integral_constant<int, 2>{}, std::true_type{});
}

// The same for the backward pass, which holds three times as much a column: one
// vector a lane up to 8192 columns.
template <class F>
int with_row_shape_bwd(int D, bool vec, F&& f) {
    using std::integral_constant;
    if (!vec) {
        if (D <= 2048) return f(integral_constant<int, 256>{}, integral_constant<int, 1>{}, std::false_type{});
        if (D <= 8192) return f(integral_constant<int, 1024>{}, integral_constant<int, 1>{}, std::false_type{});
        return f(integral_constant<int, 1024>{}, integral_constant<int, 2>{}, std::false_type{});
    }
    if (D <= 128) return f(integral_constant<int, 16>{}, integral_constant<int, 1>{}, std::true_type{});
    if (D <= 256) return f(integral_constant<int, 32>{}, integral_constant<int, 1>{}, std::true_type{});
    if (D <= 512) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{}, std::true_type{});
    if (D <= 2048) return f(integral_constant<int, 256>{}, integral_constant<int, 1>{}, std::true_type{});
    if (D <= 4096) return f(integral_constant<int, 512>{}, integral_constant<int, 1>{}, std::true_type{});
    if (D <= 8192) return f(integral_constant<int, 1024>{}, integral_constant<int, 1>{}, std::true_type{});
    return f(integral_constant<int, 1024>{}, integral_constant<int, 2>{}, std::true_type{});
}

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

inline size_t type_bytes(int t) { return t == GDN_F32 ? 4 : 2; }

// Whether rows of type t at p with stride ld take 16-byte accesses (rows of a
// null pointer do).
inline bool vec_rows(const void* p, long long ld, int t) {
    return !p || (gdn_host::aligned(p, 16) && ld * static_cast<long long>(type_bytes(t)) % 16 == 0);
}

}  // namespace
