// The norms before and after a block, fused with its gate and residual:
//   u = y rstd_y post_gamma            rstd_y = (mean(y^2) + eps)^-1/2   (u = y without post_gamma)
//   h = residual + rs scale act(gate) u                                  (factors that are absent are 1)
//   n = h rstd_h gamma                 rstd_h = (mean(h^2) + eps)^-1/2
// in fp32; h and n are rounded once, where they are written (n follows from the
// unrounded h), and n (h without gamma) may go out as e4m3 codes of 128 with
// their scales instead, what a block-scaled product reads.
//
// What bounds it: HBM for many rows (each input read once, each output written
// once, two row sums between them that never leave the registers), the one
// chain of loads, sums and stores for a few (16384 x 2048, three inputs and two
// outputs in bf16: 63 us, 5.3 TB/s; 24000 x 256, a gated head norm: 10.6 us;
// 1 x 2048: 3.1 us).  Non-temporal stores take 3-13% off the kernel and give it
// back to whoever reads n next (16384 x 2048 with a reader: 85.4 us, 86.4 with
// them).  Rows of up to 4096 columns have a
// workgroup each or share one; rows above that keep sixteen waves busy alone, and
// a workgroup a CU walks them, the next row's loads under way while a row is
// worked on (4096 x 8192: 78 us against 102 with a workgroup a row; walking rows
// of 2048 columns instead took 70 against 64).
#include <stdlib.h>

#include <algorithm>
#include <numeric>

#include "block_norm.hpp"
#include "fp8_blocks.hpp"

namespace {

template <class TY, class TR, class TP, int LPR, int NV, bool VEC>
__global__ __launch_bounds__(LPR <= 64 ? 256 : LPR) void gdn_block_norm_kernel(NormParams p) {
    constexpr int SLOTS = slots_of(LPR);
    constexpr bool kWalk = LPR == 1024;         // a workgroup walks rows
    constexpr bool kAhead = kWalk && NV == 1;  // the next one is loaded a row ahead (with two vectors a lane it does not fit)
    __shared__ float sums[2][2][LPR > 64 ? LPR / 64 : 1];
    const int tid = threadIdx.x, lane = tid % LPR;
    const int D = p.D;
    auto inside = [&](int u, int e) { return own<VEC>(8 * (lane + LPR * u), e, D); };

    struct Row {
        Oct<TY> y[NV], g[NV];
        Oct<TR> r[NV];
    };
    // Rows past the end repeat the last one and write nothing.
    auto load = [&](long long base, Row& w) {
        const long long r = min(base + tid / LPR, static_cast<long long>(p.R - 1));
#pragma unroll
        for (int u = 0; u < NV; ++u) w.y[u] = Oct<TY>::template load<VEC>(p.y, r * p.ldy, 8 * (lane + LPR * u), D);
        if (p.residual) {
#pragma unroll
            for (int u = 0; u < NV; ++u) w.r[u] = Oct<TR>::template load<VEC>(p.residual, r * p.ldr, 8 * (lane + LPR * u), D);
        }
        if (p.gate) {
            const long long g = static_cast<unsigned>(r) / p.rows_per_gate;
#pragma unroll
            for (int u = 0; u < NV; ++u) w.g[u] = Oct<TY>::template load<VEC>(p.gate, g * p.ldg, 8 * (lane + LPR * u), D);
        }
    };
    const long long step = static_cast<long long>(gridDim.x) * SLOTS;
    long long base = static_cast<long long>(blockIdx.x) * SLOTS;
    Row cur;
    load(base, cur);
    // rs post_gamma scale, and gamma, of the lane's columns
    float f[NV][8], gm[NV][8];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int c = 8 * (lane + LPR * u);
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[u][e] = p.rs;
        if (p.post_gamma) {
            Oct<TP>::template load<VEC>(p.post_gamma, 0, c, D).get(t);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[u][e] *= t[e];
        }
        if (p.scale) {
            Oct<TP>::template load<VEC>(p.scale, 0, c, D).get(t);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[u][e] *= t[e];
        }
        if (p.gamma) Oct<TP>::template load<VEC>(p.gamma, 0, c, D).get(gm[u]);
    }

    for (int parity = 0; base < p.R; parity ^= 1) {
        Row next;
        const bool more = kWalk && base + step < p.R;
        if (kAhead && more) load(base + step, next);
        const long long r = base + tid / LPR;
        const bool live = r < p.R;
        float h[NV][8];
        float ss = 0.f;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            cur.y[u].get(h[u]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (VEC && !inside(u, e)) h[u][e] = 0.f;
                if (VEC || inside(u, e)) ss = fmaf(h[u][e], h[u][e], ss);
            }
        }
        float inv = 1.f;
        if (p.post_gamma) {
            inv = rstd_of(row_sum<LPR>(ss, sums[parity][0]), p.inv_D, p.eps);
            if (p.rstd_y && live && lane == 0) p.rstd_y[r] = inv;
        }
        ss = 0.f;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            float t[8], a[8];
            if (p.gate) {
                cur.g[u].get(t);
                act8<false>(t, p.act, a, nullptr);
#pragma unroll
                for (int e = 0; e < 8; ++e) a[e] *= inv * f[u][e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) a[e] = inv * f[u][e];
            }
            if (p.residual) {
                cur.r[u].get(t);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[u][e] = fmaf(a[e], h[u][e], t[e]);
                if (VEC && !inside(u, e)) h[u][e] = 0.f;
                if (VEC || inside(u, e)) ss = fmaf(h[u][e], h[u][e], ss);
            }
            if (p.h && live) store8<TR, VEC, false>(p.h, r * p.ldh, 8 * (lane + LPR * u), D, h[u]);
        }
        inv = 1.f;
        if (p.gamma) {
            inv = rstd_of(row_sum<LPR>(ss, sums[parity][1]), p.inv_D, p.eps);
            if (p.rstd_h && live && lane == 0) p.rstd_h[r] = inv;
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int c = 8 * (lane + LPR * u);
            if (p.gamma) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h[u][e] = h[u][e] * inv * gm[u][e];
                    if (VEC && !inside(u, e)) h[u][e] = 0.f;
                }
            }
            if (p.n && live) store8<TY, VEC, false>(p.n, r * p.ldn, c, D, h[u]);
            if (p.codes) {
                if constexpr (!VEC) to_natural(h[u], c - vector_at(c, D), D);
                const uint32_t s = Fp8<GDN_E4M3>::scale_byte(max16(amax8(h[u])));
                const u32x2 w = Fp8<GDN_E4M3>::codes8(h[u], Fp8<GDN_E4M3>::inverse(s), s == 0xffu);
                if (live && c / kBlk * kBlk < D) {  // a ragged last block is filled up with zero codes
                    *reinterpret_cast<u32x2*>(p.codes + r * p.ldc + c) = w;
                    if ((lane & 15) == 0) p.scales[static_cast<long long>(c / kBlk) * p.lds + r] = static_cast<uint8_t>(s);
                }
            }
        }
        if (!more) break;
        base += step;
        if (kAhead)
            cur = next;
        else
            load(base, cur);
    }
}

// Rows as they lie in memory: how many, the bytes of one and from one to the next.
struct Span {
    const void* at;
    long long rows, bytes, step;
    long long first() const { return static_cast<long long>(reinterpret_cast<uintptr_t>(at)); }
    long long low() const { return first() + std::min(0LL, (rows - 1) * step); }
    long long high() const { return first() + std::max(0LL, (rows - 1) * step) + bytes; }
};

// Whether rows of h may be written while those of an input are read.  A row of an
// input that is a row of h itself has each value read by the lane that writes it,
// before it does; anything else has to lie apart from h for certain: in another
// range of memory, or in other columns of a common step.
bool may_share(const Span& h, const Span& in) {
    if (!h.at || !in.at || h.high() <= in.low() || in.high() <= h.low()) return true;
    if (h.at == in.at && h.rows == in.rows && h.bytes == in.bytes && (h.rows == 1 || h.step == in.step)) return true;
    const long long step = std::gcd(h.rows > 1 ? llabs(h.step) : 0, in.rows > 1 ? llabs(in.step) : 0);
    if (step == 0) return false;
    const long long at = ((in.first() - h.first()) % step + step) % step;
    return at >= h.bytes && at + in.bytes <= step;
}

}  // namespace

extern "C" int gdn_block_norm_hip(const void* y, int64_t ldy, const void* residual, int64_t ldr, const void* gate,
                                  int64_t ldg, int64_t rows_per_gate, const void* post_gamma, const void* gamma,
                                  const void* scale, float residual_scale, int act, float eps, void* h, int64_t ldh,
                                  void* n, int64_t ldn, uint8_t* codes, int64_t ldc, uint8_t* scales, int64_t lds,
                                  float* rstd_y, float* rstd_h, int64_t R, int64_t D, int type_y, int type_r, int type_p,
                                  void* stream) {
    using gdn_host::aligned;
    using gdn_host::fail;
    if (R < 0 || D <= 0) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm: R=%lld D=%lld", (long long)R, (long long)D);
    if (D > kMostColumns || R > 0x7fffffffLL)
        return fail(GDN_ERR_UNSUPPORTED, "block_norm: R=%lld D=%lld, at most 2^31 - 1 rows of %d", (long long)R, (long long)D, kMostColumns);
    if (!types_ok(type_y, type_r, type_p))
        return fail(GDN_ERR_UNSUPPORTED, "block_norm: types %d, %d, %d of y, residual and parameters", type_y, type_r, type_p);
    if (act < GDN_ACT_NONE || act > GDN_ACT_TANH) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm: act=%d", act);
    if ((R > 0 && !y) || (!h && !n && !codes)) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm: y or every output is null");
    if (!gamma && (n || rstd_h)) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm: n and rstd_h need gamma");
    if (!post_gamma && rstd_y) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm: rstd_y needs post_gamma");
    if (gate && rows_per_gate <= 0) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm: rows_per_gate=%lld", (long long)rows_per_gate);
    if (R > 1 && ((h && ldh < D) || (n && ldn < D)))
        return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm: rows of h or n overlap (ldh=%lld, ldn=%lld, D=%lld)", (long long)ldh, (long long)ldn, (long long)D);
    if (codes && (!scales || !aligned(codes, 16) || ldc % 16 != 0 || ldc < (D + kBlk - 1) / kBlk * kBlk || lds < R))
        return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm: codes need scales [D / 128, >= R], 16-byte alignment and rows padded to 128");
    const size_t by = type_bytes(type_y), br = type_bytes(type_r), bp = type_bytes(type_p);
    if (!aligned(y, by) || !aligned(residual, br) || !aligned(gate, by) || !aligned(h, br) || !aligned(n, by) ||
        !aligned(post_gamma, bp) || !aligned(gamma, bp) || !aligned(scale, bp))
        return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm: a buffer is not aligned to its elements");
    if (R == 0) return GDN_OK;
    const bool vec = D % 8 == 0 && vec_rows(y, ldy, type_y) && vec_rows(residual, ldr, type_r) && vec_rows(gate, ldg, type_y) &&
                     vec_rows(h, ldh, type_r) && vec_rows(n, ldn, type_y) && vec_rows(post_gamma, 0, type_p) &&
                     vec_rows(gamma, 0, type_p) && vec_rows(scale, 0, type_p);
    NormParams p = {};
    p.y = y, p.residual = residual, p.gate = gate, p.post_gamma = post_gamma, p.gamma = gamma, p.scale = scale;
    p.ldy = ldy, p.ldr = ldr, p.ldg = ldg;
    p.rows_per_gate = static_cast<unsigned>(rows_per_gate < R ? rows_per_gate : R);
    p.rs = residual_scale, p.eps = eps, p.act = gate ? act : GDN_ACT_NONE;
    p.h = h, p.n = n, p.ldh = ldh, p.ldn = ldn;
    p.codes = codes, p.scales = scales, p.ldc = ldc, p.lds = lds;
    p.rstd_y = rstd_y, p.rstd_h = rstd_h;
    p.R = static_cast<int>(R), p.D = static_cast<int>(D), p.inv_D = 1.f / static_cast<float>(D);
    const auto span = [&](const void* at, long long rows, long long ld, size_t size) {
        return Span{at, rows, D * static_cast<long long>(size), ld * static_cast<long long>(size)};
    };
    const Span written = span(h, R, ldh, br);
    const char* shared = nullptr;  // the input that h would be written over
    const auto check = [&](const char* name, const Span& in) {
        if (!may_share(written, in)) shared = name;
    };
    check("y", span(y, R, ldy, by));
    check("residual", span(residual, R, ldr, br));
    if (gate) check("gate", span(gate, R / rows_per_gate + (R % rows_per_gate != 0), ldg, by));
    check("post_gamma", span(post_gamma, 1, 0, bp));
    check("gamma", span(gamma, 1, 0, bp));
    check("scale", span(scale, 1, 0, bp));
    return with_types(type_y, type_r, type_p, [&](auto ty, auto tr, auto tp) {
        return with_row_shape<false>(p.D, vec, [&](auto lpr, auto nv, auto v) {
            constexpr int LPR = decltype(lpr)::value, threads = LPR <= 64 ? 256 : LPR;
            const int all = static_cast<int>((R + slots_of(LPR) - 1) / slots_of(LPR));
            if (!gdn_host::grid_fits(all, threads)) return fail(GDN_ERR_UNSUPPORTED, "block_norm: R=%lld rows of %lld are too many for a launch", (long long)R, (long long)D);
            if (shared) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm: h would be written to memory locations of %s other than its own row's", shared);
            const dim3 grid(LPR == 1024 && all > 256 ? 256 : all), block(threads);
            hipLaunchKernelGGL((gdn_block_norm_kernel<decltype(ty), decltype(tr), decltype(tp), LPR, decltype(nv)::value, decltype(v)::value>),
                               grid, block, 0, static_cast<hipStream_t>(stream), p);
            return gdn_host::check_launch("gdn_block_norm_kernel");
        });
    });
}
