// Gradients of the block norms (block_norm.hip).  With yn = y rstd_y (y without
// post_gamma), hn = h rstd_h, a = act(gate), pg, sc = post_gamma, scale or 1:
//   dH     = dh + rstd_h (t - hn mean(t hn)),   t = dn gamma      (dH = dh without gamma)
//   dres   = dH
//   e      = rs dH yn
//   dgate  = e pg sc act'(gate)                 (summed over the rows that share a gate row)
//   dpost_gamma = sum_rows e a sc, dscale = sum_rows e a pg, dgamma = sum_rows dn hn
//   dy     = rstd_y (z - yn mean(z yn)),        z = dH rs sc a pg  (dy = z without post_gamma)
// all in fp32, rounded once where written.  h is computed again from what the
// forward pass read, so nothing but the two rstd a row is kept for this.
//
// Sums over rows: a workgroup walks rows of one gate group and keeps two sums a
// column in registers, of e a (e alone where rows share a gate row: there a and
// act' are the group's own factors) and of dn hn; its sums go to the workspace
// and a second launch adds them in a fixed order, so results do not vary from
// run to run.
#include "block_norm.hpp"

namespace {

template <class TY, class TR, class TP, int LPR, int NV, bool VEC>
__global__ __launch_bounds__(LPR <= 64 ? 256 : LPR) void gdn_block_norm_bwd_kernel(NormBwdParams p) {
    constexpr int SLOTS = LPR <= 64 ? 256 / LPR : 1;
    constexpr bool kShared = LPR <= 64;  // several rows at a time: their column sums meet in LDS
    __shared__ float sums[2][2][LPR > 64 ? LPR / 64 : 1];
    __shared__ float cols[kShared ? 2 * LPR * NV * 8 : 1];
    const int tid = threadIdx.x, lane = tid % LPR;
    const int D = p.D;
    const int group = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
    const long long first = static_cast<long long>(group) * p.group_rows;
    const int end = static_cast<int>(min(first + p.group_rows, static_cast<long long>(p.R)));
    auto inside = [&](int u, int e) { return VEC ? 8 * (lane + LPR * u) < D : 8 * (lane + LPR * u) + e < D; };

    float se[NV][8], sg[NV][8];
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) se[u][e] = sg[u][e] = 0.f;

    int parity = 0;
    for (long long base = first + static_cast<long long>(chunk) * SLOTS; base < end; base += static_cast<long long>(p.chunks) * SLOTS, parity ^= 1) {
        const bool live = base + tid / LPR < end;
        const long long r = live ? base + tid / LPR : end - 1;
        Oct<TY> yr[NV], gr[NV], nr[NV];
        Oct<TR> rr[NV], hr[NV];
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int c = 8 * (lane + LPR * u);
            yr[u] = Oct<TY>::template load<VEC>(p.y, r * p.ldy, c, D);
            if (p.dh) hr[u] = Oct<TR>::template load<VEC>(p.dh, r * p.lddh, c, D);
        }
        if (p.residual) {
#pragma unroll
            for (int u = 0; u < NV; ++u) rr[u] = Oct<TR>::template load<VEC>(p.residual, r * p.ldr, 8 * (lane + LPR * u), D);
        }
        if (p.dn) {
#pragma unroll
            for (int u = 0; u < NV; ++u) nr[u] = Oct<TY>::template load<VEC>(p.dn, r * p.lddn, 8 * (lane + LPR * u), D);
        }
        if (p.gate) {
            const long long g = static_cast<unsigned>(r) / p.rows_per_gate;
#pragma unroll
            for (int u = 0; u < NV; ++u) gr[u] = Oct<TY>::template load<VEC>(p.gate, g * p.ldg, 8 * (lane + LPR * u), D);
        }
        const float ry = p.rstd_y ? p.rstd_y[r] : 1.f, rh = p.rstd_h ? p.rstd_h[r] : 1.f;

        // dH: dh, and through the second norm dn
        float dH[NV][8], hn[NV][8];
        float m = 0.f;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            if (p.dh) {
                hr[u].get(dH[u]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) dH[u][e] = 0.f;
            }
        }
        if (p.dn) {
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                const int c = 8 * (lane + LPR * u);
                float f[8], t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = p.rs * ry;
                if (p.post_gamma) {
                    Oct<TP>::template load<VEC>(p.post_gamma, 0, c, D).get(t);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= t[e];
                }
                if (p.scale) {
                    Oct<TP>::template load<VEC>(p.scale, 0, c, D).get(t);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= t[e];
                }
                if (p.gate) {
                    gr[u].get(t);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= act_f(t[e], p.act);
                }
                float yv[8];
                yr[u].get(yv);
                if (p.residual) {
                    rr[u].get(t);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) t[e] = 0.f;
                }
                float gm[8], dn[8];
                Oct<TP>::template load<VEC>(p.gamma, 0, c, D).get(gm);
                nr[u].get(dn);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    hn[u][e] = fmaf(f[e], yv[e], t[e]) * rh;
                    const float tt = inside(u, e) ? dn[e] * gm[e] : 0.f;
                    if (inside(u, e)) m = fmaf(tt, hn[u][e], m);
                    if (live && inside(u, e)) sg[u][e] = fmaf(dn[e], hn[u][e], sg[u][e]);
                    dH[u][e] = fmaf(tt, rh, dH[u][e]);
                }
            }
            m = row_sum<LPR>(m, sums[parity][0]) / static_cast<float>(D) * rh;
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) dH[u][e] = fmaf(-m, hn[u][e], dH[u][e]);
        }
        if (p.dresidual && live) {
#pragma unroll
            for (int u = 0; u < NV; ++u) store8<TR, VEC>(p.dresidual, r * D, 8 * (lane + LPR * u), D, dH[u]);
        }

        // dgate, the column sums, and z
        float q = 0.f;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int c = 8 * (lane + LPR * u);
            float ps[8], t[8], yv[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) ps[e] = 1.f;
            if (p.post_gamma) Oct<TP>::template load<VEC>(p.post_gamma, 0, c, D).get(ps);
            if (p.scale) {
                Oct<TP>::template load<VEC>(p.scale, 0, c, D).get(t);
#pragma unroll
                for (int e = 0; e < 8; ++e) ps[e] *= t[e];
            }
            yr[u].get(yv);
            if (p.gate) gr[u].get(t);
            float dg[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float yn = yv[e] * ry;
                const float ev = p.rs * dH[u][e] * yn;
                const float a = p.gate ? act_f(t[e], p.act) : 1.f;
                if (p.dgate) dg[e] = ev * ps[e] * act_grad_f(t[e], p.act);
                if (live && inside(u, e)) se[u][e] += p.shared ? ev : ev * a;
                const float z = dH[u][e] * p.rs * ps[e] * a;
                if (inside(u, e)) q = fmaf(z, yn, q);
                dH[u][e] = z;
            }
            if (p.dgate && live) store8<TY, VEC>(p.dgate, r * D, c, D, dg);
        }
        if (p.rstd_y) {
            q = row_sum<LPR>(q, sums[parity][1]) / static_cast<float>(D);
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                float yv[8];
                yr[u].get(yv);
#pragma unroll
                for (int e = 0; e < 8; ++e) dH[u][e] = ry * (dH[u][e] - yv[e] * ry * q);
            }
        }
        if (live) {
#pragma unroll
            for (int u = 0; u < NV; ++u) store8<TY, VEC>(p.dy, r * D, 8 * (lane + LPR * u), D, dH[u]);
        }
    }
    if (!p.part) return;

    // The workgroup's sums: rows of one wave by lane exchange, its waves one
    // after the other in LDS.
    float* const out = p.part + static_cast<size_t>(blockIdx.x) * 2 * D;
    if constexpr (!kShared) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (inside(u, e)) {
                    const int c = 8 * (lane + LPR * u) + e;
                    out[c] = se[u][e];
                    out[D + c] = sg[u][e];
                }
    } else {
        constexpr int kC = LPR * NV * 8;
#pragma unroll
        for (int o = LPR; o < 64; o *= 2)
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    se[u][e] += __shfl_xor(se[u][e], o);
                    sg[u][e] += __shfl_xor(sg[u][e], o);
                }
        for (int w = 0; w < 4; ++w) {
            if (tid / 64 == w && (tid & 63) < LPR) {
#pragma unroll
                for (int u = 0; u < NV; ++u)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int c = 8 * (lane + LPR * u) + e;
                        cols[c] = w == 0 ? se[u][e] : cols[c] + se[u][e];
                        cols[kC + c] = w == 0 ? sg[u][e] : cols[kC + c] + sg[u][e];
                    }
            }
            __syncthreads();
        }
        for (int c = tid; c < D; c += 256) {
            out[c] = cols[c];
            out[D + c] = cols[kC + c];
        }
    }
}

// Adds the sums of `chunks` workgroups of each group (blockIdx.y), 32 columns a
// workgroup, and writes what follows from them: the gradient of a shared gate
// row, and either the parameters' gradients (one group) or the group's part of
// them (part2).
struct SumParams {
    const float* part;
    int chunks, D;
    const void *gate, *post_gamma, *scale;
    long long ldg;
    int act;
    void *dgate, *dpost_gamma, *dscale, *dgamma;
    float* part2;
};

template <class TY, class TP>
__global__ __launch_bounds__(256) void gdn_block_norm_sum_kernel(SumParams p) {
    __shared__ float lds[2][8][32];
    const int col = threadIdx.x & 31, lane = threadIdx.x >> 5, d = blockIdx.x * 32 + col, D = p.D;
    const long long g = blockIdx.y;
    float e = 0.f, s = 0.f;
    if (d < D) {
        const float* src = p.part + static_cast<size_t>(g) * p.chunks * 2 * D + d;
#pragma unroll 4
        for (int i = lane; i < p.chunks; i += 8) {
            e += src[static_cast<size_t>(i) * 2 * D];
            s += src[static_cast<size_t>(i) * 2 * D + D];
        }
    }
    lds[0][lane][col] = e;
    lds[1][lane][col] = s;
    __syncthreads();
    if (lane > 0 || d >= D) return;
    e = s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        e += lds[0][i][col];
        s += lds[1][i][col];
    }
    const float pg = p.post_gamma ? static_cast<float>(static_cast<const TP*>(p.post_gamma)[d]) : 1.f;
    const float sc = p.scale ? static_cast<float>(static_cast<const TP*>(p.scale)[d]) : 1.f;
    if (p.gate) {
        const float x = static_cast<float>(static_cast<const TY*>(p.gate)[g * p.ldg + d]);
        if (p.dgate) static_cast<TY*>(p.dgate)[g * D + d] = static_cast<TY>(e * pg * sc * act_grad_f(x, p.act));
        e *= act_f(x, p.act);
    }
    if (p.part2) {
        p.part2[static_cast<size_t>(g) * 2 * D + d] = e;
        p.part2[static_cast<size_t>(g) * 2 * D + D + d] = s;
        return;
    }
    if (p.dpost_gamma) static_cast<TP*>(p.dpost_gamma)[d] = static_cast<TP>(e * sc);
    if (p.dscale) static_cast<TP*>(p.dscale)[d] = static_cast<TP>(e * pg);
    if (p.dgamma) static_cast<TP*>(p.dgamma)[d] = static_cast<TP>(s);
}

// How R rows with a gate row each `per` are split over workgroups: 512 of them
// in all (two a CU) while each has a row for every one of its slots.
struct Plan {
    long long groups;
    int group_rows, chunks;
};
Plan plan_rows(long long R, long long D, long long per) {
    const bool shared = per > 1 && R > 0;
    const long long rows = shared ? (per < R ? per : R) : (R > 0 ? R : 1);
    const int slots = D <= 128 ? 16 : D <= 256 ? 8 : D <= 512 ? 4 : 1;
    Plan q;
    q.group_rows = static_cast<int>(rows);
    q.groups = shared ? (R + rows - 1) / rows : 1;
    const long long most = (512 + q.groups - 1) / q.groups, need = (rows + slots - 1) / slots;
    q.chunks = static_cast<int>(need < most ? need : most);
    return q;
}

}  // namespace

extern "C" size_t gdn_block_norm_bwd_workspace_bytes(int64_t R, int64_t D, int64_t rows_per_gate) {
    if (R <= 0 || D <= 0) return 0;
    const Plan q = plan_rows(R, D, rows_per_gate);
    return static_cast<size_t>(q.groups) * (q.chunks + (q.groups > 1 ? 1 : 0)) * 2 * D * sizeof(float);
}

extern "C" int gdn_block_norm_bwd_hip(const void* dh, int64_t lddh, const void* dn, int64_t lddn, const void* y, int64_t ldy,
                                      const void* residual, int64_t ldr, const void* gate, int64_t ldg,
                                      int64_t rows_per_gate, const void* post_gamma, const void* gamma, const void* scale,
                                      float residual_scale, int act, const float* rstd_y, const float* rstd_h,
                                      void* dresidual, void* dy, void* dgate, void* dpost_gamma, void* dgamma,
                                      void* dscale, int64_t R, int64_t D, int type_y, int type_r, int type_p,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    using gdn_host::aligned;
    using gdn_host::fail;
    if (R < 0 || D <= 0) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm_bwd: R=%lld D=%lld", (long long)R, (long long)D);
    if (D > kMostColumns || R > 0x7fffffffLL)
        return fail(GDN_ERR_UNSUPPORTED, "block_norm_bwd: R=%lld D=%lld, at most 2^31 - 1 rows of %d", (long long)R, (long long)D, kMostColumns);
    if (!types_ok(type_y, type_r, type_p))
        return fail(GDN_ERR_UNSUPPORTED, "block_norm_bwd: types %d, %d, %d of y, residual and parameters", type_y, type_r, type_p);
    if (act < GDN_ACT_NONE || act > GDN_ACT_TANH) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm_bwd: act=%d", act);
    if (gate && rows_per_gate <= 0) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm_bwd: rows_per_gate=%lld", (long long)rows_per_gate);
    if ((dn != nullptr) != (gamma != nullptr && rstd_h != nullptr))
        return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm_bwd: dn, gamma and rstd_h go together");
    if ((post_gamma != nullptr) != (rstd_y != nullptr)) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm_bwd: post_gamma and rstd_y go together");
    if ((dgate && !gate) || (dresidual && !residual) || (dpost_gamma && !post_gamma) || (dgamma && !gamma) || (dscale && !scale))
        return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm_bwd: a gradient of an absent input");
    if (R > 0 && (!y || !dy || (!dh && !dn))) return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm_bwd: y, dy or both of dh and dn are null");
    const size_t by = type_bytes(type_y), br = type_bytes(type_r), bp = type_bytes(type_p);
    if (!aligned(y, by) || !aligned(dn, by) || !aligned(gate, by) || !aligned(dy, by) || !aligned(dgate, by) ||
        !aligned(dh, br) || !aligned(residual, br) || !aligned(dresidual, br) || !aligned(post_gamma, bp) ||
        !aligned(gamma, bp) || !aligned(scale, bp) || !aligned(dpost_gamma, bp) || !aligned(dgamma, bp) || !aligned(dscale, bp))
        return fail(GDN_ERR_INVALID_ARGUMENT, "block_norm_bwd: a buffer is not aligned to its elements");
    const bool shared = gate && rows_per_gate > 1;
    const bool sums = dpost_gamma || dgamma || dscale || (shared && dgate);
    const Plan q = plan_rows(R, D, gate ? rows_per_gate : 1);
    if (sums && R > 0) {
        const size_t need = gdn_block_norm_bwd_workspace_bytes(R, D, gate ? rows_per_gate : 1);
        if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
            return fail(GDN_ERR_WORKSPACE, "block_norm_bwd: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
    }
    if (q.groups > 65535) return fail(GDN_ERR_UNSUPPORTED, "block_norm_bwd: %lld gate rows, at most 65535 shared ones", q.groups);
    float* const part = sums ? static_cast<float*>(workspace) : nullptr;
    const auto s = static_cast<hipStream_t>(stream);
    if (R > 0) {
        const bool vec = D % 8 == 0 && vec_rows(dh, lddh, type_r) && vec_rows(dn, lddn, type_y) && vec_rows(y, ldy, type_y) &&
                         vec_rows(residual, ldr, type_r) && vec_rows(gate, ldg, type_y) && vec_rows(post_gamma, 0, type_p) &&
                         vec_rows(gamma, 0, type_p) && vec_rows(scale, 0, type_p) && vec_rows(dresidual, D, type_r) &&
                         vec_rows(dy, D, type_y) && vec_rows(dgate, D, type_y);
        NormBwdParams p = {};
        p.dh = dh, p.dn = dn, p.y = y, p.residual = residual, p.gate = gate, p.post_gamma = post_gamma, p.gamma = gamma, p.scale = scale;
        p.lddh = lddh, p.lddn = lddn, p.ldy = ldy, p.ldr = ldr, p.ldg = ldg;
        p.rows_per_gate = static_cast<unsigned>(gate ? (rows_per_gate < R ? rows_per_gate : R) : 1);
        p.rs = residual_scale, p.act = gate ? act : GDN_ACT_NONE;
        p.rstd_y = rstd_y, p.rstd_h = rstd_h;
        p.dresidual = dresidual, p.dy = dy, p.dgate = shared ? nullptr : dgate;
        p.part = part;
        p.R = static_cast<int>(R), p.D = static_cast<int>(D);
        p.group_rows = q.group_rows, p.chunks = q.chunks, p.shared = shared;
        const int st = with_types(type_y, type_r, type_p, [&](auto ty, auto tr, auto tp) {
            return with_row_shape_bwd(p.D, vec, [&](auto lpr, auto nv, auto v) {
                constexpr int LPR = decltype(lpr)::value;
                const dim3 grid(static_cast<unsigned>(q.groups * q.chunks)), block(LPR <= 64 ? 256 : LPR);
                hipLaunchKernelGGL((gdn_block_norm_bwd_kernel<decltype(ty), decltype(tr), decltype(tp), LPR, decltype(nv)::value, decltype(v)::value>),
                                   grid, block, 0, s, p);
                return gdn_host::check_launch("gdn_block_norm_bwd_kernel");
            });
        });
        if (st != GDN_OK || !sums) return st;
    } else if (!sums) {
        return GDN_OK;
    }
    SumParams t = {};
    t.part = part, t.chunks = R > 0 ? q.chunks : 0, t.D = static_cast<int>(D);
    t.post_gamma = post_gamma, t.scale = scale, t.act = act, t.dpost_gamma = dpost_gamma, t.dscale = dscale, t.dgamma = dgamma;
    if (shared && R > 0) t.gate = gate, t.ldg = ldg, t.dgate = dgate;
    float* const part2 = q.groups > 1 ? part + static_cast<size_t>(q.groups) * q.chunks * 2 * D : nullptr;
    t.part2 = part2;
    return with_types(type_y, type_r, type_p, [&](auto ty, auto, auto tp) {
        const auto launch = [&](long long groups) {
            hipLaunchKernelGGL((gdn_block_norm_sum_kernel<decltype(ty), decltype(tp)>), dim3((t.D + 31) / 32, static_cast<unsigned>(groups)),
                               dim3(256), 0, s, t);
            return gdn_host::check_launch("gdn_block_norm_sum_kernel");
        };
        const int st = launch(q.groups);
        if (st != GDN_OK || !part2) return st;
        t.part = part2, t.chunks = static_cast<int>(q.groups), t.part2 = nullptr, t.gate = nullptr, t.dgate = nullptr;
        return launch(1);
    });
}
