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
//
// What bounds it: HBM for many rows (16384 x 2048 in bf16, five inputs and three
// outputs: 118 us, 4.6 TB/s), with three waves a SIMD at 168 registers; the chain
// of loads and two row sums, and the second launch, for few (333 x 1001 in fp32:
// 7.0 + 3.6 us).  The next row's loads are under way while a row is worked on.
// Rows of over 8192 columns spill (2048 x 16384: 306 us, 1.75 TB/s), and fp32 ones
// of over 4096 a little.
#include "block_norm.hpp"

namespace {

template <class TY, class TR, class TP, int LPR, int NV, bool VEC>
__global__ __launch_bounds__(LPR <= 64 ? 256 : LPR) __attribute__((amdgpu_waves_per_eu(LPR >= 1024 ? 4 : VEC && NV == 1 && LPR >= 128 && sizeof(TR) == 2 ? 3 : 2))) void gdn_block_norm_bwd_kernel(NormBwdParams p) {
    constexpr int SLOTS = slots_of(LPR);
    constexpr bool kAhead = NV == 1;  // the next row is loaded a row ahead (with two vectors a lane it does not fit)
    constexpr bool kShared = LPR <= 64;  // several rows at a time: their column sums meet in LDS
    constexpr bool kLds = LPR == 1024;   // the lane's column sums lie in LDS, and its parameters are read a row
    __shared__ float sums[2][2][LPR > 64 ? LPR / 64 : 1];
    __shared__ __attribute__((aligned(16))) float cols[kShared || kLds ? 2 * LPR * NV * 8 : 1];
    const int tid = threadIdx.x, lane = tid % LPR;
    const int D = p.D;
    const int group = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
    const long long first = static_cast<long long>(group) * p.group_rows;
    const int end = static_cast<int>(min(first + p.group_rows, static_cast<long long>(p.R)));
    const long long step = static_cast<long long>(p.chunks) * SLOTS;
    auto inside = [&](int u, int e) { return own<VEC>(8 * (lane + LPR * u), e, D); };

    struct Row {
        Oct<TY> y[NV], dn[NV], g[NV];
        Oct<TR> r[NV], dh[NV];
        float ry, rh;
    };
    auto load = [&](long long base, Row& w) {
        const long long r = min(base + tid / LPR, static_cast<long long>(end - 1));
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int c = 8 * (lane + LPR * u);
            w.y[u] = Oct<TY>::template load<VEC>(p.y, r * p.ldy, c, D);
            if (p.dh) w.dh[u] = Oct<TR>::template load<VEC>(p.dh, r * p.lddh, c, D);
            if (p.residual && p.dn) w.r[u] = Oct<TR>::template load<VEC>(p.residual, r * p.ldr, c, D);
            if (p.dn) w.dn[u] = Oct<TY>::template load<VEC>(p.dn, r * p.lddn, c, D);
            if (p.gate && !p.shared) w.g[u] = Oct<TY>::template load<VEC>(p.gate, r * p.ldg, c, D);
        }
        w.ry = p.rstd_y ? p.rstd_y[r] : 1.f;
        w.rh = p.rstd_h ? p.rstd_h[r] : 1.f;
    };
    long long base = first + static_cast<long long>(chunk) * SLOTS;
    Row cur;
    if (base < end) load(base, cur);

    // The lane's columns: rs post_gamma scale (times a shared gate's act), gamma,
    // the sums of e a (of e with a shared gate) and of dn hn.
    float ps[NV][8], gm[NV][8], se[kLds ? 1 : NV][8], sg[kLds ? 1 : NV][8];
    auto params = [&](int u) {
        const int c = 8 * (lane + LPR * u);
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            ps[u][e] = p.rs;
            gm[u][e] = 0.f;
        }
        if (p.post_gamma) {
            Oct<TP>::template load<VEC>(p.post_gamma, 0, c, D).get(t);
#pragma unroll
            for (int e = 0; e < 8; ++e) ps[u][e] *= t[e];
        }
        if (p.scale) {
            Oct<TP>::template load<VEC>(p.scale, 0, c, D).get(t);
#pragma unroll
            for (int e = 0; e < 8; ++e) ps[u][e] *= t[e];
        }
        if (p.gate && p.shared) {
            float a[8];
            Oct<TY>::template load<VEC>(p.gate, group * p.ldg, c, D).get(t);
            act8<false>(t, p.act, a, nullptr);
#pragma unroll
            for (int e = 0; e < 8; ++e) ps[u][e] *= a[e];
        }
        if (p.gamma) Oct<TP>::template load<VEC>(p.gamma, 0, c, D).get(gm[u]);
    };
    // Adds v to the sums `which` (0: e a, 1: dn hn) of vector u's columns.
    auto add = [&](int which, int u, const float* v) {
        if constexpr (kLds) {
            f32x4* const at = reinterpret_cast<f32x4*>(cols + ((which * NV + u) * LPR + lane) * 8);
#pragma unroll
            for (int i = 0; i < 2; ++i) at[i] += f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) (which ? sg : se)[u][e] += v[e];
        }
    };
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        if constexpr (kLds) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                reinterpret_cast<f32x4*>(cols + (((i >> 1) * NV + u) * LPR + lane) * 8)[i & 1] = f32x4{0.f, 0.f, 0.f, 0.f};
        } else {
            params(u);
#pragma unroll
            for (int e = 0; e < 8; ++e) se[u][e] = sg[u][e] = 0.f;
        }
    }

    for (int parity = 0; base < end; parity ^= 1) {
        Row next;
        const bool more = base + step < end;
        if (kAhead && more) load(base + step, next);
        const long long r = base + tid / LPR;
        const bool live = r < end;

        // The gate's act (a, of a gate a token) and derivative (da), y rstd_y.
        float a[NV][8], da[NV][8], yn[NV][8], dH[NV][8], hn[NV][8];
        float m = 0.f;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            if constexpr (kLds) params(u);
            float t[8];
            if (p.gate && !p.shared) {
                cur.g[u].get(t);
                act8<true>(t, p.act, a[u], da[u]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) a[u][e] = 1.f;
            }
            cur.y[u].get(yn[u]);
#pragma unroll
            for (int e = 0; e < 8; ++e) yn[u][e] = !VEC || inside(u, e) ? yn[u][e] * cur.ry : 0.f;
            if (p.dh) {
                cur.dh[u].get(dH[u]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) dH[u][e] = 0.f;
            }
            if (p.dn) {  // h again, and what comes through the second norm
                float dn[8];
                if (p.residual) {
                    cur.r[u].get(t);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) t[e] = 0.f;
                }
                cur.dn[u].get(dn);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    hn[u][e] = fmaf(ps[u][e] * a[u][e], yn[u][e], t[e]) * cur.rh;
                    const float tt = dn[e] * gm[u][e];
                    if (inside(u, e)) m = fmaf(tt, hn[u][e], m);
                    dn[e] = live ? dn[e] * hn[u][e] : 0.f;
                    dH[u][e] = fmaf(tt, cur.rh, dH[u][e]);
                }
                add(1, u, dn);
            }
        }
        if (p.dn) {
            m = row_sum<LPR>(m, sums[parity][0]) * p.inv_D * cur.rh;
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) dH[u][e] = fmaf(-m, hn[u][e], dH[u][e]);
        }
        if (p.dresidual && live) {
#pragma unroll
            for (int u = 0; u < NV; ++u) store8<TR, VEC, true>(p.dresidual, r * D, 8 * (lane + LPR * u), D, dH[u]);
        }

        // dgate, the column sums, and z (which takes dH's place)
        float q = 0.f;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            float dg[8], ea[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float ev = dH[u][e] * yn[u][e];  // without rs, which the sums' launch puts in
                if (p.dgate) dg[e] = ev * ps[u][e] * da[u][e];
                ea[e] = live ? ev * a[u][e] : 0.f;
                dH[u][e] *= ps[u][e] * a[u][e];
                if (inside(u, e)) q = fmaf(dH[u][e], yn[u][e], q);
            }
            add(0, u, ea);
            if (p.dgate && live) store8<TY, VEC, true>(p.dgate, r * D, 8 * (lane + LPR * u), D, dg);
        }
        if (p.rstd_y) {
            q = row_sum<LPR>(q, sums[parity][1]) * p.inv_D;
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) dH[u][e] = cur.ry * fmaf(-yn[u][e], q, dH[u][e]);
        }
        if (live) {
#pragma unroll
            for (int u = 0; u < NV; ++u) store8<TY, VEC, true>(p.dy, r * D, 8 * (lane + LPR * u), D, dH[u]);
        }
        if (!more) break;
        base += step;
        if (kAhead)
            cur = next;
        else
            load(base, cur);
    }
    if (!p.part) return;

    // The workgroup's sums: rows of one wave by lane exchange, its waves one
    // after the other in LDS.
    float* const out = p.part + static_cast<size_t>(blockIdx.x) * 2 * D;
    if constexpr (!kShared) {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int c = 8 * (lane + LPR * u);
            store8<float, VEC, true>(out, 0, c, D, kLds ? cols + (u * LPR + lane) * 8 : se[kLds ? 0 : u]);
            store8<float, VEC, true>(out, D, c, D, kLds ? cols + ((NV + u) * LPR + lane) * 8 : sg[kLds ? 0 : u]);
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
                        const int at = 8 * (lane + LPR * u), c = (VEC ? at : vector_at(at, D)) + e;
                        if (!VEC && !inside(u, e)) continue;
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

// Adds the sums of `chunks` workgroups of each of `groups` groups (one, at
// blockIdx.y, where there are more than kGroups), 16 columns a workgroup, 64 rows
// of sums at a time, and writes what follows from them: the gradient of a shared
// gate row, and the parameters' gradients or (part2) the group's part of them.
constexpr int kGroups = 32;
struct SumParams {
    const float* part;
    int groups, share;  // share: the 64 rows' part for a group, 64 / (groups up to a power of two)
    int chunks, D;
    float rs;
    const void *gate, *post_gamma, *scale;
    long long ldg;
    int act;
    void *dgate, *dpost_gamma, *dscale, *dgamma;
    float* part2;
};

template <class TY, class TP>
__global__ __launch_bounds__(1024) void gdn_block_norm_sum_kernel(SumParams p) {
    __shared__ float lds[2][64][17];
    const int col = threadIdx.x & 15, lane = threadIdx.x >> 4, d = blockIdx.x * 16 + col, D = p.D, S = p.share;
    const long long first = blockIdx.y;
    float e = 0.f, s = 0.f;
    if (d < D && lane / S < p.groups) {
        const float* src = p.part + static_cast<size_t>(first + lane / S) * p.chunks * 2 * D + d;
#pragma unroll 4
        for (int i = lane % S; i < p.chunks; i += S) {
            e += src[static_cast<size_t>(i) * 2 * D];
            s += src[static_cast<size_t>(i) * 2 * D + D];
        }
    }
    lds[0][lane][col] = e;
    lds[1][lane][col] = s;
    __syncthreads();
    const float pg = d < D && p.post_gamma ? static_cast<float>(static_cast<const TP*>(p.post_gamma)[d]) : 1.f;
    const float sc = d < D && p.scale ? static_cast<float>(static_cast<const TP*>(p.scale)[d]) : 1.f;
    // Of group lane / 2, the sum of e (even lanes; then what it makes for the gate) or of s.
    const int g = lane >> 1, which = lane & 1;
    float sum = 0.f;
    if (g < p.groups) {
        for (int i = 0; i < S; ++i) sum += lds[which][g * S + i][col];
        if (which == 0) {
            sum *= p.rs;
            if (p.gate && d < D) {
                float x[8], a[8], da[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(static_cast<const TY*>(p.gate)[(first + g) * p.ldg + d]);
                act8<true>(x, p.act, a, da);
                if (p.dgate) static_cast<TY*>(p.dgate)[(first + g) * D + d] = static_cast<TY>(sum * pg * sc * da[0]);
                sum *= a[0];
            }
        }
    }
    __syncthreads();
    lds[which][g][col] = sum;
    __syncthreads();
    if (threadIdx.x >= 16 || d >= D) return;
    e = s = 0.f;
    for (int i = 0; i < p.groups; ++i) {
        e += lds[0][i][col];
        s += lds[1][i][col];
    }
    if (p.part2) {
        p.part2[static_cast<size_t>(first) * 2 * D + d] = e;
        p.part2[static_cast<size_t>(first) * 2 * D + D + d] = s;
        return;
    }
    if (p.dpost_gamma) static_cast<TP*>(p.dpost_gamma)[d] = static_cast<TP>(e * sc);
    if (p.dscale) static_cast<TP*>(p.dscale)[d] = static_cast<TP>(e * pg);
    if (p.dgamma) static_cast<TP*>(p.dgamma)[d] = static_cast<TP>(s);
}

// How R rows with a gate row each `per` are split over workgroups: 512 of them in
// all, two a CU, while each has a row for every one of its slots (16384 x 2048:
// 118 us with 512, 171 with 256, 134 with 1024).  Rows of over 2048 columns have
// workgroups of eight waves and more, 256 of them (8192 x 4096: 129 us, 134 with
// 512); rows of 513 to 1024 have two waves, and 1024 workgroups if each walks
// four rows at least (bf16, 16384 x 1024: 67 us, 99 with 512; 1500 rows: 20.8,
// 19.2 with 512; fp32, 8192 x 1024: 63.5 against 59).
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
    const long long all = D > 2048 ? 256 : D > 512 && D <= 1024 && R >= 4096 ? 1024 : 512, most = (all + q.groups - 1) / q.groups, need = (rows + slots - 1) / slots;
    q.chunks = static_cast<int>(need < most ? need : most);
    return q;
}

}  // namespace

extern "C" size_t gdn_block_norm_bwd_workspace_bytes(int64_t R, int64_t D, int64_t rows_per_gate) {
    if (R <= 0 || D <= 0) return 0;
    const Plan q = plan_rows(R, D, rows_per_gate);
    return static_cast<size_t>(q.groups) * (q.chunks + (q.groups > kGroups ? 1 : 0)) * 2 * D * sizeof(float);
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
        p.R = static_cast<int>(R), p.D = static_cast<int>(D), p.inv_D = 1.f / static_cast<float>(D);
        p.group_rows = q.group_rows, p.chunks = q.chunks, p.shared = shared;
        const int st = with_types(type_y, type_r, type_p, [&](auto ty, auto tr, auto tp) {
            return with_row_shape<true>(p.D, vec, [&](auto lpr, auto nv, auto v) {
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
    t.rs = residual_scale;
    t.part = part, t.chunks = R > 0 ? q.chunks : 0, t.D = static_cast<int>(D);
    t.post_gamma = post_gamma, t.scale = scale, t.act = act, t.dpost_gamma = dpost_gamma, t.dscale = dscale, t.dgamma = dgamma;
    if (shared && R > 0) t.gate = gate, t.ldg = ldg, t.dgate = dgate;
    // Up to kGroups groups in one launch; more in one that sums each and one that adds them.
    const bool apart = q.groups > kGroups;
    float* const part2 = apart ? part + static_cast<size_t>(q.groups) * q.chunks * 2 * D : nullptr;
    t.part2 = part2, t.groups = apart ? 1 : static_cast<int>(q.groups);
    t.share = 64;
    while (t.share * t.groups > 64) t.share /= 2;
    return with_types(type_y, type_r, type_p, [&](auto ty, auto, auto tp) {
        const auto launch = [&](long long count) {
            hipLaunchKernelGGL((gdn_block_norm_sum_kernel<decltype(ty), decltype(tp)>), dim3((t.D + 15) / 16, static_cast<unsigned>(count)),
                               dim3(1024), 0, s, t);
            return gdn_host::check_launch("gdn_block_norm_sum_kernel");
        };
        const int st = launch(apart ? q.groups : 1);
        if (st != GDN_OK || !apart) return st;
        t.part = part2, t.chunks = static_cast<int>(q.groups), t.part2 = nullptr, t.rs = 1.f, t.gate = nullptr, t.dgate = nullptr;
        return launch(1);
    });
}
