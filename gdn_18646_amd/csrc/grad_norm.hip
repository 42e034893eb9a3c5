// The 2-norm of many tensors together, and their clipping to it:
//   norm = sqrt(sum over tensors, elements of g^2)
//   out = g min(1, max_norm / (norm + 1e-6))
//
// Squares are summed in 64 bits: those of no 32-bit number leave their range, and
// the sum of billions keeps every bit that the 32-bit result has.  At two
// instructions an element that is far below what reading them costs.
//
// The tensors' table travels in the launch's parameter block (kTensors a launch, or
// kFew), so a call copies nothing and can be captured.  They are cut into chunks, which a fixed
// number of workgroups takes in turn; each leaves one sum, and the sums are added in a
// fixed order: by a launch of one workgroup, or, where the tensors fit one launch, by
// every workgroup of the clipping one for itself (at most kGroups sums from the L2).
//
// Bound by reading: the norm of 404 MB (bf16, 48 tensors) takes 72 us, 5.6 TB/s, where a
// copy of 512 MB moves 5.3.  Clipping reads twice; up to some 256 MB the second read
// comes from the last-level cache: 202 MB in and out in 94 us on the same tensors again and
// again, of which that cache keeps parts, and in 101 on three sets in turn.
#include <math.h>

#include <algorithm>
#include <exception>
#include <vector>

#include "gdn_common.hpp"

namespace {

using namespace gdn;

constexpr int kTensors = 128;    // a launch: 28 bytes each of the 4 KB that parameters may have
constexpr int kFew = 16;         // of a smaller table, for calls with no more: 12 tensors take 6.1 us of host time and 7.0 clipped, with the full one 6.7 and 8.0
constexpr int kGroups = 2048;    // workgroups a launch: eight a CU
constexpr int kChunk = 16384;    // elements
constexpr int kThreads = 256;
constexpr int64_t kMost = int64_t{1} << 37;  // elements of a tensor: a launch's chunks are numbered in 31 bits
static_assert(kMost / kChunk * kTensors < int64_t{1} << 31, "chunks of a launch");

template <int MOST>
struct GradTable {
    static constexpr int most = MOST;
    const void* grad[MOST];
    void* out[MOST];
    long long n[MOST];
    unsigned first[MOST];  // the tensor's first chunk
    unsigned f32[(MOST + 31) / 32], f32_out[(MOST + 31) / 32];  // bits: fp32, else bf16
    unsigned chunks;
    int count;
    __host__ __device__ static bool bit(const unsigned* b, int i) { return b[i / 32] >> (i % 32) & 1u; }
};

// The tensor of a chunk: the last one whose first chunk is no later.
template <class Table>
__device__ __forceinline__ int tensor_of(const Table& t, unsigned chunk) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first[mid] <= chunk)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

template <class T>
struct Vec {
    static constexpr int n = 16 / sizeof(T);
    __device__ __forceinline__ static u32x4 load(const T* p) {
        u32x4 w;
        __builtin_memcpy(&w, p, 16);  // whole loads at any address
        return w;
    }
    __device__ __forceinline__ static void get(const u32x4 w, float* f) {
        if constexpr (sizeof(T) == 2) {
            unpack8(w, f);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
        }
    }
};

__device__ __forceinline__ void add_square(double& s, float f) {
    const double d = f;
    s = fma(d, d, s);
}

// A chunk's `m` elements from p on: the thread's squares.
template <class T>
__device__ __forceinline__ void add_squares(const T* p, int m, double (&s)[4]) {
    using V = Vec<T>;
    constexpr int kStep = kThreads * V::n, kDeep = 8;
    int at = static_cast<int>(threadIdx.x) * V::n;
    for (; at + (kDeep - 1) * kStep + V::n <= m; at += kDeep * kStep) {
        u32x4 w[kDeep];
#pragma unroll
        for (int i = 0; i < kDeep; ++i) w[i] = V::load(p + at + i * kStep);
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
            float f[V::n];
            V::get(w[i], f);
#pragma unroll
            for (int j = 0; j < V::n; ++j) add_square(s[j % 4], f[j]);
        }
    }
    for (; at < m; at += kStep) {
        if (at + V::n <= m) {
            float f[V::n];
            V::get(V::load(p + at), f);
#pragma unroll
            for (int j = 0; j < V::n; ++j) add_square(s[j % 4], f[j]);
        } else {
            for (int j = at; j < m; ++j) add_square(s[0], static_cast<float>(p[j]));
        }
    }
}

// Sum over the workgroup, in a fixed order, the same in every thread.
template <int THREADS>
__device__ __forceinline__ double group_sum(double v, double* slot) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) v += slot[i];
    return v;
}

template <class Table>
__global__ __launch_bounds__(kThreads) void gdn_square_sums_kernel(Table t, double* sums) {
    __shared__ double slot[kThreads / 64];
    double s[4] = {0., 0., 0., 0.};
    for (unsigned c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = tensor_of(t, c);
        const long long at = static_cast<long long>(c - t.first[i]) * kChunk;
        const int m = static_cast<int>(min(t.n[i] - at, static_cast<long long>(kChunk)));
        if (Table::bit(t.f32, i))
            add_squares(static_cast<const float*>(t.grad[i]) + at, m, s);
        else
            add_squares(static_cast<const bf16*>(t.grad[i]) + at, m, s);
    }
    const double v = group_sum<kThreads>((s[0] + s[1]) + (s[2] + s[3]), slot);
    if (threadIdx.x == 0) sums[blockIdx.x] = v;
}

// The sum of n partial sums, each thread's share first.
template <int THREADS>
__device__ __forceinline__ double total(const double* sums, int n, double* slot) {
    double s[4] = {0., 0., 0., 0.};
    int i = threadIdx.x;
    for (; i + 3 * THREADS < n; i += 4 * THREADS) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += sums[i + j * THREADS];
    }
    for (; i < n; i += THREADS) s[0] += sums[i];
    return group_sum<THREADS>((s[0] + s[1]) + (s[2] + s[3]), slot);
}

// norm from n partial sums; the total of the squares at `all` where it is not null.
__global__ __launch_bounds__(1024) void gdn_grad_norm_kernel(const double* sums, int n, float* norm, double* all) {
    __shared__ double slot[16];
    const double v = total<1024>(sums, n, slot);
    if (threadIdx.x != 0) return;
    *norm = static_cast<float>(sqrt(v));
    if (all) *all = v;
}

// o = p f 2^e.  e is 0 but for factors below fp32's normal numbers, which would lose bits
// there (all of them below 2^-150) while their products may be anything up to 4: for those f
// is 1/2 to 1, so that no product overflows, and the power of two is exact where the result is normal.
template <class T, class O>
__device__ __forceinline__ void scale_chunk(const T* p, O* o, int m, float f, int e) {
    using V = Vec<T>;
    constexpr int kStep = kThreads * V::n, kDeep = 4;
    const auto put = [&](int at, const u32x4 w) {
        float v[V::n];
        V::get(w, v);
        typedef O vec __attribute__((ext_vector_type(V::n), aligned(sizeof(O))));  // whole stores at any address
        vec r;
#pragma unroll
        for (int j = 0; j < V::n; ++j) r[j] = static_cast<O>(__builtin_amdgcn_ldexpf(v[j] * f, e));
        // Past the caches, which hold gradients yet to be read: 202 MB of bf16 into other
        // tensors take 94 us with the norm, 108 through them; in place 94 either way (the same
        // tensors again and again; three sets in turn 101, in place 117).
        __builtin_nontemporal_store(r, reinterpret_cast<vec*>(o + at));
    };
    int at = static_cast<int>(threadIdx.x) * V::n;
    for (; at + (kDeep - 1) * kStep + V::n <= m; at += kDeep * kStep) {
        u32x4 w[kDeep];
#pragma unroll
        for (int i = 0; i < kDeep; ++i) w[i] = V::load(p + at + i * kStep);
#pragma unroll
        for (int i = 0; i < kDeep; ++i) put(at + i * kStep, w[i]);
    }
    for (; at < m; at += kStep) {
        if (at + V::n <= m) {
            put(at, V::load(p + at));
        } else {
            for (int j = at; j < m; ++j) o[j] = static_cast<O>(__builtin_amdgcn_ldexpf(static_cast<float>(p[j]) * f, e));
        }
    }
}

// n partial sums (one: the total); norm: null where another launch writes it.
template <class Table>
__global__ __launch_bounds__(kThreads) void gdn_clip_kernel(Table t, const double* sums, int n, double max_norm, float* norm) {
    __shared__ double slot[kThreads / 64];
    const double root = sqrt(total<kThreads>(sums, n, slot));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(root);
    const double q = max_norm / (root + 1e-6);
    int e = 0;
    const float f = q >= 1. ? 1.f : static_cast<float>(q < 0x1p-126 ? frexp(q, &e) : q);  // NaN stays NaN, and inf / inf is one
    for (unsigned c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = tensor_of(t, c);
        const long long at = static_cast<long long>(c - t.first[i]) * kChunk;
        const int m = static_cast<int>(min(t.n[i] - at, static_cast<long long>(kChunk)));
        const bool f32 = Table::bit(t.f32, i), f32_out = Table::bit(t.f32_out, i);
        if (f == 1.f && t.grad[i] == t.out[i]) continue;  // in place, within the norm: as it is
        if (f32) {
            const float* const p = static_cast<const float*>(t.grad[i]) + at;
            if (f32_out)
                scale_chunk(p, static_cast<float*>(t.out[i]) + at, m, f, e);
            else
                scale_chunk(p, static_cast<bf16*>(t.out[i]) + at, m, f, e);
        } else {
            const bf16* const p = static_cast<const bf16*>(t.grad[i]) + at;
            if (f32_out)
                scale_chunk(p, static_cast<float*>(t.out[i]) + at, m, f, e);
            else
                scale_chunk(p, static_cast<bf16*>(t.out[i]) + at, m, f, e);
        }
    }
}

size_t bytes_of(int type) { return type == GDN_F32 ? 4 : 2; }

// Partial sums of all launches, then the total.
size_t sums_of(int64_t count) { return static_cast<size_t>((count + kTensors - 1) / kTensors) * kGroups; }

int check(const char* who, const gdn_grad_t* grads, int64_t count, const float* norm, bool clip, const void* workspace, size_t bytes) {
    using gdn_host::aligned;
    using gdn_host::fail;
    if (count < 0 || count > 1 << 24) return fail(GDN_ERR_INVALID_ARGUMENT, "%s: %lld tensors", who, (long long)count);
    if (!norm || !aligned(norm, 4) || (count > 0 && !grads)) return fail(GDN_ERR_INVALID_ARGUMENT, "%s: null pointer argument", who);
    if (!workspace || !aligned(workspace, 8) || bytes < gdn_grad_norm_workspace_bytes(count))
        return fail(GDN_ERR_WORKSPACE, "%s: workspace of %zu bytes (8-byte aligned), %zu needed", who, bytes, gdn_grad_norm_workspace_bytes(count));
    for (int64_t i = 0; i < count; ++i) {
        const gdn_grad_t& g = grads[i];
        if ((g.type != GDN_BF16 && g.type != GDN_F32) || (clip && g.type_out != GDN_BF16 && g.type_out != GDN_F32))
            return fail(GDN_ERR_UNSUPPORTED, "%s: type of tensor %lld (bf16 and fp32 are supported)", who, (long long)i);
        if (g.n < 0 || g.n > kMost) return fail(GDN_ERR_INVALID_ARGUMENT, "%s: tensor %lld has %lld elements", who, (long long)i, (long long)g.n);
        if (g.n > 0 && (!g.grad || !aligned(g.grad, bytes_of(g.type)) || (clip && (!g.out || !aligned(g.out, bytes_of(g.type_out))))))
            return fail(GDN_ERR_INVALID_ARGUMENT, "%s: tensor %lld is null or unaligned", who, (long long)i);
    }
    return GDN_OK;
}

// What is written must not be read or written as another tensor.
int check_apart(const char* who, const gdn_grad_t* grads, int64_t count) try {
    using gdn_host::fail;
    struct Span {
        uintptr_t from, to;
        int64_t i;
    };
    std::vector<Span> out;
    out.reserve(static_cast<size_t>(count));
    for (int64_t i = 0; i < count; ++i)
        if (grads[i].n > 0) {
            const auto at = reinterpret_cast<uintptr_t>(grads[i].out);
            out.push_back({at, at + static_cast<size_t>(grads[i].n) * bytes_of(grads[i].type_out), i});
        }
    const auto before = [](const Span& a, const Span& b) { return a.from < b.from; };
    if (!std::is_sorted(out.begin(), out.end(), before)) std::sort(out.begin(), out.end(), before);
    for (size_t k = 1; k < out.size(); ++k)
        if (out[k].from < out[k - 1].to)
            return fail(GDN_ERR_INVALID_ARGUMENT, "%s: tensors %lld and %lld share memory", who, (long long)out[k - 1].i, (long long)out[k].i);
    for (int64_t i = 0; i < count; ++i) {
        const gdn_grad_t& g = grads[i];
        if (g.n == 0) continue;
        const auto from = reinterpret_cast<uintptr_t>(g.grad), to = from + static_cast<size_t>(g.n) * bytes_of(g.type);
        auto k = std::lower_bound(out.begin(), out.end(), Span{to, 0, 0}, before);  // the first that begins behind it
        while (k != out.begin() && (--k)->to > from)
            if (k->i != i || k->from != from || g.type != g.type_out)
                return fail(GDN_ERR_INVALID_ARGUMENT, "%s: the result of tensor %lld lies over tensor %lld", who, (long long)k->i, (long long)i);
    }
    return GDN_OK;
} catch (const std::exception& e) {
    return gdn_host::fail(GDN_ERR_INVALID_ARGUMENT, "%s: %lld tensors: %s", who, (long long)count, e.what());
}

// Calls f(table) for the tensors that have elements, up to Table::most at a time.
template <class Table, class F>
int for_tables(const gdn_grad_t* grads, int64_t count, bool clip, F&& f) {
    Table t = {};
    const auto flush = [&]() {
        const int st = t.count ? f(t) : GDN_OK;
        t = Table();
        return st;
    };
    for (int64_t i = 0; i < count; ++i) {
        const gdn_grad_t& g = grads[i];
        if (g.n == 0) continue;
        const int64_t chunks = (g.n + kChunk - 1) / kChunk;
        if (t.count == Table::most) {
            const int st = flush();
            if (st != GDN_OK) return st;
        }
        const int k = t.count++;
        t.grad[k] = g.grad, t.out[k] = clip ? g.out : nullptr, t.n[k] = g.n, t.first[k] = t.chunks;
        t.f32[k / 32] |= (g.type == GDN_F32 ? 1u : 0u) << (k % 32);
        t.f32_out[k / 32] |= (clip && g.type_out == GDN_F32 ? 1u : 0u) << (k % 32);
        t.chunks += static_cast<unsigned>(chunks);
    }
    return flush();
}

template <class Table>
unsigned groups_of(const Table& t) { return std::min<unsigned>(t.chunks, kGroups); }

}  // namespace

extern "C" size_t gdn_grad_norm_workspace_bytes(int64_t count) {
    return count < 0 ? 0 : (sums_of(count) + 1) * sizeof(double);
}

namespace {

// The partial sums of every tensor; their number in *n, the launches in *launches.
template <class Table>
int square_sums(const gdn_grad_t* grads, int64_t count, double* sums, int64_t* n, int* launches, hipStream_t stream) {
    *n = 0;
    *launches = 0;
    return for_tables<Table>(grads, count, false, [&](const Table& t) {
        const unsigned groups = groups_of(t);
        hipLaunchKernelGGL(gdn_square_sums_kernel<Table>, dim3(groups), dim3(kThreads), 0, stream, t, sums + *n);
        *n += groups;
        ++*launches;
        return gdn_host::check_launch("gdn_square_sums_kernel");
    });
}

int finish_norm(const double* sums, int64_t n, float* norm, double* all, hipStream_t stream) {
    hipLaunchKernelGGL(gdn_grad_norm_kernel, dim3(1), dim3(1024), 0, stream, sums, static_cast<int>(n), norm, all);
    return gdn_host::check_launch("gdn_grad_norm_kernel");
}

template <class Table>
int norm_of(const gdn_grad_t* grads, int64_t count, float* norm, double* sums, hipStream_t s) {
    int64_t n;
    int launches;
    const int st = square_sums<Table>(grads, count, sums, &n, &launches, s);
    return st == GDN_OK ? finish_norm(sums, n, norm, nullptr, s) : st;
}

template <class Table>
int clip(const gdn_grad_t* grads, int64_t count, double max_norm, float* norm, double* sums, hipStream_t s) {
    int64_t n;
    int launches, st = square_sums<Table>(grads, count, sums, &n, &launches, s);
    if (st != GDN_OK) return st;
    double* const all = sums + n;
    const bool one = launches == 1;
    if (!one) {
        st = finish_norm(sums, n, norm, all, s);
        if (st != GDN_OK) return st;
    }
    return for_tables<Table>(grads, count, true, [&](const Table& t) {
        hipLaunchKernelGGL(gdn_clip_kernel<Table>, dim3(groups_of(t)), dim3(kThreads), 0, s, t, one ? sums : all, one ? static_cast<int>(n) : 1,
                           max_norm, one ? norm : nullptr);
        return gdn_host::check_launch("gdn_clip_kernel");
    });
}

}  // namespace

extern "C" int gdn_grad_norm_hip(const gdn_grad_t* grads, int64_t count, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = check("grad_norm", grads, count, norm, false, workspace, workspace_bytes);
    if (st != GDN_OK) return st;
    const auto f = count <= kFew ? norm_of<GradTable<kFew>> : norm_of<GradTable<kTensors>>;
    return f(grads, count, norm, static_cast<double*>(workspace), static_cast<hipStream_t>(stream));
}

extern "C" int gdn_clip_grad_norm_hip(const gdn_grad_t* grads, int64_t count, double max_norm, float* norm, void* workspace,
                                      size_t workspace_bytes, void* stream) {
    if (!(max_norm >= 0)) return gdn_host::fail(GDN_ERR_INVALID_ARGUMENT, "clip_grad_norm: max_norm=%g", max_norm);
    int st = check("clip_grad_norm", grads, count, norm, true, workspace, workspace_bytes);
    if (st == GDN_OK) st = check_apart("clip_grad_norm", grads, count);
    if (st != GDN_OK) return st;
    const auto f = count <= kFew ? clip<GradTable<kFew>> : clip<GradTable<kTensors>>;
    return f(grads, count, max_norm, norm, static_cast<double*>(workspace), static_cast<hipStream_t>(stream));
}
