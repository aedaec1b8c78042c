// The global norm of many tensors and their scaling by it, for gfx950.
//
//   norm = sqrt(sum x^2) or max |x| over every element of every tensor;  out = x * min(1, max_norm / (norm + eps)).
//
// The tensors' addresses and sizes travel in the kernels' arguments, TABLE of them to a launch: no table in device
// memory to copy and none kept.  A workgroup owns one piece of one tensor (found by bisection of the pieces before
// each), so sums of squares land in a fixed place each and are added in a fixed order: no atomics, the same bits every
// time.  Squares are summed in 64 bits: neither their range (1e20^2 overflows 32 bits) nor the length of the sum
// matters, and one 64-bit FMA per element stays well under the time of its load.  HBM-bound: one read for the norm, one
// read (from the Infinity Cache where the tensors fit) and one write for the scaling.  1.41 GB of bf16 in
// 84 tensors: 846 us, 5.0 TB/s over the three passes.  320 small fp32 tensors (80 MB): 64 us of kernels, in seven launches.
// Tensors at addresses that are no multiple of 16 bytes go element by element: 80 MB of bf16, norm 38 us against 17, scaling 46
// against 28.
#include <algorithm>
#include <vector>

#include "gdn_common.h"
#include "gdn_host.h"
#include "gdn_vec.h"
#include "../../include/gdn_mi355x.h"

namespace gdn {
namespace clip {

constexpr int NT = 256;
constexpr int V = 8;
constexpr int STEP = NT * V;     // elements a workgroup takes at a time
constexpr int TABLE = 120;       // tensors to a launch: 32 bytes each, under the 4 KiB of kernel arguments
constexpr int MAX_PARTS = 4096;  // pieces aimed at over all tensors, beyond one per tensor

struct Entry {
    const void *x;
    void *y;
    int64_t n;
    int first;  // the first piece of this tensor in the launch
    int dt;
};
struct Table {
    Entry e[TABLE];
    int count, part0;  // part0: the launch's first piece among all
    int64_t piece;     // elements of a piece, a multiple of STEP
};

__device__ __forceinline__ int find(const Table &t, int b) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.e[mid].first <= b) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Both start addresses allow vector loads (pieces start at multiples of STEP).
__device__ __forceinline__ bool wide(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <bool INF>
__device__ __forceinline__ double add(double s, float x) {
    if constexpr (INF) {
        const double a = fabs((double)x);
        return a > s || a != a ? a : s;  // a NaN stays
    } else {
        return fma((double)x, (double)x, s);
    }
}
template <bool INF>
__device__ __forceinline__ double join(double a, double b) {
    if constexpr (INF) return b > a || b != b ? b : a;
    else return a + b;
}

// The workgroup's value of s, in thread 0, joined in a fixed order.
template <bool INF>
__device__ __forceinline__ double block_join(double s) {
    __shared__ double red[NT];
    red[threadIdx.x] = s;
    __syncthreads();
#pragma unroll
    for (int h = NT / 2; h >= 1; h >>= 1) {
        if ((int)threadIdx.x < h) red[threadIdx.x] = join<INF>(red[threadIdx.x], red[threadIdx.x + h]);
        __syncthreads();
    }
    return red[0];
}

template <bool INF>
__global__ __launch_bounds__(NT) void norm_kernel(const Table t, double *part) {
    const Entry &e = t.e[find(t, blockIdx.x)];
    const int64_t i0 = (blockIdx.x - e.first) * t.piece, end = min(e.n, i0 + t.piece);
    double s[2] = {0., 0.};
    if (wide(e.x)) {
        int64_t i = i0 + threadIdx.x * V;
        for (; i + STEP + V <= end; i += 2 * STEP) {
            float a[V], b[V];
            ops::loadv<V>(e.x, i, e.dt, a);
            ops::loadv<V>(e.x, i + STEP, e.dt, b);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s[0] = add<INF>(s[0], a[j]);
                s[1] = add<INF>(s[1], b[j]);
            }
        }
        for (; i < end; i += STEP) {
            if (i + V <= end) {
                float a[V];
                ops::loadv<V>(e.x, i, e.dt, a);
#pragma unroll
                for (int j = 0; j < V; ++j) s[0] = add<INF>(s[0], a[j]);
            } else {
                for (int64_t j = i; j < end; ++j) s[0] = add<INF>(s[0], load_as_f32(e.x, j, e.dt));
            }
        }
    } else {
        for (int64_t i = i0 + threadIdx.x; i < end; i += NT) s[0] = add<INF>(s[0], load_as_f32(e.x, i, e.dt));
    }
    const double r = block_join<INF>(join<INF>(s[0], s[1]));
    if (threadIdx.x == 0) part[t.part0 + blockIdx.x] = r;
}

// norm[0] = the norm; factor[0] = what the tensors are multiplied by.
template <bool INF>
__global__ __launch_bounds__(NT) void total_kernel(const double *part, int n, double max_norm, double eps, float *norm,
                                                   float *factor) {
    double s = 0.;
    for (int i = threadIdx.x; i < n; i += NT) s = join<INF>(s, part[i]);
    s = block_join<INF>(s);
    if (threadIdx.x == 0) {
        if (!INF) s = sqrt(s);
        norm[0] = (float)s;
        const double f = max_norm / (s + eps);
        factor[0] = (float)(f > 1. ? 1. : f);  // NaN stays
    }
}

__global__ __launch_bounds__(NT) void scale_kernel(const Table t, const float *factor) {
    const float f = factor[0];
    const Entry &e = t.e[find(t, blockIdx.x)];
    if (f == 1.f && e.x == e.y) return;
    const int64_t i0 = (blockIdx.x - e.first) * t.piece, end = min(e.n, i0 + t.piece);
    if (wide(e.x) && wide(e.y)) {
        for (int64_t i = i0 + threadIdx.x * V; i < end; i += STEP) {
            if (i + V <= end) {
                float a[V];
                ops::loadv<V>(e.x, i, e.dt, a);
#pragma unroll
                for (int j = 0; j < V; ++j) a[j] *= f;
                ops::storev<V>(e.y, i, e.dt, a);
            } else {
                for (int64_t j = i; j < end; ++j) store_from_f32(e.y, j, load_as_f32(e.x, j, e.dt) * f, e.dt);
            }
        }
    } else {
        for (int64_t i = i0 + threadIdx.x; i < end; i += NT)
            store_from_f32(e.y, i, load_as_f32(e.x, i, e.dt) * f, e.dt);
    }
}

// Elements of a piece: few pieces for few elements (the smallest piece keeps every thread busy 4 times), about
// MAX_PARTS for many.
static int64_t piece_of(int64_t total) {
    const int64_t p = (total + MAX_PARTS - 1) / MAX_PARTS;
    return std::max<int64_t>(4 * STEP, (p + STEP - 1) / STEP * STEP);
}
static int64_t bytes_of(int dt) { return dt == DT_F32 ? 4 : 2; }

}  // namespace clip
}  // namespace gdn

using namespace gdn;

extern "C" size_t gdn_clip_grad_norm_workspace_bytes(const int64_t *numel, int count) {
    if (!numel || count <= 0) return 256;
    int64_t total = 0, parts = 0;
    for (int i = 0; i < count; ++i) total += std::max<int64_t>(numel[i], 0);
    const int64_t piece = clip::piece_of(total);
    for (int i = 0; i < count; ++i) parts += (std::max<int64_t>(numel[i], 0) + piece - 1) / piece;
    return 256 + align_up256((size_t)parts * sizeof(double));
}

extern "C" int gdn_clip_grad_norm(const void *const *x, void *const *y, const int64_t *numel, const int *dtypes,
                                  int count, int norm_inf, double max_norm, double eps, float *norm, void *workspace,
                                  size_t workspace_bytes, void *stream) {
    clear_error();
    if (count < 0) return fail(GDN_ERR_INVALID, "count must be >= 0");
    if (!norm || (count && (!x || !numel || !dtypes))) return fail(GDN_ERR_INVALID, "null pointer");
    if (y && !(max_norm >= 0.)) return fail(GDN_ERR_INVALID, "max_norm must be >= 0");
    int64_t total = 0;
    for (int i = 0; i < count; ++i) {
        if (numel[i] < 0) return fail(GDN_ERR_INVALID, "tensor %d has a negative size", i);
        if (dtypes[i] != GDN_F32 && dtypes[i] != GDN_BF16 && dtypes[i] != GDN_F16)
            return fail(GDN_ERR_INVALID, "tensor %d has an unknown dtype code", i);
        if (numel[i] && (!x[i] || (y && !y[i]))) return fail(GDN_ERR_INVALID, "tensor %d has a null pointer", i);
        total += numel[i];
    }
    const int64_t piece = clip::piece_of(total);
    if (y) {
        // every output is written by one workgroup per piece, beside the others: none may share memory with another
        // output, nor with an input other than its own
        struct Span {
            uintptr_t lo, hi;
            int i, out;
        };
        try {
            // most callers' lists run through memory in order: the two are merged then, not sorted
            std::vector<Span> s[2];
            const auto less = [](const Span &a, const Span &b) { return a.lo < b.lo; };
            for (int i = 0; i < count; ++i) {
                if (!numel[i]) continue;
                const uintptr_t o = reinterpret_cast<uintptr_t>(y[i]), in = reinterpret_cast<uintptr_t>(x[i]);
                const uintptr_t len = (uintptr_t)(numel[i] * clip::bytes_of(dtypes[i]));
                s[0].push_back({o, o + len, i, 1});
                if (o != in) s[1].push_back({in, in + len, i, 0});
            }
            for (auto &v : s)
                if (!std::is_sorted(v.begin(), v.end(), less)) std::sort(v.begin(), v.end(), less);
            std::vector<Span> all(s[0].size() + s[1].size());
            std::merge(s[0].begin(), s[0].end(), s[1].begin(), s[1].end(), all.begin(), less);
            uintptr_t out_end = 0, any_end = 0;
            int out_i = 0, any_i = 0;
            for (const Span &v : all) {
                if (v.lo < out_end || (v.out && v.lo < any_end))
                    return fail(GDN_ERR_INVALID, "tensors %d and %d share memory that is written", v.i,
                                v.lo < out_end ? out_i : any_i);
                if (v.out && v.hi > out_end) { out_end = v.hi; out_i = v.i; }
                if (v.hi > any_end) { any_end = v.hi; any_i = v.i; }
            }
        } catch (...) {
            return fail(GDN_ERR_WORKSPACE, "out of host memory");
        }
    }
    const size_t need = gdn_clip_grad_norm_workspace_bytes(numel, count);
    if (!workspace || workspace_bytes < need)
        return fail(GDN_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %zu bytes required",
                    workspace_bytes, need);
    float *factor = static_cast<float *>(workspace);
    double *part = reinterpret_cast<double *>(static_cast<char *>(workspace) + 256);
    hipStream_t st = static_cast<hipStream_t>(stream);
    int64_t parts = 0;
    for (int pass = 0; pass < (y ? 2 : 1); ++pass) {
        clip::Table t;
        t.piece = piece;
        t.count = 0;
        int64_t blocks = 0, part0 = 0;
        for (int i = 0; i <= count; ++i) {
            const int64_t nb = i < count ? (numel[i] + piece - 1) / piece : 0;
            if (t.count && (i == count || t.count == clip::TABLE || blocks + nb > (1 << 23))) {
                t.part0 = (int)part0;
                {
                    Timed tm(pass ? "clip_scale" : "clip_norm", st);
                    const dim3 grid((unsigned)blocks), block(clip::NT);
                    if (pass) hipLaunchKernelGGL(clip::scale_kernel, grid, block, 0, st, t, factor);
                    else if (norm_inf) hipLaunchKernelGGL(clip::norm_kernel<true>, grid, block, 0, st, t, part);
                    else hipLaunchKernelGGL(clip::norm_kernel<false>, grid, block, 0, st, t, part);
                }
                const int rc = check_launch(st, "gdn_clip_grad_norm");
                if (rc) return rc;
                part0 += blocks;
                blocks = 0;
                t.count = 0;
            }
            if (nb) {
                t.e[t.count++] = {x[i], y ? y[i] : nullptr, numel[i], (int)blocks, dtypes[i]};
                blocks += nb;
            }
        }
        if (pass == 0) {
            parts = part0;
            Timed tm("clip_total", st);
            if (norm_inf)
                hipLaunchKernelGGL(clip::total_kernel<true>, dim3(1), dim3(clip::NT), 0, st, part, (int)parts,
                                   max_norm, eps, norm, factor);
            else
                hipLaunchKernelGGL(clip::total_kernel<false>, dim3(1), dim3(clip::NT), 0, st, part, (int)parts,
                                   max_norm, eps, norm, factor);
            const int rc = check_launch(st, "gdn_clip_grad_norm");
            if (rc) return rc;
        }
    }
    return GDN_OK;
}
