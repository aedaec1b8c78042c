// Matrix products with plain results, and the join of a split contraction's parts, for gfx950.
#include "gdn_product.h"

namespace gdn {
namespace mm {

// Lanes hold rows of the result and registers its columns: four consecutive columns to a store.
template <class S, bool F16, bool ACC>
__global__ __launch_bounds__(S::NT, S::WAVES_EU) void product_kernel(const Args g, const Result r) {
    __shared__ __attribute__((aligned(16))) char lds[S::LDS];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wm = w / S::WN, wn = w % S::WN;
    products<S, F16>(g, lds, [&](int tm, int tn, const acc_t(&acc)[S::TM][S::TN]) {
        const int64_t m0 = (int64_t)tm * S::BM + wm * (S::BM / S::WM) + 4 * (lane >> 5);
        const int64_t n0 = (int64_t)tn * S::BN + wn * (S::BN / S::WN) + (lane & 31);
        const int e = ACC ? 0 : exponent_of(r);
#pragma unroll
        for (int j = 0; j < S::TN; ++j) {
            const int64_t n = n0 + 32 * j;
            if (n >= g.b.rows) continue;
            float f = 1.f;
            if constexpr (!ACC) f = r.row ? r.row[n] : 1.f;
#pragma unroll
            for (int i = 0; i < S::TM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int64_t m = m0 + 32 * i + 8 * q;
                    float x[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                    if constexpr (ACC) {
                        float *to = r.acc + ((int64_t)blockIdx.z * g.b.rows + n) * g.a.rows + m;
                        if (m + 3 < g.a.rows && g.a.rows % 4 == 0) {
                            float4 v = make_float4(x[0], x[1], x[2], x[3]);
                            if (r.add) {
                                const float4 o = *reinterpret_cast<const float4 *>(to);
                                v = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
                            }
                            *reinterpret_cast<float4 *>(to) = v;
                        } else {
                            for (int k = 0; k < 4; ++k)
                                if (m + k < g.a.rows) to[k] = r.add ? to[k] + x[k] : x[k];
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[k] = f == 0.f ? 0.f : ldexpf(x[k], e) * f;
                        const int64_t at = n * r.ldy + m;
                        if (m + 3 < g.a.rows && r.ldy % 4 == 0) {
                            store4_from_f32(r.y, at, make_float4(x[0], x[1], x[2], x[3]), r.dt);
                        } else {
                            for (int k = 0; k < 4; ++k)
                                if (m + k < g.a.rows) store_from_f32(r.y, at + k, x[k], r.dt);
                        }
                    }
                }
        }
    });
}

constexpr int NT = 256;

__global__ __launch_bounds__(NT) void finish_kernel(const Result r, int splits, int64_t rows, int64_t cols) {
    const int64_t i = (block_index() * NT + threadIdx.x) * 4, size = rows * cols;
    if (i >= size) return;
    const int e = exponent_of(r);
    for (int64_t k = i; k < min(i + 4, size); ++k) {
        float s = 0.f;
        for (int z = 0; z < splits; ++z) s += r.acc[z * size + k];
        const int64_t n = k / cols;
        const float f = r.row ? r.row[n] : 1.f;
        store_from_f32(r.y, n * r.ldy + (k - n * cols), f == 0.f ? 0.f : ldexpf(s, e) * f, r.dt);
    }
}

void finish(const Result &r, int splits, int64_t rows, int64_t cols, hipStream_t st) {
    Timed tm("product_join", st);
    hipLaunchKernelGGL(finish_kernel, grid_of((rows * cols + 4 * NT - 1) / (4 * NT)), dim3(NT), 0, st, r, splits, rows, cols);
}

template <class S>
static void launch(Args &g, bool f16, int splits, const Result &r, hipStream_t st) {
    const dim3 grid = tiles_of<S>(g, splits);
    if (f16 && r.acc) hipLaunchKernelGGL((product_kernel<S, true, true>), grid, dim3(S::NT), 0, st, g, r);
    else if (f16) hipLaunchKernelGGL((product_kernel<S, true, false>), grid, dim3(S::NT), 0, st, g, r);
    else if (r.acc) hipLaunchKernelGGL((product_kernel<S, false, true>), grid, dim3(S::NT), 0, st, g, r);
    else hipLaunchKernelGGL((product_kernel<S, false, false>), grid, dim3(S::NT), 0, st, g, r);
}

void multiply(Args g, bool f16, const Plan &p, const Result &r, hipStream_t st) {
    Timed tm("product", st);
    if (p.shape == BIG) launch<Big>(g, f16, p.splits, r, st);
    else if (p.shape == MID) launch<Mid>(g, f16, p.splits, r, st);
    else if (p.shape == FEW) launch<Few>(g, f16, p.splits, r, st);
    else launch<One>(g, f16, p.splits, r, st);
}

// Few rows: narrow tiles, several to a compute unit, whose loads hide one another's latency.  Else the large tile where
// three quarters of the 256 compute units get one (split along the contraction if need be, 8 blocks to a part at least).
Plan plan(int64_t rows, int64_t cols, int64_t blocks, int max_splits) {
    const auto tiles = [&](int64_t bm, int64_t bn) { return ((cols + bm - 1) / bm) * ((rows + bn - 1) / bn); };
    const auto split = [&](int64_t t, int64_t want) {
        int64_t s = want / t;
        if (s > blocks / 8) s = blocks / 8;
        if (s > max_splits) s = max_splits;
        return (int)(s < 1 ? 1 : s);
    };
    if (rows <= 32) return {ONE, split(tiles(128, 32), 1024)};
    if (rows <= 64) return {FEW, split(tiles(128, 64), 768)};
    const int64_t big = tiles(256, 256);
    const int s = split(big, 256);
    if (big * s >= 192) return {BIG, s};
    return {MID, split(tiles(128, 128), 512)};
}

}  // namespace mm
}  // namespace gdn
