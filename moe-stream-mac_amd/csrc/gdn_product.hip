// Matrix products with plain results, and the join of a split contraction's parts, for gfx950.
#include "gdn_product.h"

namespace gdn {
namespace mm {

enum : int { OUT16 = 0, OUT32 = 1, PARTS = 2 };

template <class S, bool F16, int KIND, bool DOWN>
__global__ __launch_bounds__(S::NT, S::WAVES_EU) void product_kernel(const Args g, const Result r) {
    __shared__ __attribute__((aligned(16))) char lds[S::LDS + S::STORE];
    const int w = wave_index(), wm = w / S::WN, wn = w % S::WN;
    char *st = lds + S::LDS + w * 4096;
    const Extent ext = extent_of<S>(g);
    products<S, F16, DOWN>(g, ext, lds, [&](int tm, int tn, acc_t(&acc)[S::TM][S::TN]) {
        const int lane = lane_here();
        const int64_t m0 = (int64_t)tm * S::BM + wm * (S::BM / S::WM), n0 = (int64_t)tn * S::BN + wn * (S::BN / S::WN);
        const int e = KIND == PARTS ? 0 : exponent_of(r);
#pragma unroll
        for (int j = 0; j < S::TN; j += 2) {
            const int64_t n = n0 + 16 * j, rows = ext.rows_b - n;
            if (rows <= 0) break;
            float f[2] = {1.f, 1.f};
            if constexpr (KIND != PARTS)
                if (r.row) {
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj) f[jj] = r.row[n + min((int64_t)(16 * jj + (lane & 15)), rows - 1)];
                }
            const auto scaled = [&](float x, int jj) { return f[jj] == 0.f ? 0.f : ldexpf(x, e) * f[jj]; };
            if constexpr (KIND == OUT16) {
#pragma unroll
                for (int i = 0; i < S::TM; i += 4) {
                    const int64_t m = m0 + 16 * i;
#pragma unroll
                    for (int ii = 0; ii < 4; ++ii)
#pragma unroll
                        for (int jj = 0; jj < 2; ++jj) {
                            const acc_t &x = acc[i + ii][j + jj];
                            put16(lane, st, ii, jj, ops::pack2_cvt(scaled(x[0], jj), scaled(x[1], jj), r.dt),
                                  ops::pack2_cvt(scaled(x[2], jj), scaled(x[3], jj), r.dt));
                        }
                    store_rows(lane, st, static_cast<char *>(r.y) + (n * r.ldy + m) * 2, (uint32_t)(r.ldy * 2), rows,
                               (g.a.rows - m) * 2, 2);
                }
            } else {
#pragma unroll
                for (int i = 0; i < S::TM; i += 2) {
                    const int64_t m = m0 + 16 * i;
#pragma unroll
                    for (int ii = 0; ii < 2; ++ii)
#pragma unroll
                        for (int jj = 0; jj < 2; ++jj) {
                            float x[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                x[k] = KIND == PARTS ? acc[i + ii][j + jj][k] : scaled(acc[i + ii][j + jj][k], jj);
                            put32(lane, st, ii, jj, x);
                        }
                    if constexpr (KIND == OUT32) {
                        store_rows(lane, st, static_cast<char *>(r.y) + (n * r.ldy + m) * 4, (uint32_t)(r.ldy * 4), rows,
                                   (g.a.rows - m) * 4, 4);
                    } else {
                        char *to = reinterpret_cast<char *>(r.acc + ((int64_t)blockIdx.z * g.b.rows + n) * r.ldp + m);
                        if (r.add) add_rows(lane, st, to, (uint32_t)(r.ldp * 4), rows, (r.ldp - m) * 4);
                        store_rows(lane, st, to, (uint32_t)(r.ldp * 4), rows, (r.ldp - m) * 4, 4);
                    }
                }
            }
        }
    });
}

constexpr int NT = 256;

// Four columns to a thread.
template <int DT>
__global__ __launch_bounds__(NT) void finish_kernel(const Result r, int splits, int64_t rows, int64_t cols) {
    const int64_t per = r.ldp / 4, i = block_index() * NT + threadIdx.x, n = i / per, m = (i - n * per) * 4;
    if (n >= rows) return;
    const int e = exponent_of(r);
    const int64_t at = r.place ? r.place[n] : n;
    const float f = at < 0 ? 0.f : r.row ? r.row[at] : 1.f;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (at < 0) splits = 0;
#pragma unroll 8
    for (int z = 0; z < splits; ++z) {
        const float4 v = *reinterpret_cast<const float4 *>(r.acc + (z * rows + at) * r.ldp + m);
        s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = f == 0.f ? 0.f : ldexpf(s[k], e) * f;
    ops::store_first<4, DT>(r.y, n * r.ldy + m, cols - m, s);
}

void finish(const Result &r, int splits, int64_t rows, int64_t cols, hipStream_t st) {
    Timed tm("product_join", st);
    const dim3 grid = grid_of((rows * (r.ldp / 4) + NT - 1) / NT), block(NT);
    if (r.dt == DT_F32) hipLaunchKernelGGL((finish_kernel<DT_F32>), grid, block, 0, st, r, splits, rows, cols);
    else if (r.dt == DT_BF16) hipLaunchKernelGGL((finish_kernel<DT_BF16>), grid, block, 0, st, r, splits, rows, cols);
    else hipLaunchKernelGGL((finish_kernel<DT_F16>), grid, block, 0, st, r, splits, rows, cols);
}

template <class S, bool F16>
static void launch(Args &g, int splits, const Result &r, hipStream_t st) {
    const dim3 grid = tiles_of<S>(g, splits);
    if (g.down) hipLaunchKernelGGL((product_kernel<S, F16, PARTS, true>), grid, dim3(S::NT), 0, st, g, r);
    else if (r.acc) hipLaunchKernelGGL((product_kernel<S, F16, PARTS, false>), grid, dim3(S::NT), 0, st, g, r);
    else if (r.dt == DT_F32) hipLaunchKernelGGL((product_kernel<S, F16, OUT32, false>), grid, dim3(S::NT), 0, st, g, r);
    else hipLaunchKernelGGL((product_kernel<S, F16, OUT16, false>), grid, dim3(S::NT), 0, st, g, r);
}
template <class S>
static void launch(Args &g, bool f16, int splits, const Result &r, hipStream_t st) {
    if (f16) launch<S, true>(g, splits, r, st);
    else launch<S, false>(g, splits, r, st);
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
