// Matrix products with plain results, and the join of a split contraction's parts, for gfx950.
#include "gdn_product.h"

namespace gdn {
namespace mm {

enum : int { OUT16 = 0, OUT32 = 1, PARTS = 2 };

template <class S, bool F16, int KIND, int DOWN>
__global__ __launch_bounds__(S::NT, S::WAVES_EU) void product_kernel(const Args g, const Result r) {
    __shared__ __attribute__((aligned(16))) char lds[S::LDS + S::STORE];
    const int w = wave_index(), wm = w / S::WN, wn = w % S::WN;
    char *st = lds + S::LDS + w * 4096;
    const Extent ext = extent_of<S>(g);
    const int z = part_of(g).z;
    products<S, F16, DOWN>(g, ext, lds, [&](int tm, int tn, acc_t(&acc)[S::TM][S::TN]) {
        const int lane = lane_here();
        const int64_t m0 = (int64_t)tm * S::BM + wm * (S::BM / S::WM), n0 = (int64_t)tn * S::BN + wn * (S::BN / S::WN);
        const int e = KIND == PARTS ? 0 : exponent_of(r);
        const float by = KIND != PARTS && r.by ? r.by[0] : 1.f;
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
            const auto scaled = [&](float x, int jj) { return f[jj] == 0.f ? 0.f : ldexpf(x, e) * (f[jj] * by); };
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
                        char *to = reinterpret_cast<char *>(r.acc + ((int64_t)z * g.b.rows + n) * r.ldp + m);
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
    for (int k = 0; k < 4; ++k) s[k] = f == 0.f ? 0.f : ldexpf(s[k], e) * (r.by ? f * r.by[0] : f);
    ops::store_first<4, DT>(r.y, n * r.ldy + m, cols - m, s);
}

void finish(const Result &r, int splits, int64_t rows, int64_t cols, hipStream_t st) {
    Timed tm("product_join", st);
    const dim3 grid = grid_of((rows * (r.ldp / 4) + NT - 1) / NT), block(NT);
    if (r.dt == DT_F32) hipLaunchKernelGGL((finish_kernel<DT_F32>), grid, block, 0, st, r, splits, rows, cols);
    else if (r.dt == DT_BF16) hipLaunchKernelGGL((finish_kernel<DT_BF16>), grid, block, 0, st, r, splits, rows, cols);
    else hipLaunchKernelGGL((finish_kernel<DT_F16>), grid, block, 0, st, r, splits, rows, cols);
}

template <class S, bool F16, int DOWN>
static void launch(Args &g, int splits, const Result &r, hipStream_t st) {
    const dim3 grid = tiles_of<S>(g, splits);
    if (r.acc) hipLaunchKernelGGL((product_kernel<S, F16, PARTS, DOWN>), grid, dim3(S::NT), 0, st, g, r);
    else if constexpr (DOWN != DOWN_A) {  // always in parts
        if (r.dt == DT_F32) hipLaunchKernelGGL((product_kernel<S, F16, OUT32, DOWN>), grid, dim3(S::NT), 0, st, g, r);
        else hipLaunchKernelGGL((product_kernel<S, F16, OUT16, DOWN>), grid, dim3(S::NT), 0, st, g, r);
    }
}
template <class S>
static void launch(Args &g, bool f16, int splits, const Result &r, hipStream_t st) {
    if (g.across == DOWN_A) {
        if (f16) launch<S, true, DOWN_A>(g, splits, r, st);
        else launch<S, false, DOWN_A>(g, splits, r, st);
        return;
    }
    if constexpr (S::BN >= 128) {
        if (g.across == DOWN_B) {
            if (f16) launch<S, true, DOWN_B>(g, splits, r, st);
            else launch<S, false, DOWN_B>(g, splits, r, st);
            return;
        }
    }
    launch<S, false, 0>(g, splits, r, st);  // fp16 terms along the contraction only meet epilogues of their own
}

void multiply(Args g, bool f16, const Plan &p, const Result &r, hipStream_t st) {
    Timed tm("product", st);
    if (p.shape == BIG) launch<Big>(g, f16, p.splits, r, st);
    else if (p.shape == MID) launch<Mid>(g, f16, p.splits, r, st);
    else if (p.shape == FEW) launch<Few>(g, f16, p.splits, r, st);
    else launch<One>(g, f16, p.splits, r, st);
}

// Few rows: narrow tiles, several to a compute unit, whose loads hide one another's latency, and enough parts of the contraction
// to fill the card.  Else the tile and the split that take least by a count of rounds over the 256 compute units.  A block of BK
// takes a 256 x 256 tile 1.5 us (1.45 PFLOP/s in all), a 128 x 128 tile 1.0 us with another beside it on the compute unit and 0.6
// without; a tile's first loads and results as much as five and four blocks; parts of a split contraction are written and read
// back at 4.5 TB/s.
Plan plan(int64_t rows, int64_t cols, int64_t blocks, int max_splits, bool large) {
    const auto tiles = [&](int64_t bm, int64_t bn) { return ((cols + bm - 1) / bm) * ((rows + bn - 1) / bn); };
    const auto most = [&](int64_t least) {  // parts of at least this many blocks
        const int64_t s = blocks / least;
        return (int)(s < 1 ? 1 : s > max_splits ? max_splits : s);
    };
    if (rows <= 64 && !large) {
        const int64_t t = rows <= 32 ? tiles(128, 32) : tiles(128, 64), want = rows <= 32 ? 1024 : 768;
        const int64_t s = want / t < most(8) ? want / t : most(8);
        return {rows <= 32 ? ONE : FEW, (int)(s < 1 ? 1 : s)};
    }
    Plan best{MID, 1};
    double least = 1e30;
    for (int s = 1; s <= most(4); ++s) {
        const double n = (double)((blocks + s - 1) / s), join = s > 1 ? 8e-6 * s * rows * cols / 4.5 + 5. : 0.;
        const int64_t big = tiles(256, 256) * s, mid = tiles(128, 128) * s;
        const double tb = (double)((big + 255) / 256) * (n + 5.) * 1.5 + join;
        const int64_t rest = mid % 512;
        const double tm = ((double)(mid / 512) + (rest > 256 ? 1. : rest > 0 ? 0.6 : 0.)) * (n + 4.) + join;
        if (tb < least) { least = tb; best = {BIG, s}; }
        if (tm < least) { least = tm; best = {MID, s}; }
    }
    return best;
}

}  // namespace mm
}  // namespace gdn
