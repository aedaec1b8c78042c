// Frozen weights in microscaled 4-bit floating point (MXFP4), and products with them, for gfx950.
//
// A weight [N][K] is cut along K into blocks of 32.  A block's elements are q 2^(s - 127): s its scale, one byte (255: NaN), q
// one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (e2m1), two to a byte, the even one low.  K is filled up to whole blocks with
// zeros.  Quantisation: 2^(s - 127) takes the block's largest magnitude to [4, 8); elements round to the nearest, ties to the
// even code, and end at 6; a block with an infinite or NaN element has scale 255.
//
// Every q 2^(s - 127) is a bf16 number, so products run on bf16 matrix instructions and lose nothing to the weight.  x keeps its
// bits too: one bf16 term for bf16, two for fp16, three for fp32.
//   y = x W^T:  up to 64 tokens read the 4-bit weight itself, which is what bounds them (step_kernel); more get a bf16 copy
//   of the weight in the workspace first (gdn_product.h), 4.25 bits read and 16 written for 2 M products each.  8192 x 2048 bf16:
//   16 tokens 16 us so and 33 with a copy, 32 20 and 32, 64 29 and 30.
//   dx = dy W:  as the latter, with a copy that lies along N.
// 8192 tokens through 2048 -> 8192 bf16, both ways: 418 us, of them 24 for the copies and 390 for the products.  One token: 5.4 us
// of kernel for 8.9 MB, latency.
#include "gdn_common.h"
#include "gdn_host.h"
#include "gdn_product.h"
#include "gdn_terms.h"
#include "../../include/gdn_mi355x.h"

namespace gdn {
namespace mx {

using namespace mm;

constexpr int NT = 256;
constexpr int MOST = 64;                 // tokens that read the 4-bit weight itself
constexpr int WAVES = 8;                 // along K, for these
constexpr int64_t KEPT = 1 << 26;        // elements of the copy at a time
typedef float f4 __attribute__((ext_vector_type(4)));

// i / d, in 32 bits where that does (a division in 64 bits costs more than the rest of a streaming kernel's work on 16 bytes).
__device__ __forceinline__ int64_t divided(int64_t i, uint32_t d) { return i >> 32 ? i / d : (uint32_t)i / d; }

// ------------------------------------------------------------------------------------------------ quantisation

// Four lanes to a block, eight elements to a lane.
template <int DT>
__global__ __launch_bounds__(NT) void quantize_kernel(const void *w, uint32_t *codes, uint8_t *scales, int64_t N, int64_t K,
                                                      int64_t ld, int64_t blocks) {
    const int64_t i = block_index() * NT + threadIdx.x, n = divided(i, (uint32_t)blocks * 4), c = (i - n * blocks * 4) * 8;
    if (n >= N) return;  // whole blocks
    float x[8];
    ops::load_first<8, DT>(w, n * ld + c, K - c, x);
    uint32_t top = 0;  // magnitudes are ordered as their bits, NaN above all
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    // the largest magnitude's biased exponent less 2 (a subnormal one's is 0, and so is the scale's)
    const bool odd = top >= 0x7f800000u;
    const uint32_t e = odd ? 255u : max(top >> 23, 2u) - 2u;
    const float scale = __uint_as_float(e << 23);  // only its exponent counts
    uint32_t out = 0;
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, x[0], x[1], scale, 0);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, x[2], x[3], scale, 1);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, x[4], x[5], scale, 2);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, x[6], x[7], scale, 3);
    codes[i] = odd ? 0u : out;
    if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)e;
}

typedef float f2 __attribute__((ext_vector_type(2)));

// The scale as the conversions take it, and eight codes as bf16 numbers (four pairs).
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(s << 23); }
__device__ __forceinline__ u4 values_of(uint32_t c, float s) {
    return u4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3))};
}

// Eight elements to a thread: rows of K elements.
template <int DT>
__global__ __launch_bounds__(NT) void values_kernel(const uint32_t *codes, const uint8_t *scales, void *out, int64_t N, int64_t K,
                                                    int64_t blocks) {
    const int64_t i = block_index() * NT + threadIdx.x, n = divided(i, (uint32_t)blocks * 4), u = i - n * blocks * 4;
    if (n >= N) return;
    const uint32_t c = codes[i];
    const float s = scale_of(scales[i >> 2]);
    float x[8];
#define GDN_PAIR(j)                                                          \
    {                                                                        \
        const f2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, j);      \
        x[2 * j] = v[0];                                                     \
        x[2 * j + 1] = v[1];                                                 \
    }
    GDN_PAIR(0) GDN_PAIR(1) GDN_PAIR(2) GDN_PAIR(3)
#undef GDN_PAIR
    ops::store_first<8, DT>(out, n * K + u * 8, K - u * 8, x);
}

// The same as an operand: bf16 rows `kp` elements apart, zeros behind the last (a NaN scale reaches no column that is not there).
__global__ __launch_bounds__(NT) void operand_kernel(const uint32_t *codes, const uint8_t *scales, uint16_t *out, int64_t N,
                                                     int64_t K, int64_t blocks, int64_t kp) {
    const int64_t i = block_index() * NT + threadIdx.x, n = divided(i, (uint32_t)(kp / 8)), u = i - n * (kp / 8);
    if (n >= N) return;
    u4 v = u4{0, 0, 0, 0};
    if (u * 8 < K) {
        v = values_of(codes[n * blocks * 4 + u], scale_of(scales[n * blocks + (u >> 2)]));
        if (u * 8 + 8 > K) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (u * 8 + j >= K) v[j / 2] &= j % 2 ? 0xffffu : 0xffff0000u;
        }
    }
    *reinterpret_cast<u4 *>(out + n * kp + u * 8) = v;
}

// The weight's rows [0, N) as bf16 numbers along N: out[k][n], rows np apart, zeros behind the last; 64 x 64 to a workgroup.
__global__ __launch_bounds__(NT) void across_kernel(const uint32_t *codes, const uint8_t *scales, uint16_t *out, int64_t N,
                                                    int64_t K, int64_t blocks, int64_t np, int64_t tiles_k, int64_t tiles) {
    __shared__ uint16_t tile[64][66];
    const int64_t t = block_index();
    if (t >= tiles) return;
    const int64_t n0 = t / tiles_k * 64, u0 = t % tiles_k * 8;  // eight units of eight elements
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int nl = h * 32 + threadIdx.x / 8, ul = threadIdx.x % 8;
        const int64_t n = n0 + nl, u = u0 + ul;
        uint32_t c = 0;
        float s = 1.f;
        if (n < N && u < blocks * 4) {
            c = codes[n * blocks * 4 + u];
            s = scale_of(scales[n * blocks + (u >> 2)]);
        }
        const u4 v = values_of(c, s);
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t *>(&tile[nl][ul * 8 + 2 * j]) = v[j];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int kl = h * 32 + threadIdx.x / 8, nl = threadIdx.x % 8 * 8;
        if (u0 * 8 + kl >= K) continue;
        uint32_t b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = tile[nl + 2 * j][kl] | (uint32_t)tile[nl + 2 * j + 1][kl] << 16;
        *reinterpret_cast<uint4 *>(out + (u0 * 8 + kl) * np + n0 + nl) = make_uint4(b[0], b[1], b[2], b[3]);
    }
}

// ------------------------------------------------------------------------------------------------ few tokens

// The bf16 terms of eight numbers, cut off one after the other (as in gdn_terms.hip).
template <int TERMS>
__device__ __forceinline__ void split(float (&x)[8], u4 (&t)[TERMS]) {
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
        uint32_t b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            b[j] = __float_as_uint(x[j]) >> 16 | (x[j] != x[j] ? 0x40u : 0u);
            const float back = __uint_as_float(b[j] << 16);
            x[j] = fabsf(back) <= 3.4028234e38f ? x[j] - back : 0.f;
        }
        t[k] = u4{b[0] | b[1] << 16, b[2] | b[3] << 16, b[4] | b[5] << 16, b[6] | b[7] << 16};
    }
}

struct StepArgs {
    const void *x;
    const uint4 *codes;
    const uint8_t *scales;
    void *y;
    int64_t ld, N;
    int M, K, blocks, dt;
};

// 16 rows of the weight to a workgroup, its WAVES waves taking groups of four blocks along K in turn.  Lane (r, g) holds block g
// of row r, 32 elements in 16 bytes: four matrix instructions, of which each takes eight elements of every lane's block, the
// order along K being the same for both operands.  x comes through the caches.
template <int DT, int TILES, bool WIDE>
__global__ __launch_bounds__(64 * WAVES) void step_kernel(const StepArgs a) {
    constexpr int TERMS = DT == DT_BF16 ? 1 : DT == DT_F16 ? 2 : 3;
    constexpr int AHEAD = 2;  // groups of blocks whose codes are loaded together
    __shared__ f4 part[WAVES][TILES][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16, n = min(n0 + r, a.N - 1);
    const uint4 *codes = a.codes + n * a.blocks;
    const uint8_t *scales = a.scales + n * a.blocks;
    f4 acc[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) acc[t] = f4{0.f, 0.f, 0.f, 0.f};
    for (int b0 = w * 4; b0 < a.blocks; b0 += AHEAD * WAVES * 4) {
        uint4 c[AHEAD];
        uint32_t e[AHEAD];
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int b = b0 + h * WAVES * 4 + g;
            c[h] = b < a.blocks ? codes[b] : make_uint4(0, 0, 0, 0);
            e[h] = b < a.blocks ? scales[b] : 127;
        }
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int b = b0 + h * WAVES * 4 + g;
            const float s = scale_of(e[h]);
            const uint32_t cw[4] = {c[h].x, c[h].y, c[h].z, c[h].w};
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const bf8 A = __builtin_bit_cast(bf8, values_of(cw[m], s));
                const int k = b * 32 + 8 * m;
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    const int64_t token = min(16 * t + r, a.M - 1);
                    u4 B[TERMS];
                    if constexpr (WIDE) {  // bf16 rows of whole vectors need no conversion
                        typedef u4 any4 __attribute__((aligned(2)));
                        B[0] = u4{0, 0, 0, 0};
                        if (k < a.K) B[0] = *reinterpret_cast<const any4 *>(static_cast<const uint16_t *>(a.x) + token * a.ld + k);
                    } else {
                        float x[8];
                        ops::load_first<8, DT>(a.x, token * a.ld + k, a.K - k, x);
                        split<TERMS>(x, B);
                    }
#pragma unroll
                    for (int q = 0; q < TERMS; ++q)
                        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, __builtin_bit_cast(bf8, B[q]), acc[t], 0, 0, 0);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) part[w][t][lane] = acc[t];
    __syncthreads();
    // lane (token, g) of a part holds rows 4 g to 4 g + 3
    for (int i = threadIdx.x; i < TILES * 256; i += 64 * WAVES) {
        const int row = i & 15, token = i >> 4, t = token >> 4, at = (token & 15) + 16 * (row >> 2);
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) s += part[k][t][at][row & 3];
        if (token < a.M && n0 + row < a.N) store_from_f32(a.y, token * a.N + n0 + row, s, DT);
    }
}

template <int DT, bool WIDE>
static void launch_step(const StepArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)((a.N + 15) / 16)), block(64 * WAVES);
    if (a.M <= 16) hipLaunchKernelGGL((step_kernel<DT, 1, WIDE>), grid, block, 0, st, a);
    else if (a.M <= 32) hipLaunchKernelGGL((step_kernel<DT, 2, WIDE>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((step_kernel<DT, 4, WIDE>), grid, block, 0, st, a);
}

// ------------------------------------------------------------------------------------------------ host

static int64_t blocks_of(int64_t K) { return (K + 31) / 32; }

static int check(int64_t N, int64_t K, int dt) {
    if (N < 0 || K <= 0) return fail(GDN_ERR_INVALID, "N must be >= 0 and K > 0");
    if (dt != GDN_F32 && dt != GDN_BF16 && dt != GDN_F16) return fail(GDN_ERR_INVALID, "unknown dtype code");
    if (N > 1 << 24 || K > 1 << 18) return fail(GDN_ERR_UNSUPPORTED, "more than 2^24 rows or 2^18 columns are not supported");
    return GDN_OK;
}

static int check_weight(const void *codes, const void *scales) {
    if (!codes || !scales) return fail(GDN_ERR_INVALID, "null pointer");
    if (!aligned_to(codes, 16)) return fail(GDN_ERR_INVALID, "the codes must lie on 16 bytes");
    return GDN_OK;
}

// A product of M rows of `in` elements with the weight: out elements a row; the contraction runs over `in`.
struct Sizes {
    int64_t kp, piece, pieces;  // elements of a row in whole blocks; rows of the weight at a time
    int terms;
    Plan plan;
};

static Sizes sizes(int64_t M, int64_t K, int64_t N, int dt, bool back) {
    Sizes s{};
    s.terms = dt == GDN_BF16 ? 1 : dt == GDN_F16 ? 2 : 3;
    int64_t most = KEPT / padded(K) / 256 * 256;
    if (most < 256) most = 256;
    s.pieces = (N + most - 1) / most;
    s.piece = s.pieces > 1 ? most : N;
    s.kp = back ? padded(s.piece) : padded(K);
    s.plan = back ? plan(M, K, s.terms * s.kp / BK, 16) : plan(M, s.piece, s.terms * s.kp / BK, 16);
    return s;
}

static bool direct(const void *p, int64_t ld, int64_t cols, int dt) {
    return dt == GDN_BF16 && cols % BK == 0 && ld % 8 == 0 && aligned_to(p, 16) && pitch_fits(ld * 2);
}

struct Space {
    char *base;
    size_t at = 0;
    char *take(size_t n) {
        char *p = base ? base + at : nullptr;
        at += align_up256(n);
        return p;
    }
};
struct Buffers {
    char *w, *x;
    float *acc;
};
static Buffers place(Space &sp, const Sizes &s, int64_t M, int64_t K, bool back, bool copy) {
    Buffers b{};
    b.w = sp.take((size_t)(back ? K : s.piece) * s.kp * 2);
    if (copy) b.x = sp.take((size_t)M * s.terms * s.kp * 2);
    const bool parts = s.plan.splits > 1 || (back && s.pieces > 1);
    if (parts) b.acc = reinterpret_cast<float *>(sp.take((size_t)s.plan.splits * M * columns_of(back ? K : s.piece) * 4));
    return b;
}

// The operand that the weight's copy meets: rows as they lie, or their terms.
static void operand(Args &g, const Source &x, const Sizes &s, char *copy, bool as_it_lies, hipStream_t st) {
    const int64_t kp = padded(x.cols);
    g.b.rows = x.rows;
    g.kit = (int)(kp / BK);
    g.nseg = s.terms;
    if (as_it_lies) {
        g.b.p = static_cast<const char *>(x.p);
        g.b.ld = x.ld * 2;
    } else {
        terms(x, s.terms, false, nullptr, 0, copy, st);
        g.b.p = copy;
        g.b.ld = s.terms * kp * 2;
        for (int t = 0; t < 3; ++t) g.b.off[t] = t * kp * 2;
    }
}

}  // namespace mx
}  // namespace gdn

using namespace gdn;
using namespace gdn::mx;

extern "C" int gdn_mxfp4_quantize(const void *w, void *codes, void *scales, int64_t N, int64_t K, int64_t w_stride, int dtype,
                                  void *stream) {
    clear_error();
    if (const int rc = check(N, K, dtype)) return rc;
    if (N == 0) return GDN_OK;
    if (!w) return fail(GDN_ERR_INVALID, "null pointer");
    if (const int rc = check_weight(codes, scales)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t blocks = blocks_of(K);
    const dim3 grid = grid_of((N * blocks * 4 + NT - 1) / NT);
    {
        Timed tm("mxfp4_quantize", st);
        uint32_t *c = static_cast<uint32_t *>(codes);
        uint8_t *s = static_cast<uint8_t *>(scales);
#define GDN_QUANTIZE(DT) hipLaunchKernelGGL((quantize_kernel<DT>), grid, dim3(NT), 0, st, w, c, s, N, K, w_stride, blocks)
        if (dtype == GDN_F32) GDN_QUANTIZE(DT_F32);
        else if (dtype == GDN_BF16) GDN_QUANTIZE(DT_BF16);
        else GDN_QUANTIZE(DT_F16);
#undef GDN_QUANTIZE
    }
    return check_launch(st, "gdn_mxfp4_quantize");
}

extern "C" int gdn_mxfp4_dequantize(const void *codes, const void *scales, void *out, int64_t N, int64_t K, int dtype,
                                    void *stream) {
    clear_error();
    if (const int rc = check(N, K, dtype)) return rc;
    if (N == 0) return GDN_OK;
    if (!out) return fail(GDN_ERR_INVALID, "null pointer");
    if (const int rc = check_weight(codes, scales)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t blocks = blocks_of(K);
    {
        Timed tm("mxfp4_values", st);
#define GDN_VALUES(DT)                                                                                              \
    hipLaunchKernelGGL((values_kernel<DT>), grid_of((N * blocks * 4 + NT - 1) / NT), dim3(NT), 0, st,         \
                       static_cast<const uint32_t *>(codes), static_cast<const uint8_t *>(scales), out, N, K, blocks)
        if (dtype == GDN_F32) GDN_VALUES(DT_F32);
        else if (dtype == GDN_BF16) GDN_VALUES(DT_BF16);
        else GDN_VALUES(DT_F16);
#undef GDN_VALUES
    }
    return check_launch(st, "gdn_mxfp4_dequantize");
}

extern "C" size_t gdn_mxfp4_linear_workspace_bytes(int64_t M, int64_t K, int64_t N, int dtype, int aligned, int backward) {
    if (M <= 0 || K <= 0 || N <= 0 || M > 1 << 24 || N > 1 << 24 || K > 1 << 18) return 0;
    if (!backward && M <= MOST) return 0;
    const bool copy = !aligned || dtype != GDN_BF16 || (backward ? N : K) % BK;
    Space sp{nullptr};
    place(sp, sizes(M, K, N, dtype, backward), M, K, backward, copy);
    return sp.at;
}

static int check_linear(int64_t M, int64_t K, int64_t N, int64_t ld, int64_t cols, int dt) {
    if (M < 0 || N <= 0) return fail(GDN_ERR_INVALID, "M must be >= 0, N and K > 0");
    if (const int rc = check(N, K, dt)) return rc;
    if (M > 1 << 24) return fail(GDN_ERR_UNSUPPORTED, "more than 2^24 tokens are not supported");
    if (M > 1 && ld < cols) return fail(GDN_ERR_INVALID, "rows overlap");
    return GDN_OK;
}

extern "C" int gdn_mxfp4_linear(const void *x, const void *codes, const void *scales, void *y, void *workspace,
                                size_t workspace_bytes, int64_t M, int64_t K, int64_t N, int64_t x_stride, int dtype,
                                void *stream) {
    clear_error();
    if (const int rc = check_linear(M, K, N, x_stride, K, dtype)) return rc;
    if (M == 0) return GDN_OK;
    if (!x || !y) return fail(GDN_ERR_INVALID, "null pointer");
    if (const int rc = check_weight(codes, scales)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t blocks = blocks_of(K);
    if (M <= MOST) {
        const StepArgs a{x, static_cast<const uint4 *>(codes), static_cast<const uint8_t *>(scales), y, x_stride, N, (int)M, (int)K,
                         (int)blocks, dtype};
        Timed tm("mxfp4_step", st);
        if (dtype == GDN_F32) launch_step<DT_F32, false>(a, st);
        else if (dtype == GDN_F16) launch_step<DT_F16, false>(a, st);
        else if (K % 8 == 0) launch_step<DT_BF16, true>(a, st);
        else launch_step<DT_BF16, false>(a, st);
    } else {
        const Sizes s = sizes(M, K, N, dtype, false);
        const bool as_it_lies = direct(x, x_stride, K, dtype);
        Space need{nullptr}, sp{static_cast<char *>(workspace)};
        place(need, s, M, K, false, !as_it_lies);
        if (!workspace || workspace_bytes < need.at)
            return fail(GDN_ERR_WORKSPACE, "the workspace holds %zu bytes, %zu are needed", workspace_bytes, need.at);
        const Buffers b = place(sp, s, M, K, false, !as_it_lies);
        Args g{};
        operand(g, Source{x, dtype, M, K, x_stride, nullptr, 0, nullptr, nullptr}, s, b.x, as_it_lies, st);
        const int elem = dtype == GDN_F32 ? 4 : 2;
        for (int64_t n0 = 0; n0 < N; n0 += s.piece) {
            const int64_t rows = N - n0 < s.piece ? N - n0 : s.piece;
            {
                Timed tm("mxfp4_values", st);
                hipLaunchKernelGGL(operand_kernel, grid_of((rows * (s.kp / 8) + NT - 1) / NT), dim3(NT), 0, st,
                                   static_cast<const uint32_t *>(codes) + n0 * blocks * 4,
                                   static_cast<const uint8_t *>(scales) + n0 * blocks, reinterpret_cast<uint16_t *>(b.w), rows, K, blocks,
                                   s.kp);
            }
            g.a = Operand{b.w, s.kp * 2, rows, {0, 0, 0}, 0};
            const Result r{static_cast<char *>(y) + n0 * elem, N, dtype, nullptr, nullptr, 0, {0, 0}, b.acc, columns_of(rows), 0,
                           nullptr, nullptr};
            multiply(g, false, s.plan, r, st);
            if (r.acc) finish(r, s.plan.splits, M, rows, st);
        }
    }
    return check_launch(st, "gdn_mxfp4_linear");
}

extern "C" int gdn_mxfp4_linear_bwd(const void *dy, const void *codes, const void *scales, void *dx, void *workspace,
                                    size_t workspace_bytes, int64_t M, int64_t K, int64_t N, int64_t dy_stride, int dtype,
                                    void *stream) {
    clear_error();
    if (const int rc = check_linear(M, K, N, dy_stride, N, dtype)) return rc;
    if (M == 0) return GDN_OK;
    if (!dy || !dx) return fail(GDN_ERR_INVALID, "null pointer");
    if (const int rc = check_weight(codes, scales)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t blocks = blocks_of(K);
    const Sizes s = sizes(M, K, N, dtype, true);
    const bool as_it_lies = direct(dy, dy_stride, N, dtype);
    Space need{nullptr}, sp{static_cast<char *>(workspace)};
    place(need, s, M, K, true, !as_it_lies);
    if (!workspace || workspace_bytes < need.at)
        return fail(GDN_ERR_WORKSPACE, "the workspace holds %zu bytes, %zu are needed", workspace_bytes, need.at);
    const Buffers b = place(sp, s, M, K, true, !as_it_lies);
    const int elem = dtype == GDN_F32 ? 4 : 2;
    for (int64_t n0 = 0; n0 < N; n0 += s.piece) {
        const int64_t rows = N - n0 < s.piece ? N - n0 : s.piece, np = padded(rows), tiles_k = (K + 63) / 64;
        const int64_t tiles = np / 64 * tiles_k;
        Args g{};
        const Source part{static_cast<const char *>(dy) + n0 * elem, dtype, M, rows, dy_stride, nullptr, 0, nullptr, nullptr};
        operand(g, part, s, b.x, as_it_lies, st);
        {
            Timed tm("mxfp4_across", st);
            hipLaunchKernelGGL(across_kernel, grid_of(tiles), dim3(NT), 0, st, static_cast<const uint32_t *>(codes) + n0 * blocks * 4,
                               static_cast<const uint8_t *>(scales) + n0 * blocks, reinterpret_cast<uint16_t *>(b.w), rows, K,
                               blocks, np, tiles_k, tiles);
        }
        g.a = Operand{b.w, np * 2, K, {0, 0, 0}, 0};
        const Result r{dx, K, dtype, nullptr, nullptr, 0, {0, 0}, b.acc, columns_of(K), n0 > 0, nullptr, nullptr};
        multiply(g, false, s.plan, r, st);
        if (r.acc && n0 + rows == N) finish(r, s.plan.splits, M, K, st);
    }
    return check_launch(st, "gdn_mxfp4_linear_bwd");
}
