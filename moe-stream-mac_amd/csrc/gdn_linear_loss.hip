// Cross entropy of the logits z = x W^T without keeping them, and its gradients, for gfx950.
//
// For token i and word v, z_iv = <x_i, W_v>, M_i = max_v z_iv, s_i = sum_v e^{z_iv - M_i}, target t_i:
//   loss_i = log s_i + M_i - z_{i,t_i},    p_iv = e^{z_iv - M_i} / s_i,
//   dx_i = d_i sum_v (p_iv - [v = t_i]) W_v,    dW_v = sum_i d_i (p_iv - [v = t_i]) x_i
// for the cotangents d_i of the losses.
//
// Forward: one product whose tiles of logits end in registers, each as the maximum and the sum of exponentials of its words per
// token; a second kernel joins them.  Backward: the words in pieces; of each piece the logits again (their normaliser is known
// only after the last word), from them the differences p - [v = t] as 16-bit terms, then two more products, which read them
// along the words for dx, with the weight's rows across, and across for dW.  What is stored at any time is one piece of
// differences: 2^26 of them, or those of 256 words.
//
// Words lie along registers and tokens along lanes, so that maxima and sums run within a lane.
//
// Tokens that do not count (prompts, padding) are left out: from COMPACT tokens on, the others' hidden states are gathered into
// the workspace, in their order, and every product forms the tiles of these alone.  How many there are only the device knows, so
// launches are for all of them and workgroups without a token end at once.  Fewer tokens are taken as they lie: bf16, 2048
// tokens of 2048 channels, 32000 words and both gradients take 1372 us as they lie and 1380 gathered if all count, 1345 and 1237
// if a fifth does not; 1024 take 804 and 811, 784 and 739; fp32, 2048 tokens 2968 and 2977, 2883 and 2716, 1024 1703 and 1707,
// 1663 and 1600.
//
// Precision.  bf16 differences are two bf16 terms, each off by half a step of what it rounds: 2^-16 of a difference of any size,
// so that gradients lose nothing but their own rounding; x and W are their own operands.  (In one fp16 term, 11 bits that end at
// 2^-40, training took 2960 us instead of 4280, gradients were 1.2e-3 of the whole away from those of 32-bit sums instead of
// 1.5e-4, and the rows of dW of words that no token expects were coarse or zero.)  fp16: two fp16 terms of a difference times
// 2^15, 2^-22 of it or 2^-40; what that leaves out is below fp16 results, which end at 2^-25, unless cotangents times x pass
// 2^15.  x is an fp16 number times a power of two there for dW (gdn_terms.hip).  Of a token's cotangent the differences carry a
// factor of 0.75 to 1.5 and its sum for dx, or its x for dW, the power of two that is left, so that it costs no rounding of its
// own.  fp32 operands are two fp16 terms under a power of two (2^-22 of a number, or 2^-39 of the largest under it), and every
// product three pairs of them; for the logits each token has a power of its own, so that no token costs another its bits; a
// difference's second term is stored times 2^11, so that small probabilities keep their bits (2^-22 of them down to 2^-29, 2^-51
// below).  Up to WIDE fp32 tokens, forward and backward: three bf16 terms, which hold a number of any magnitude as it is, and
// six pairs; those left out are below 2^-21 of the factors.
//
// Of few tokens (up to ROWS, 16-bit inputs) the differences' terms are rows of one operand for dx, so that the weight, which
// lies along the channels, is read once.  2048 x 32000 bf16, forward and dx: 8 tokens 109 us so, 118 with terms side by side; 64
// 115 and 123; 100 145 and 158; 256 180 and 174; 511 273 and 267.
//
// Measured, bf16, 8192 tokens of which a fifth does not count, 2048 x 32000, both gradients: 634 us for the statistics (1.35
// PFLOP/s), then four pieces with 241 for the differences, 349 for dx and 300 for dW (1.26 and 1.47 PFLOP/s over both terms); on
// another card 686, 247, 381 and 323.  The matrix units are busy 66, 42, 55 and 70 % of the time.  Results and exponentials of a
// tile do not run beside another's products, which is what is lost most.
#include "gdn_common.h"
#include "gdn_host.h"
#include "gdn_product.h"
#include "gdn_terms.h"
#include "../../include/gdn_mi355x.h"

namespace gdn {
namespace ll {

using namespace mm;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int NT = 256;
constexpr int64_t COMPACT = 2048;
constexpr int64_t ROWS = 128;
// dx of fewer tokens is formed in up to 32 parts of the words, of others in 16: bf16 with dx, 32000 words of 256 channels, 64
// tokens 65 us and 75, 256 85 and 98, 511 104 and 114; fp32, 513 tokens, 50001 words of 1001 channels, both gradients, 1224 and 1075.
constexpr int64_t FEW_TOKENS = 512;
constexpr int64_t KEPT = 1 << 26;  // differences of a piece, if that is 256 words or more; statistics of the parts of the words
constexpr int64_t MOST_TOKENS = 1 << 20;  // three slots of 16 bits for each are a row pitch that a product takes
constexpr int WIDE = 128;          // up to here fp32 numbers are three bf16 terms, and a forward call reads the words as they lie
constexpr int SHIFT = 15;          // fp16 differences are stored times 2^15
constexpr int TOP = 14;            // largest magnitudes of scaled operands: [2^14, 2^15)

enum : int { E_X = 0, E_W = 1 };

// ------------------------------------------------------------------------------------------------ tokens that count

struct Tokens {      // of COMPACT tokens and more
    int *count;      // how many count
    int *index;      // [N] their places
    int *place;      // [N] a token's place among them, -1 for one that does not count
    int64_t *target; // [N] their targets
};

// One workgroup; the order of the tokens is kept.  Tokens that do not count have loss 0.
__global__ __launch_bounds__(1024) void tokens_kernel(const int64_t *targets, int64_t N, int64_t ignore, Tokens t, float *loss) {
    constexpr int ROUNDS = 8, STEP = ROUNDS * 1024;  // tokens whose loads are under way together
    __shared__ int sums[2][16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int before = 0;  // tokens that count before this step's
    for (int64_t s0 = 0; s0 < N; s0 += STEP) {
        const int64_t n0 = s0 + w * (ROUNDS * 64) + lane;
        int64_t v[ROUNDS];
        int own = 0, total = 0;
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) v[i] = n0 + i * 64 < N ? targets[n0 + i * 64] : ignore;
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) own += __popcll(__ballot(v[i] != ignore));
        int *sum = sums[s0 / STEP & 1];  // two: a wave may be a step ahead of another
        if (lane == 0) sum[w] = own;
        __syncthreads();
        int c = before;
        for (int i = 0; i < 16; ++i) {
            if (i < w) c += sum[i];
            total += sum[i];
        }
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
            const int64_t n = n0 + i * 64;
            const bool live = v[i] != ignore;
            const uint64_t all = __ballot(live);
            const int at = c + __popcll(all & ((1ull << lane) - 1));
            if (n < N) t.place[n] = live ? at : -1;
            if (live) {
                t.index[at] = (int)n;
                t.target[at] = v[i];
            } else if (loss && n < N) {
                loss[n] = 0.f;
            }
            c += __popcll(all);
        }
        before += total;
    }
    if (threadIdx.x == 0) *t.count = before;
}

// ------------------------------------------------------------------------------------------------ forward

struct StatArgs {
    const int64_t *targets;
    float2 *part;  // [parts][N]: maximum and sum of a part of the words
    float *zt;     // [N] the target's logit
    const int *exps, *each;  // SCALED: the words' exponent is exps[E_W], a token's each[n]
    int64_t N, V, v0;  // word of the operand's first row
    int part0;
};

// The statistics of a wave's words, `rows` - m0 of 16 TM, for its 16 TN tokens from n0 on.
template <int TM, int TN, bool SCALED>
__device__ __forceinline__ void statistics(const StatArgs &a, int64_t rows, int64_t tokens, int64_t m0, int64_t n0, int64_t part,
                                           acc_t (&acc)[TM][TN]) {
    const int lane = lane_here();
    const int words = (int)min((int64_t)(16 * TM), rows - m0);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int64_t n = n0 + 16 * j + (lane & 15);
        const bool live = n < tokens;
        const int e = SCALED && live ? -(a.exps[E_W] + a.each[n]) : 0;
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if constexpr (SCALED) acc[i][j][q] = ldexpf(acc[i][j][q], e);
                if (words < 16 * TM && 16 * i + 4 * (lane >> 4) + q >= words) acc[i][j][q] = -INFINITY;
                mx = fmaxf(mx, acc[i][j][q]);
            }
        mx = fmaxf(mx, lane_xor16(mx));
        mx = fmaxf(mx, lane_xor32(mx));
        const float ref = mx == -INFINITY ? 0.f : mx;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) s += __builtin_amdgcn_exp2f((acc[i][j][q] - ref) * LOG2E);
        s += lane_xor16(s);
        s += lane_xor32(s);
        if (live && lane < 16) a.part[part * a.N + n] = make_float2(mx, s);
        const int64_t t = live ? a.targets[n] - a.v0 - m0 : -1;
        const bool here = t >= 0 && t < words && ((t >> 2 & 3) == (lane >> 4));
        if (__any(here)) {
            const int tl = here ? (int)t - 4 * (lane >> 4) : -1;
            float z = 0.f;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (tl == 16 * i + q) z = acc[i][j][q];
            if (here) a.zt[n] = z;
        }
    }
}

// Waves leave the statistics of their own words.
template <class S, bool F16, bool SCALED>
__global__ __launch_bounds__(S::NT, S::WAVES_EU) void stat_kernel(const Args g, const StatArgs a) {
    __shared__ __attribute__((aligned(16))) char lds[S::LDS];
    const int w = wave_index(), wm = w / S::WN, wn = w % S::WN;
    const Extent ext = extent_of<S>(g);
    products<S, F16>(g, ext, lds, [&](int tm, int tn, acc_t(&acc)[S::TM][S::TN]) {
        const int64_t m0 = (int64_t)tm * S::BM + wm * (S::BM / S::WM), n0 = (int64_t)tn * S::BN + wn * (S::BN / S::WN);
        statistics<S::TM, S::TN, SCALED>(a, g.a.rows, ext.rows_b, m0, n0, a.part0 + tm * S::WM + wm, acc);
    });
}

// Few tokens and fp32 words, forward: read once, as they lie, and split in registers into three bf16 terms, which hold them exactly
// and at any magnitude, so that they need no scale.  Six products of terms; those left out are below 2^-21 of the factors.  The
// tokens' terms, 16 TN rows of three slots, go through LDS, two stages of 64 along the contraction; a wave's 32 words stay its
// own and go to registers, a stage ahead.  64765 x 4096 weights (1.06 GB, 208 us at a copy's rate): 32 tokens 229 to 255 us, 118
// tokens 444 to 489, where the conversions and one wave to a SIMD hold it back; through a copy of the words in terms, as weights
// off 16 bytes take it, 1109 and 1199.  128 tokens, 32000 x 2048: 123 and 363; 129 tokens, by two fp16 terms, 277.
template <int TN>
struct Wide {
    static constexpr int NT = 256, BM = 128, BN = 16 * TN, TM = 2, SLOT = BN * BK * 2, STAGE = 3 * SLOT;
    static constexpr int WAVES_EU = TN > 4 ? 1 : 2;
};
struct WideArgs {
    const float *w;
    int64_t ld, rows;
    Operand x;
    int kit;
};

// The first terms of x, cut off, and in x what they leave: NaN of infinities and NaN.
__device__ __forceinline__ uint4 cut(float (&x)[8]) {
    uint32_t b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        b[k] = __float_as_uint(x[k]);
        x[k] -= __uint_as_float(b[k] & 0xffff0000u);
    }
    uint4 y;
    y.x = b[0] >> 16 | (b[1] & 0xffff0000u);
    y.y = b[2] >> 16 | (b[3] & 0xffff0000u);
    y.z = b[4] >> 16 | (b[5] & 0xffff0000u);
    y.w = b[6] >> 16 | (b[7] & 0xffff0000u);
    return y;
}

template <int TN>
__global__ __launch_bounds__(256, Wide<TN>::WAVES_EU) void wide_kernel(const WideArgs g, const StatArgs a) {
    typedef Wide<TN> S;
    __shared__ __attribute__((aligned(16))) char lds[2 * S::STAGE];
    const int lane = threadIdx.x & 63, w = wave_index();
    const int64_t m0 = (int64_t)blockIdx.x * S::BM + w * 32;
    const float *row[S::TM];
#pragma unroll
    for (int i = 0; i < S::TM; ++i) row[i] = g.w + min(m0 + 16 * i + (lane & 15), g.rows - 1) * g.ld + 8 * (lane >> 4);
    Side<S, S::BN, false> b[3];
#pragma unroll
    for (int t = 0; t < 3; ++t) b[t].start(g.x, g.x.off[t], 0, g.x.rows, 0, 0);
    float4 now[2][S::TM][2], next[2][S::TM][2];
    const auto load = [&](float4(&to)[2][S::TM][2], char *stage) {
#pragma unroll
        for (int t = 0; t < 3; ++t) {
#pragma unroll
            for (int r = 0; r < Side<S, S::BN, false>::LOADS; ++r) b[t].load(stage + t * S::SLOT, r, w);
            b[t].next(g.x);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < S::TM; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) to[s][i][h] = *reinterpret_cast<const float4 *>(row[i] + s * 32 + h * 4);
#pragma unroll
        for (int i = 0; i < S::TM; ++i) row[i] += BK;
    };
    uint32_t at[2];
    places<false, 0>(at, lane, 0, 0);
    acc_t acc[S::TM][TN];
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = acc_t{0.f, 0.f, 0.f, 0.f};
    load(now, lds);
    for (int k = 0; k < g.kit; ++k) {
        const char *stage = lds + (k & 1) * S::STAGE;
        stage_barrier();
        if (k + 1 < g.kit) load(next, lds + (~k & 1) * S::STAGE);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u4 x[S::TM][3];
#pragma unroll
            for (int i = 0; i < S::TM; ++i) {
                const float4 lo = now[s][i][0], hi = now[s][i][1];
                float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int t = 0; t < 3; ++t) x[i][t] = __builtin_bit_cast(u4, cut(v));
            }
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                u4 y[3];
#pragma unroll
                for (int t = 0; t < 3; ++t) y[t] = fragment<false, 0>(stage + t * S::SLOT, at, s, j);
#pragma unroll
                for (int t = 2; t >= 0; --t)  // the smallest first
#pragma unroll
                    for (int i = 0; i < S::TM; ++i)
#pragma unroll
                        for (int c = 0; c <= t; ++c) acc[i][j] = mfma<false>(x[i][c], y[t - c], acc[i][j]);
            }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < S::TM; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) now[s][i][h] = next[s][i][h];
    }
    statistics<S::TM, TN, false>(a, g.rows, g.x.rows, m0, 0, blockIdx.x * 4 + w, acc);
}

// Joins a token's parts: TOKENS tokens to a workgroup, NT / TOKENS threads to a token.
template <int TOKENS>
__global__ __launch_bounds__(NT) void join_kernel(const int64_t *targets, const float2 *part, int parts, const float *zt,
                                                  int64_t N, int64_t V, int64_t ignore, float *loss, float2 *stat,
                                                  const int *index, const int *count, int64_t n0) {
    constexpr int P = NT / TOKENS;
    __shared__ float2 red[P][TOKENS];
    const int tl = threadIdx.x % TOKENS, p0 = threadIdx.x / TOKENS;
    const int64_t n = block_index() * TOKENS + tl;
    const bool any = n < N && (!count || n0 + n < *count);
    float m = -INFINITY, s = 0.f;
    if (any) {
#pragma unroll 8
        for (int p = p0; p < parts; p += P) {
            const float2 o = part[(int64_t)p * N + n];
            const float b = fmaxf(m, o.x), r = b == -INFINITY ? 0.f : b;
            s = s * __builtin_amdgcn_exp2f((m - r) * LOG2E) + o.y * __builtin_amdgcn_exp2f((o.x - r) * LOG2E);
            m = b;
        }
    }
    red[p0][tl] = make_float2(m, s);
    __syncthreads();
#pragma unroll
    for (int h = P / 2; h >= 1; h /= 2) {
        if (p0 < h) {
            const float2 o = red[p0 + h][tl];
            const float b = fmaxf(m, o.x), r = b == -INFINITY ? 0.f : b;
            s = s * __builtin_amdgcn_exp2f((m - r) * LOG2E) + o.y * __builtin_amdgcn_exp2f((o.x - r) * LOG2E);
            m = b;
            red[p0][tl] = make_float2(m, s);
        }
        __syncthreads();
    }
    if (p0 || !any) return;
    const int64_t t = targets[n];
    float l = logf(s) - (zt[n] - m);
    if (t < 0 || t >= V) l = NAN;
    if (t == ignore) l = 0.f;
    loss[index ? index[n] : n] = l;
    if (stat) stat[n] = make_float2(m, 1.f / s);
}

// The losses' sum, or mean over the tokens that count, and what a token's cotangent is multiplied by.
__global__ __launch_bounds__(1024) void total_kernel(const float *loss, const int64_t *targets, int64_t N, int64_t ignore,
                                                     int mean, float *total, float *factor) {
    __shared__ double red[1024];
    __shared__ int64_t count[1024];
    double s = 0.;
    int64_t c = 0;
    for (int64_t i = threadIdx.x; i < N; i += 1024) {
        s += (double)loss[i];
        c += targets[i] != ignore;
    }
    red[threadIdx.x] = s;
    count[threadIdx.x] = c;
    __syncthreads();
    for (int h = 512; h >= 1; h >>= 1) {
        if ((int)threadIdx.x < h) {
            red[threadIdx.x] += red[threadIdx.x + h];
            count[threadIdx.x] += count[threadIdx.x + h];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const double n = mean ? (double)(count[0] > 0 ? count[0] : 1) : 1.;
        total[0] = (float)(red[0] / n);
        factor[0] = (float)(1. / n);
    }
}

// ------------------------------------------------------------------------------------------------ backward

// The token's cotangent, 0 where it does not count and NaN where its target is no word, as power[n] times factor[n], a power of two
// and what is left, of magnitude 0.75 to 1.5 (larger only within a factor of 1.5 of the largest fp32 number): differences times it
// and 2^15 are below 2^16, and the smallest lose half a bit at most to the factor.  part = partial maxima of the powers.
__global__ __launch_bounds__(NT) void cotangent_kernel(const int64_t *targets, const float *dloss, int64_t stride,
                                                       const float *mean, int64_t N, int64_t V, int64_t ignore, float *power,
                                                       float *factor, float *part, const int *index, const int *count) {
    __shared__ float red[NT];
    float m = 0.f;
    if (count) N = *count;
    for (int64_t n = (int64_t)blockIdx.x * NT + threadIdx.x; n < N; n += (int64_t)PARTS * NT) {
        const int64_t t = targets[n];
        float x = dloss[(index ? index[n] : n) * stride];
        if (mean) x *= mean[0];
        if (t < 0 || t >= V) x = NAN;
        if (t == ignore) x = 0.f;
        float p = x, f = 1.f;  // 0, infinities and NaN
        if (x != 0.f && fabsf(x) <= 3.4028234e38f) {
            int e;
            f = frexpf(x, &e);
            if (fabsf(f) < 0.75f || e > 127) {
                f *= 2.f;
                --e;
            }
            p = ldexpf(1.f, e);
            m = fmaxf(m, p);
        }
        power[n] = p;
        factor[n] = f;
    }
    red[threadIdx.x] = m;
    __syncthreads();
    for (int h = NT / 2; h >= 1; h >>= 1) {
        if ((int)threadIdx.x < h) red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + h]);
        __syncthreads();
    }
    if (threadIdx.x == 0) part[blockIdx.x] = red[0];
}

struct DiffArgs {
    const int64_t *targets;
    const float2 *stat;
    const float *power, *factor;  // cotangents
    const int *exps, *each;  // SCALED: the logits' scale
    uint16_t *p;      // kp to a row and term: rows `row` apart, a next term `second` on
    int64_t v0, kp, row, second;
};

// x as it was rounded: the compiler may round a product or sum to 16 bits at once in one place and in two steps in another, and
// terms that are taken in two places have to belong to the same number.
__device__ __forceinline__ float as_rounded(float x) {
    asm volatile("" : "+v"(x));
    return x;
}

// What a term leaves of x: the next term, times 2^LOW where it is stored so.
template <bool F16, bool SCALED>
__device__ __forceinline__ float left_of(float x) {
    if constexpr (F16) return (x - __half2float(__float2half(x))) * (SCALED ? (float)(1 << LOW) : 1.f);
    return x - bf16_to_f32(f32_to_bf16_cvt(x));
}

// The differences of a piece of words, factor (p - [v = t]), fp16 ones times 2^SHIFT, in TERMS terms; zeros for tokens that do not
// count.  SCALED: the logits have a scale, and second terms are stored times 2^LOW.
template <class S, bool F16, bool SCALED, int TERMS>
__global__ __launch_bounds__(S::NT, S::WAVES_EU) void diff_kernel(const Args g, const DiffArgs a) {
    constexpr int DT = F16 ? DT_F16 : DT_BF16;
    __shared__ __attribute__((aligned(16))) char lds[S::LDS + S::STORE];
    const int w = wave_index(), wm = w / S::WN, wn = w % S::WN;
    char *store = lds + S::LDS + w * 4096;
    const Extent ext = extent_of<S>(g);
    products<S, F16>(g, ext, lds, [&](int tm, int tn, acc_t(&acc)[S::TM][S::TN]) {
        const int lane = lane_here();
        const int64_t m0 = (int64_t)tm * S::BM + wm * (S::BM / S::WM), n0 = (int64_t)tn * S::BN + wn * (S::BN / S::WN);
        const int words = (int)min((int64_t)(S::BM / S::WM), g.a.rows - m0);  // of this wave's; may be negative
#pragma unroll
        for (int j = 0; j < S::TN; ++j) {
            const int64_t n = n0 + 16 * j + (lane & 15);
            const bool in = n < ext.rows_b;
            const int e = SCALED && in ? -(a.exps[E_W] + a.each[n]) : 0;
            const float2 st = in ? a.stat[n] : make_float2(0.f, 0.f);
            const bool live = in && a.power[n] != 0.f;
            const float scale = live ? a.factor[n] * (F16 ? (float)(1 << SHIFT) : 1.f) : 0.f, inv = st.y * scale;
            const int64_t hot = live ? a.targets[n] - a.v0 - m0 - 4 * (lane >> 4) : -1;
#pragma unroll
            for (int i = 0; i < S::TM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float z = acc[i][j][q];
                    if constexpr (SCALED) z = ldexpf(z, e);
                    acc[i][j][q] = __builtin_amdgcn_exp2f((z - st.x) * LOG2E) * inv;
                }
            if (__any(hot >= 0 && hot < S::BM / S::WM)) {  // rare: a wave has 64 or 128 words
                const int at = hot >= 0 && hot < S::BM / S::WM ? (int)hot : -1;
#pragma unroll
                for (int i = 0; i < S::TM; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (at == 16 * i + q) acc[i][j][q] -= scale;
            }
#pragma unroll
            for (int i = 0; i < S::TM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[i][j][q] = as_rounded(acc[i][j][q]);
            if (words < S::BM / S::WM || !__all(live)) {
                const int left = live ? words - 4 * (lane >> 4) : 0;
#pragma unroll
                for (int i = 0; i < S::TM; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (16 * i + q >= left) acc[i][j][q] = 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < S::TN; j += 2) {
            const int64_t n = n0 + 16 * j, rows = ext.rows_b - n;
            if (rows <= 0) break;
#pragma unroll
            for (int i = 0; i < S::TM; i += 4) {
                const int64_t m = m0 + 16 * i;
                if (m >= a.kp) break;
#pragma unroll 1
                for (int t = 0; t < TERMS; ++t) {
#pragma unroll
                    for (int ii = 0; ii < 4; ++ii)
#pragma unroll
                        for (int jj = 0; jj < 2; ++jj) {
                            float y[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                y[k] = acc[i + ii][j + jj][k];
                                if (t > 0) y[k] = left_of<F16, SCALED>(y[k]);
                                if (TERMS > 2 && t > 1) y[k] = left_of<F16, SCALED>(y[k]);
                            }
                            put16(lane, store, ii, jj, ops::pack2_cvt(y[0], y[1], DT), ops::pack2_cvt(y[2], y[3], DT));
                        }
                    uint16_t *to = a.p + n * a.row + t * a.second + m;
                    store_rows(lane, store, reinterpret_cast<char *>(to), (uint32_t)(a.row * 2), rows, (a.kp - m) * 2, 2);
                }
            }
        }
    });
}

// ------------------------------------------------------------------------------------------------ host

struct Sizes {
    int64_t N, H, V, hp, np, piece, pieces;  // hp, np: H and N in whole blocks; piece: words at a time
    bool f16, scaled;  // terms are fp16; and of operands times a power of two
    int terms;         // of an operand
    bool compact;
    int wslots;    // terms of the weight's rows
    bool rows;     // the differences' two terms are rows of one operand, else side by side
    int64_t prows; // rows of the differences
    int pterms;    // their terms side by side
    int slots;     // terms of the operands that meet them, as they are laid out: the weight for dx, x for dW
    int pairs;     // of terms, in these products
    int64_t parts, tokens;  // parts of the words with statistics of their own; tokens at a time in the forward pass
    Plan px, pw;
};

// The segments of a product over kp elements: a's terms `first` elements apart, b's `second`.
//   one term of a, two of b:  both pairs
//   two terms (fp16):         all pairs but that of the second ones.  a has three slots in the backward pass, as terms() makes
//                             them; the third meets b's second term, stored times 2^LOW
//   three terms (bf16):       all pairs but those below 2^-16 of the first, the smallest first
static void segments(Args &g, const Sizes &s, bool back, int64_t kp, int64_t first, int64_t second) {
    const auto pair = [&](int i, int j) {
        g.a.off[g.nseg] = i * first * 2;
        g.b.off[g.nseg++] = j * second * 2;
    };
    g.kit = (int)(kp / BK);
    g.nseg = 0;
    if (s.terms == 3)
        for (int i = 2; i >= 0; --i)
            for (int k = i; k >= 0; --k) pair(k, i - k);
    else {
        pair(0, 0);
        if (s.terms == 2) pair(1, 0);
        if (s.terms == 2 || back) pair(back && s.terms == 2 ? 2 : 0, 1);
    }
}

static bool direct(const void *p, int64_t ld, int64_t H, int dt) {
    return dt != GDN_F32 && H % BK == 0 && ld % 8 == 0 && aligned_to(p, 16) && pitch_fits(ld * 2);
}

// The same however the operands lie: what they ask for is room for copies, no more.
static Sizes sizes(int64_t N, int64_t H, int64_t V, int dt, bool dx) {
    Sizes s{};
    s.N = N; s.H = H; s.V = V;
    s.hp = padded(H);
    s.np = padded(N);
    const bool any = dt == GDN_F32 && N <= WIDE;  // three bf16 terms hold numbers of any magnitude
    s.terms = any ? 3 : dt == GDN_F32 ? 2 : 1;
    s.scaled = s.terms == 2;
    s.f16 = s.scaled || dt == GDN_F16;
    s.compact = N >= COMPACT;
    s.rows = N <= ROWS && dx && s.terms == 1;
    s.prows = s.rows ? 2 * N : N;
    s.pterms = s.rows ? 1 : any ? 3 : 2;
    s.slots = s.terms == 1 ? 1 : 3;
    s.pairs = any ? 6 : s.scaled ? 3 : 2;
    s.wslots = s.terms > 1 && dx ? s.slots : s.terms;
    int64_t most = KEPT / s.np / 256 * 256;
    if (most < 256) most = 256;
    s.pieces = (V + most - 1) / most;
    s.piece = ((V + s.pieces - 1) / s.pieces + 255) / 256 * 256;
    s.pieces = (V + s.piece - 1) / s.piece;
    s.parts = 2 * s.pieces * ((s.piece + 127) / 128);  // two waves to 128 words at most
    s.tokens = KEPT / s.parts / 256 * 256;
    if (s.tokens < 256) s.tokens = 256;
    if (s.tokens > N) s.tokens = N;
    const int64_t words = s.piece < V ? s.piece : V;
    s.px = plan(s.prows, H, (s.rows ? 1 : s.pairs) * padded(words) / BK, N < FEW_TOKENS ? 32 : 16);
    s.pw = plan(words, H, s.pairs * s.np / BK, 8, true);
    return s;
}

// Whether the weight is read as fp32 numbers: few tokens, rows of whole blocks, 16 bytes aligned.
static bool wide(const void *p, int64_t ld, int64_t N, int64_t H, int dt) {
    return dt == GDN_F32 && N <= WIDE && H % BK == 0 && ld % 4 == 0 && aligned_to(p, 16);
}

struct Space {
    char *base;
    size_t at = 0;
    template <class T>
    T *take(int64_t n) {
        T *p = base ? reinterpret_cast<T *>(base + at) : nullptr;
        at += align_up256((size_t)n * sizeof(T));
        return p;
    }
};

struct Buffers {
    uint16_t *x, *w, *xt, *p;
    float *part, *zt, *power, *factor, *most, *acc_x, *acc_w;
    float2 *stats;
    int *exps, *each;
    Tokens tokens;
};

static Buffers place(Space &sp, const Sizes &s, bool dx, bool dw, bool bwd, bool copy_x, bool copy_w) {
    Buffers b{};
    const int t = s.terms;
    const int64_t words = s.piece < s.V ? s.piece : s.V;
    b.exps = sp.take<int>(2);
    b.most = sp.take<float>(1);
    b.part = sp.take<float>(3 * PARTS);
    if (s.compact) {
        b.tokens.count = sp.take<int>(1);
        b.tokens.index = sp.take<int>(s.N);
        b.tokens.place = sp.take<int>(s.N);
        b.tokens.target = sp.take<int64_t>(s.N);
    }
    if (s.scaled) b.each = sp.take<int>(s.N);
    if (copy_x || s.compact) b.x = sp.take<uint16_t>(s.N * t * s.hp);
    if (copy_w) b.w = sp.take<uint16_t>(words * s.wslots * s.hp);
    if (!bwd) {
        b.stats = sp.take<float2>(s.parts * s.tokens);
        b.zt = sp.take<float>(s.tokens);
        return b;
    }
    b.power = sp.take<float>(s.N);
    b.factor = sp.take<float>(s.N);
    b.p = sp.take<uint16_t>(s.prows * s.pterms * padded(words));
    if (dx) b.acc_x = sp.take<float>((int64_t)s.px.splits * s.prows * columns_of(s.H));
    if (dw) {
        b.xt = sp.take<uint16_t>(s.H * s.slots * s.np);
        if (s.pw.splits > 1) b.acc_w = sp.take<float>((int64_t)s.pw.splits * words * columns_of(s.H));
    }
    return b;
}

static Buffers place_wide(Space &sp, const Sizes &s) {
    Buffers b{};
    b.x = sp.take<uint16_t>(s.N * 3 * s.hp);
    b.stats = sp.take<float2>((s.V + 127) / 128 * 4 * s.N);
    b.zt = sp.take<float>(s.N);
    return b;
}

static int check(int64_t N, int64_t H, int64_t V, int64_t x_ld, int64_t w_ld, int dt) {
    if (N < 0 || H <= 0 || V <= 0) return fail(GDN_ERR_INVALID, "N must be >= 0, H and V > 0");
    if (dt != GDN_F32 && dt != GDN_BF16 && dt != GDN_F16) return fail(GDN_ERR_INVALID, "unknown dtype code");
    if (N > MOST_TOKENS || V > 1 << 24 || H > 1 << 17)
        return fail(GDN_ERR_UNSUPPORTED, "more than 2^20 tokens, 2^24 words or 2^17 channels are not supported");
    if ((N > 1 && x_ld < H) || (V > 1 && w_ld < H)) return fail(GDN_ERR_INVALID, "rows overlap");
    return GDN_OK;
}

template <class S>
static void launch_stat(Args &g, const StatArgs &a, const Sizes &s, hipStream_t st) {
    const dim3 grid = tiles_of<S>(g, 1), block(S::NT);
    if (s.scaled) hipLaunchKernelGGL((stat_kernel<S, true, true>), grid, block, 0, st, g, a);
    else if (s.f16) hipLaunchKernelGGL((stat_kernel<S, true, false>), grid, block, 0, st, g, a);
    else hipLaunchKernelGGL((stat_kernel<S, false, false>), grid, block, 0, st, g, a);
}
// Scaled operands come with more than 128 tokens, three terms with no more: plan() never gives those the narrow tiles, nor these the
// large one (128 tokens need no fewer rounds of it).
template <class S>
static void launch_diff(Args &g, const DiffArgs &a, const Sizes &s, hipStream_t st) {
    const dim3 grid = tiles_of<S>(g, 1), block(S::NT);
    if constexpr (S::BN >= 128) {
        if (s.scaled) hipLaunchKernelGGL((diff_kernel<S, true, true, 2>), grid, block, 0, st, g, a);
    }
    if constexpr (S::BN <= 128) {
        if (s.terms == 3) hipLaunchKernelGGL((diff_kernel<S, false, false, 3>), grid, block, 0, st, g, a);
    }
    if (s.terms > 1) return;
    if (s.f16) hipLaunchKernelGGL((diff_kernel<S, true, false, 2>), grid, block, 0, st, g, a);
    else hipLaunchKernelGGL((diff_kernel<S, false, false, 2>), grid, block, 0, st, g, a);
}

#define GDN_BY_SHAPE(shape, call)              \
    switch (shape) {                           \
        case BIG: call(Big); break;            \
        case MID: call(Mid); break;            \
        case FEW: call(Few); break;            \
        default: call(One); break;             \
    }

}  // namespace ll
}  // namespace gdn

using namespace gdn;
using namespace gdn::ll;

static size_t need(const Sizes &s, bool dx, bool dw, bool bwd, bool copy_x, bool copy_w) {
    Space sp{nullptr};
    place(sp, s, dx, dw, bwd, copy_x, copy_w);
    return sp.at;
}

extern "C" size_t gdn_linear_loss_workspace_bytes(int64_t N, int64_t H, int64_t V, int dtype, int aligned, int want_dx,
                                                  int want_dw) {
    if (N <= 0 || H <= 0 || V <= 0 || N > MOST_TOKENS || V > 1 << 24 || H > 1 << 17) return 0;
    const bool copy = !aligned || dtype == GDN_F32 || H % BK, bwd = want_dx || want_dw;
    const Sizes s = sizes(N, H, V, dtype, want_dx);
    const size_t bytes = need(s, want_dx, want_dw, bwd, copy, copy);
    if (bwd || !wide(nullptr, 0, N, H, dtype)) return bytes;
    Space sp{nullptr};  // what the forward call needs for an aligned weight; x alone may be what is not aligned
    place_wide(sp, s);
    return aligned || bytes < sp.at ? sp.at : bytes;
}

extern "C" int gdn_linear_loss_fwd(const void *x, const void *w, const int64_t *targets, float *loss, float *stat, float *total,
                                   float *factor, void *workspace, size_t workspace_bytes, int64_t N, int64_t H, int64_t V,
                                   int64_t x_stride, int64_t w_stride, int64_t ignore_index, int reduction, int dtype,
                                   void *stream) {
    clear_error();
    if (const int rc = check(N, H, V, x_stride, w_stride, dtype)) return rc;
    if (reduction < 0 || reduction > 2) return fail(GDN_ERR_INVALID, "unknown reduction");
    if (reduction && (!total || !factor)) return fail(GDN_ERR_INVALID, "null pointer");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (N == 0 && !reduction) return GDN_OK;
    if (N > 0) {
        if (!x || !w || !targets || !loss || !workspace) return fail(GDN_ERR_INVALID, "null pointer");
        const bool dw = direct(w, w_stride, H, dtype);
        const Sizes s = sizes(N, H, V, dtype, false);
        const bool dx = !s.compact && direct(x, x_stride, H, dtype);
        const bool few = wide(w, w_stride, N, H, dtype);
        Space size{nullptr}, sp{static_cast<char *>(workspace)};
        if (few) place_wide(size, s);
        else place(size, s, false, false, false, !dx, !dw);
        if (workspace_bytes < size.at)
            return fail(GDN_ERR_WORKSPACE, "the workspace holds %zu bytes, %zu are needed", workspace_bytes, size.at);
        const Buffers b = few ? place_wide(sp, s) : place(sp, s, false, false, false, !dx, !dw);
        const int *exps = nullptr;
        const Tokens &tk = b.tokens;  // empty without
        const int64_t *tt = s.compact ? tk.target : targets;
        const Source sx{x, dtype, N, H, x_stride, s.compact ? nullptr : targets, ignore_index, tk.index, tk.count};
        const Source sw{w, dtype, V, H, w_stride, nullptr, 0, nullptr, nullptr};
        if (s.compact)
            hipLaunchKernelGGL(tokens_kernel, dim3(1), dim3(1024), 0, st, targets, N, ignore_index, tk, loss);
        if (s.scaled) {
            maxima({sx, sw}, b.part, st);
            int *to = stat ? reinterpret_cast<int *>(stat + 2 * N) : b.exps;
            exponents(b.part, TOP, to, b.most, st);  // b.most is not read
            exps = to;
            row_exponents(sx, TOP, b.each, st);
        }
        if (few) terms(sx, 3, false, nullptr, E_X, b.x, st);
        else if (!dx) terms(sx, s.terms, s.f16, b.each, EACH_ROW, b.x, st);
        // operands that are used as they lie need no pieces
        const int64_t step = dw ? V : s.piece;
        for (int64_t n0 = 0; n0 < N; n0 += s.tokens) {
            const int64_t tokens = N - n0 < s.tokens ? N - n0 : s.tokens;
            const int shape = plan(tokens, dw ? V : s.piece, s.slots * s.hp / BK, 1).shape;
            int parts = 0;
            if (few) {  // all tokens
                const Operand rows{reinterpret_cast<const char *>(b.x), 3 * s.hp * 2, N, {0, s.hp * 2, s.hp * 4}, 0};
                const WideArgs g{static_cast<const float *>(w), w_stride, V, rows, (int)(s.hp / BK)};
                const StatArgs a{tt, b.stats, b.zt, nullptr, nullptr, N, V, 0, 0};
                const dim3 grid((unsigned)((V + 127) / 128));
                Timed tm("loss_stat", st);
                if (N <= 32) hipLaunchKernelGGL((wide_kernel<2>), grid, dim3(256), 0, st, g, a);
                else if (N <= 64) hipLaunchKernelGGL((wide_kernel<4>), grid, dim3(256), 0, st, g, a);
                else hipLaunchKernelGGL((wide_kernel<8>), grid, dim3(256), 0, st, g, a);
                parts = 4 * (int)grid.x;
            }
            for (int64_t v0 = 0; v0 < V && !few; v0 += step) {
                const int64_t words = V - v0 < step ? V - v0 : step;
                Args g{};
                segments(g, s, false, s.hp, s.hp, s.hp);
                g.a.ld = g.b.ld = s.terms * s.hp * 2;
                g.a.rows = words;
                g.b.rows = tokens;
                g.live = tk.count;
                g.live0 = n0;
                g.a.p = reinterpret_cast<const char *>(b.w);
                g.b.p = reinterpret_cast<const char *>(b.x) + n0 * s.terms * s.hp * 2;
                if (dw) {
                    g.a.p = static_cast<const char *>(w);
                    g.a.ld = w_stride * 2;
                } else {
                    Source part = sw;
                    part.p = static_cast<const char *>(w) + v0 * w_stride * (dtype == GDN_F32 ? 4 : 2);
                    part.rows = words;
                    terms(part, s.terms, s.f16, exps, E_W, b.w, st);
                }
                if (dx) {
                    g.b.p = static_cast<const char *>(x) + n0 * x_stride * 2;
                    g.b.ld = x_stride * 2;
                }
                const StatArgs a{tt + n0, b.stats, b.zt, exps, s.scaled ? b.each + n0 : nullptr, tokens, V, v0, parts};
                Timed tm("loss_stat", st);
#define GDN_STAT(S)                                \
    launch_stat<S>(g, a, s, st);                   \
    parts += g.mt * S::WM
                GDN_BY_SHAPE(shape, GDN_STAT)
#undef GDN_STAT
            }
            Timed tm("loss_join", st);
            float2 *to = stat ? reinterpret_cast<float2 *>(stat) + n0 : nullptr;
            const int *index = s.compact ? tk.index + n0 : nullptr;
            float *each = s.compact ? loss : loss + n0;
            // 128 bytes of a part's tokens at a time, or all threads on the parts of one of few
            if (tokens > 64)
                hipLaunchKernelGGL((join_kernel<16>), grid_of((tokens + 15) / 16), dim3(NT), 0, st, tt + n0, b.stats, parts, b.zt,
                                   tokens, V, ignore_index, each, to, index, tk.count, n0);
            else
                hipLaunchKernelGGL((join_kernel<1>), grid_of(tokens), dim3(NT), 0, st, tt + n0, b.stats, parts, b.zt, tokens, V,
                                   ignore_index, each, to, index, tk.count, n0);
        }
    }
    if (reduction)
        hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, st, loss, targets, N, ignore_index, reduction == 2, total,
                           factor);
    return check_launch(st, "gdn_linear_loss_fwd");
}

extern "C" int gdn_linear_loss_bwd(const void *x, const void *w, const int64_t *targets, const float *stat, const float *dloss,
                                   int64_t dloss_stride, const float *factor, void *dx, void *dw, void *workspace,
                                   size_t workspace_bytes, int64_t N, int64_t H, int64_t V, int64_t x_stride, int64_t w_stride,
                                   int64_t ignore_index, int dtype, void *stream) {
    clear_error();
    if (const int rc = check(N, H, V, x_stride, w_stride, dtype)) return rc;
    if (dloss_stride < 0 || dloss_stride > 1) return fail(GDN_ERR_INVALID, "the cotangents' stride must be 0 or 1");
    if (!dx && !dw) return GDN_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (N == 0) return fail(GDN_ERR_INVALID, "no tokens: the gradients are zeros, which this call does not write");
    if (!x || !w || !targets || !stat || !dloss || !workspace) return fail(GDN_ERR_INVALID, "null pointer");
    const bool direct_w = direct(w, w_stride, H, dtype);
    const Sizes s = sizes(N, H, V, dtype, dx);
    const bool direct_x = !s.compact && direct(x, x_stride, H, dtype);
    const size_t bytes = need(s, dx, dw, true, !direct_x, !direct_w);
    if (workspace_bytes < bytes)
        return fail(GDN_ERR_WORKSPACE, "the workspace holds %zu bytes, %zu are needed", workspace_bytes, bytes);
    Space sp{static_cast<char *>(workspace)};
    const Buffers b = place(sp, s, dx, dw, true, !direct_x, !direct_w);
    const int elem = dtype == GDN_F32 ? 4 : 2, t = s.terms, shift = s.f16 ? -SHIFT : 0;
    const Tokens &tk = b.tokens;  // empty without
    const int64_t *tt = s.compact ? tk.target : targets;
    const Source sx{x, dtype, N, H, x_stride, s.compact ? nullptr : targets, ignore_index, tk.index, tk.count};
    const Source sw{w, dtype, V, H, w_stride, nullptr, 0, nullptr, nullptr};
    if (s.compact) hipLaunchKernelGGL(tokens_kernel, dim3(1), dim3(1024), 0, st, targets, N, ignore_index, tk, nullptr);
    hipLaunchKernelGGL(cotangent_kernel, dim3(PARTS), dim3(NT), 0, st, tt, dloss, dloss_stride, factor, N, V, ignore_index,
                       b.power, b.factor, b.part + 2 * PARTS, tk.index, tk.count);
    // what is stored times a power of two: both operands, for which the forward call has found it, or x across in fp16
    const int *exps = s.scaled ? reinterpret_cast<const int *>(stat + 2 * N) : b.exps;
    const bool scaled_x = dtype == GDN_F16 && dw;
    if (scaled_x) {
        Source none = sw;
        none.rows = 0;
        maxima({sx, none}, b.part, st);
    }
    if (dw) exponents(b.part, TOP, scaled_x ? b.exps : nullptr, b.most, st);
    if (s.scaled) row_exponents(sx, TOP, b.each, st);
    if (!direct_x) terms(sx, t, s.f16, b.each, EACH_ROW, b.x, st);
    if (dw) terms_across(sx, s.slots, s.f16, s.f16 ? exps : nullptr, E_X, Factors{b.power, b.most}, b.xt, st);
    const int shape = plan(N, s.piece, s.slots * s.hp / BK, 1).shape;
    for (int64_t v0 = 0; v0 < V; v0 += s.piece) {
        const int64_t words = V - v0 < s.piece ? V - v0 : s.piece, kp = padded(words);
        Source part = sw;
        part.p = static_cast<const char *>(w) + v0 * w_stride * elem;
        part.rows = words;
        Args g{};
        segments(g, s, false, s.hp, s.hp, s.hp);
        g.b.ld = t * s.hp * 2;
        g.a.rows = words;
        g.b.rows = N;
        g.live = tk.count;
        g.a.p = reinterpret_cast<const char *>(b.w);
        g.b.p = reinterpret_cast<const char *>(b.x);
        if (direct_w) {
            g.a.p = static_cast<const char *>(part.p);
            g.a.ld = w_stride * 2;
        } else {
            g.a.ld = s.wslots * s.hp * 2;
            terms(part, s.wslots, s.f16, s.scaled ? exps : nullptr, E_W, b.w, st);
        }
        if (direct_x) {
            g.b.p = static_cast<const char *>(x);
            g.b.ld = x_stride * 2;
        }
        const int64_t second = s.rows ? N * kp : kp;
        const DiffArgs a{tt, reinterpret_cast<const float2 *>(stat), b.power, b.factor, exps, b.each, b.p, v0, kp, s.pterms * kp,
                         second};
        {
            Timed tm("loss_diff", st);
#define GDN_DIFF(S) launch_diff<S>(g, a, s, st)
            GDN_BY_SHAPE(shape, GDN_DIFF)
#undef GDN_DIFF
        }
        if (dx) {
            Args h{};
            segments(h, s, !s.rows, kp, s.hp, kp);
            h.across = DOWN_A;
            h.down = words;
            h.a.p = g.a.p;
            h.a.ld = g.a.ld;
            h.a.rows = H;
            h.a.width = (direct_w ? H : s.hp) * 2;
            h.b.ld = s.pterms * kp * 2;
            h.b.p = reinterpret_cast<const char *>(b.p);
            h.b.rows = s.prows;
            h.live = tk.count;
            // parts without a block of the last piece add nothing
            const Result r{dx, H, dtype, b.power, exps, shift, {0, s.scaled ? -1 : 0}, b.acc_x, columns_of(H), v0 > 0, nullptr,
                           tk.place};
            multiply(h, s.f16, s.px, r, st);
            if (v0 + words == V) finish(r, s.px.splits * (int)(s.prows / N), N, H, st);  // terms as rows are parts too
        }
        if (dw) {
            Args h{};
            segments(h, s, true, s.np, s.np, second);
            h.a.p = reinterpret_cast<const char *>(b.xt);
            h.a.ld = s.slots * s.np * 2;
            h.a.rows = H;
            h.b.p = reinterpret_cast<const char *>(b.p);
            h.b.ld = s.pterms * kp * 2;
            h.b.rows = words;
            h.b.width = kp * 2;
            h.across = DOWN_B;
            h.down = N;
            h.live = tk.count;
            h.live_k = 1;
            Result r{static_cast<char *>(dw) + v0 * H * elem, H, dtype, nullptr, exps, shift, {s.f16 ? -1 : 0, 0}, nullptr,
                     columns_of(H), 0, b.most, nullptr};
            if (s.pw.splits > 1) r.acc = b.acc_w;
            multiply(h, s.f16, s.pw, r, st);
            if (r.acc) finish(r, s.pw.splits, words, H, st);
        }
    }
    return check_launch(st, "gdn_linear_loss_bwd");
}
