// Linear attention with a log decay for each head, forward and backward, for gfx950: the kernels that walk the chunks.
//
// Per value head h (reading key head h / (Hv / Hk)), with a_t = e^{g_t}:
//   S_t = a_t S_{t-1} + v_t k_t^T,   y_t = scale S_t q_t.
// In chunks of C tokens with G_r the running sum of g inside the chunk, S the state entering it:
//   Y  = diag(scale e^G) Q S^T + P V,   P_rs = scale e^{G_r - G_s} (q_r . k_s) for s <= r,
//   S' = e^{G_C} S + sum_s e^{G_C - G_s} v_s k_s^T.
// The gradients are the same expression with the roles exchanged.  With O = LA(Q', K', V') for the above and RLA for its
// time reverse (r >= s in the place of s <= r, the state's cotangent in the place of the state):
//   dQ = LA(dY, V, K),   dK = RLA(V, dY, Q),   dV = RLA(K, Q, dY),
// dg_t is what the loss draws from everything before t through everything from t on.  In t's chunk, with a_r = q_r . (dq_r
// from the state entering it), b_s = k_s . (dk_s from the cotangent of the state leaving it) and M_rs = P_rs (dy_r . v_s):
//   dg_t = c + sum_{r >= t} a_r + sum_{s < t} b_s + sum_{r >= t > s} M_rs,   c = e^{G_C} <dS', S>,
// sums without cancellation, and c by the chain c = D - sum b, D of the chunk before = c + sum a, from D = <dS_T, S_T> on.  A
// chunk whose decay is below 2^-30 starts the chain anew with c = 0, which is nearer than the difference of two fp32 sums:
// rounding errors do not outlive what they belong to.
// So one kernel, pass_kernel, computes all four.  Where there are few heads, the sequence is cut into segments: seg_kernel
// sums each segment's state from nothing, scan_kernel joins them to the states entering each segment, and the passes run all
// segments at once.
//
// Inputs in bf16 use v_mfma_f32_16x16x32_bf16, whose operands q, k, v and dy are exact; fp32 and fp16 inputs are held as fp32
// and use v_mfma_f32_16x16x4_f32.  Sums and states are fp32, decays' sums fp64.  What bf16 rounds besides:
//   P and the state as operands of Y, once (2^-8 of an element at most, as the output's own rounding);
//   the state in the passes that a and b are formed from, in two terms (2^-17): the chain subtracts them;
//   e^{G_C - G_s} v_s in three terms (2^-26): the final state is an fp32 output.
#pragma once

#include <type_traits>

#include "gdn_common.h"
#include "gdn_host.h"
#include "gdn_vec.h"

namespace gdn {
namespace la {

constexpr int NT = 256;
constexpr int C = 64;  // tokens of a chunk
constexpr double LOG2E = 1.4426950408889634074;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16;
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));

// A 16 x 32 operand: lane l holds row l % 16 at the 8 indices 8 (l / 16) + j of the summed axis.
struct F32Frag {
    float v[8];
};
template <typename ET>
using Frag = std::conditional_t<std::is_same_v<ET, float>, F32Frag, bf8>;

// acc += A B^T over 32 summed indices; accumulator element e of lane l is (row 4 (l / 16) + e, column l % 16).
__device__ __forceinline__ f4 mma(const bf8 &a, const bf8 &b, f4 acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f4 mma(const F32Frag &a, const F32Frag &b, f4 acc) {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], acc, 0, 0, 0);
    return acc;
}

// The operand whose summed axis is contiguous: p is the lane's first element.
__device__ __forceinline__ bf8 row_frag(const bf16 *p) { return *reinterpret_cast<const bf8 *>(p); }
__device__ __forceinline__ F32Frag row_frag(const float *p) {
    F32Frag f;
    const f4 a = *reinterpret_cast<const f4 *>(p), b = *reinterpret_cast<const f4 *>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f.v[j] = a[j];
        f.v[4 + j] = b[j];
    }
    return f;
}

// The operand whose summed axis runs down the rows k0 .. k0 + 31 of a tile: lane 4 c + i of 16 holds column c0 + c cs + i.
// bf16: the LDS's transposing read, where the four lanes 4 j .. 4 j + 3 of 16 give the addresses of row j's four quads of
// columns and lane 4 c + i receives column i of quad c, rows 0 to 3.
__device__ __forceinline__ bf8 col_frag(const bf16 *t, int ld, int k0, int c0, int cs) {
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const int l = threadIdx.x & 63, li = l & 15, g = l >> 4;
    const bf16 *p = t + (k0 + 8 * g + (li >> 2)) * ld + c0 + (li & 3) * cs;
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)p);
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + 4 * ld));
    return __builtin_bit_cast(bf8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ F32Frag col_frag(const float *t, int ld, int k0, int c0, int cs) {
    const int l = threadIdx.x & 63, li = l & 15, g = l >> 4;
    const float *p = t + (k0 + 8 * g) * ld + c0 + (li >> 2) * cs + (li & 3);
    F32Frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = p[j * ld];
    return f;
}

// x as the sum of N operands (fp32: itself).
template <int N>
__device__ __forceinline__ void split(const float (&x)[8], bf8 (&o)[N]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float r = x[j];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const bf16 h = (bf16)r;
            o[n][j] = h;
            r -= (float)h;
        }
    }
}
template <int N>
__device__ __forceinline__ void split(const float (&x)[8], F32Frag (&o)[N]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[0].v[j] = x[j];
}
__device__ __forceinline__ void to_f32(const bf8 &a, float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)a[j];
}
__device__ __forceinline__ void to_f32(const F32Frag &a, float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = a.v[j];
}

template <typename ET>
constexpr int pad() { return std::is_same_v<ET, float> ? 4 : 8; }  // 16 bytes: rows of a 16-byte read in other banks

// A tensor [B][T][heads][D], channels contiguous; value head h reads head h / div.
struct Ten {
    const void *p;
    int64_t sb, st, sh;
    int div, vec;  // vec: every 8-channel piece is 16-byte aligned and D % 8 == 0
    __host__ __device__ int64_t at(int b, int64_t t, int h) const { return b * sb + t * st + (h / div) * sh; }
};

// A [ROWS][W] tile in registers on its way from memory to LDS; rows >= n and columns >= w are zero.
template <typename ET, int ROWS, int W>
struct Tile {
    static constexpr int PER = ROWS * W / 8 / NT;
    static_assert(PER * NT * 8 == ROWS * W, "a tile splits evenly");
    std::conditional_t<std::is_same_v<ET, float>, float, uint32_t> x[PER][std::is_same_v<ET, float> ? 8 : 4];
    __device__ __forceinline__ void fetch(const Ten &t, int64_t at, int n, int w, int dt) {
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int v = threadIdx.x + p * NT, r = v / (W / 8), c = (v % (W / 8)) * 8;
            const int64_t i = at + r * t.st + c;
#pragma unroll
            for (int j = 0; j < (int)(sizeof(x[p]) / 4); ++j) x[p][j] = 0;
            if (r >= n || c >= w) continue;
            if (t.vec) {
                if constexpr (std::is_same_v<ET, float>) {
                    ops::loadv<8>(t.p, i, dt, x[p]);
                } else {
                    const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(t.p) + i);
                    x[p][0] = u.x; x[p][1] = u.y; x[p][2] = u.z; x[p][3] = u.w;
                }
            } else if constexpr (std::is_same_v<ET, float>) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < w) x[p][j] = load_as_f32(t.p, i + j, dt);
            } else {
                const uint16_t *s = static_cast<const uint16_t *>(t.p) + i;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < w) x[p][j / 2] |= (uint32_t)s[j] << (16 * (j & 1));
            }
        }
    }
    __device__ __forceinline__ void store(ET *dst) const {
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int v = threadIdx.x + p * NT, r = v / (W / 8), c = (v % (W / 8)) * 8;
            ET *d = dst + r * (W + pad<ET>()) + c;
            if constexpr (std::is_same_v<ET, float>) {
                *reinterpret_cast<float4 *>(d) = make_float4(x[p][0], x[p][1], x[p][2], x[p][3]);
                *reinterpret_cast<float4 *>(d + 4) = make_float4(x[p][4], x[p][5], x[p][6], x[p][7]);
            } else {
                *reinterpret_cast<uint4 *>(d) = make_uint4(x[p][0], x[p][1], x[p][2], x[p][3]);
            }
        }
    }
};

struct Gate {
    const void *p;
    int64_t sb, st, sh;
    int dt;
    // log decays below -1e4 (-inf: nothing is kept) run as -1e4, whose exponential is 0 and whose differences are finite
    __device__ __forceinline__ float load(int b, int64_t t, int h) const {
        const float g = load_as_f32(p, b * sb + t * st + h * sh, dt);
        return g < -1e4f ? -1e4f : g;
    }
};

// Of one chunk: G (in powers of two), and the weights of its outputs and sources, e^{G_r} and e^{G_C - G_s} (reverse: the
// other way round), the scale in the outputs' (reverse: the sources').
struct Decays {
    double G[C];
    float wo[C], ws[C], total;
    // wave 0; g of token t in lane t, 0 past the end
    template <bool REV>
    __device__ __forceinline__ void set(float g, float scale) {
        const int l = threadIdx.x & 63;
        const double s = wave_prefix_sum((double)g * LOG2E), end = readlane_f64(s, C - 1);
        {
            const float in = __builtin_amdgcn_exp2f((float)s), out = __builtin_amdgcn_exp2f((float)(end - s));
            G[l] = s;
            wo[l] = REV ? out : in * scale;
            ws[l] = REV ? in * scale : out;
        }
        if (l == 0) total = __builtin_amdgcn_exp2f((float)end);
    }
};

enum Kind { Y, DQ, DK, DV };  // what a pass computes

struct Pass {
    Ten Q, K, V, X;
    Gate g;
    const float *s_in;  // states entering the segments, head (b, h) at s_in + (b Hv + h) s_head, segment j at + j s_seg; or NULL
    float *s_out;       // the state leaving the last segment (reverse: the first), [B][Hv][..], or NULL
    int64_t s_head, s_seg;
    int s_t;            // states are [v'][k'] (0) or [k'][v'] (1)
    void *o;            // [B][T][heads][dv] contiguous
    float *dot;         // per token [slices][B][Hv][T]: DQ, DK X . (O from the state); DV the pairs that cross it, X = v
    float *decay;       // DK: of each chunk, [B][Hv][nc]
    int B, T, Hv, dk, dv, slices, nseg, cps, nc;  // cps: chunks of a segment, nc: of the sequence
    int dt, o_dt, o_vec;
    float scale;
};

// fp32 tiles of 256 channels leave no room for P and X, which then take the place of Q' once that is used.
template <typename ET, int D>
constexpr bool p_over_q() { return std::is_same_v<ET, float> && D > 128; }

template <typename ET, int D, int NV, int KIND>
struct Shared {
    static constexpr int LV = 64 * NV + pad<ET>(), LP = C + pad<ET>();
    static constexpr bool TAKEN = p_over_q<ET, D>();
    ET Q[C * (D + pad<ET>())], K[C * (D + pad<ET>())], V[C * LV];
    ET own_p[TAKEN ? 8 : C * LP], own_x[KIND == DV && !TAKEN ? C * LV : 8];
    Decays d;
    float dot[4][C];
    double cross[KIND == DV ? 4 : 1][C];
    __device__ __forceinline__ ET *p() { return TAKEN ? Q : own_p; }
    __device__ __forceinline__ ET *x() { return TAKEN ? Q + C * LP : own_x; }
};

// The state of a wave: K' rows 32 T + 8 (l / 16) + 4 (t & 1) + e of tile t = 2 T, 2 T + 1 by its columns 16 NV w + ...: what
// lane l holds of two tiles is 8 consecutive K' rows of one column, an operand as it stands.
template <int D, int NV>
struct State {
    f4 s[D / 16][NV];
    // the lane's column of tile n
    static __device__ __forceinline__ int col(int n) {
        const int l = threadIdx.x & 63, li = l & 15, w = threadIdx.x >> 6;
        return 16 * NV * w + 4 * NV * (li >> 2) + 4 * n + (li & 3);
    }
    template <typename F>
    __device__ __forceinline__ void each(int dk, int dv, int c0, F f) {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = 32 * (t >> 1) + 8 * g + 4 * (t & 1) + e, v = c0 + col(n);
                    f(s[t][n], e, k, v, k < dk && v < dv);
                }
    }
    __device__ __forceinline__ void load(const float *p, int dk, int dv, int c0, int tr) {
        each(dk, dv, c0, [&](f4 &x, int e, int k, int v, bool in) {
            x[e] = p && in ? p[tr ? (int64_t)k * dv + v : (int64_t)v * dk + k] : 0.f;
        });
    }
    __device__ __forceinline__ void store(float *p, int dk, int dv, int c0, int tr) {
        each(dk, dv, c0, [&](f4 &x, int e, int k, int v, bool in) {
            if (in) p[tr ? (int64_t)k * dv + v : (int64_t)v * dk + k] = x[e];
        });
    }
    // s = total s + sum over 32 rows of the tiles: K'^T diag(weights) V', the weighted V' in NS terms
    template <int NS, typename ET>
    __device__ __forceinline__ void add(const ET *sK, int k0, const Frag<ET> (&vw)[NV][NS]) {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
            const Frag<ET> a = col_frag(sK, D + pad<ET>(), k0, 32 * (t >> 1) + 4 * (t & 1), 8);
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int n = 0; n < NV; ++n) s[t][n] = mma(a, vw[n][i], s[t][n]);
        }
    }
};

template <typename ET, int N>
__device__ __forceinline__ void weigh(const Frag<ET> &v, const float *w, Frag<ET> (&o)[N]) {
    float x[8];
    to_f32(v, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= w[j];
    split(x, o);
}

// One segment of one value head, 64 NV columns of V'.
template <typename ET, int D, int NV, int KIND>
__global__ __launch_bounds__(NT) void pass_kernel(const Pass a) {
    constexpr bool F32 = std::is_same_v<ET, float>, REV = KIND >= DK, DOT = KIND == DQ || KIND == DK;
    constexpr int NS = F32 ? 1 : 3, NH = F32 || !DOT ? 1 : 2;  // terms of the weighted V', of the state as an operand
    constexpr int LK = D + pad<ET>(), LV = 64 * NV + pad<ET>(), LP = C + pad<ET>(), RT = C / 16;
    constexpr bool TAKEN = Shared<ET, D, NV, KIND>::TAKEN;
    __shared__ __attribute__((aligned(16))) Shared<ET, D, NV, KIND> sh;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, li = l & 15, g = l >> 4;
    int id = blockIdx.x;
    const int slice = id % a.slices;
    id /= a.slices;
    const int h = id % a.Hv;
    id /= a.Hv;
    const int b = id % a.B, seg = id / a.B, c0 = slice * 64 * NV;
    const int first = seg * a.cps, last = min(a.nc, first + a.cps) - 1;
    const int64_t head = (int64_t)b * a.Hv + h;

    State<D, NV> S;
    S.load(a.s_in ? a.s_in + head * a.s_head + seg * a.s_seg : nullptr, a.dk, a.dv, c0, a.s_t);

    Tile<ET, C, D> tq, tk;
    Tile<ET, C, 64 * NV> tv, tx;
    float tg = 0.f;
    const auto fetch = [&](int c) {
        const int64_t t0 = (int64_t)c * C;
        const int n = min((int64_t)C, a.T - t0);
        tq.fetch(a.Q, a.Q.at(b, t0, h), n, a.dk, a.dt);
        tk.fetch(a.K, a.K.at(b, t0, h), n, a.dk, a.dt);
        tv.fetch(a.V, a.V.at(b, t0, h) + c0, n, a.dv - c0, a.dt);
        if constexpr (KIND == DV && !TAKEN) tx.fetch(a.X, a.X.at(b, t0, h) + c0, n, a.dv - c0, a.dt);
        if (w == 0) tg = l < n ? a.g.load(b, t0 + l, h) : 0.f;
    };
    for (int i = first - 1; i <= last; ++i) {
        if (i >= first) {
            __syncthreads();
            tq.store(sh.Q);
            tk.store(sh.K);
            tv.store(sh.V);
            if constexpr (KIND == DV && !TAKEN) tx.store(sh.x());
            if (w == 0) sh.d.template set<REV>(tg, a.scale);
            __syncthreads();
        }
        if (i < last) fetch(REV ? first + last - i - 1 : i + 1);
        if (i < first) continue;
        const int c = REV ? first + last - i : i;
        const int64_t t0 = (int64_t)c * C;
        const int n = min((int64_t)C, a.T - t0);

        // O = diag(wo) S Q'^T, later + P V', transposed: a lane holds one token, 4 NV consecutive columns
        f4 O[RT][NV];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int x = 0; x < NV; ++x) O[rt][x] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int T = 0; T < D / 32; ++T) {
            Frag<ET> f[NV][NH];
#pragma unroll
            for (int x = 0; x < NV; ++x) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[e] = S.s[2 * T][x][e];
                    y[4 + e] = S.s[2 * T + 1][x][e];
                }
                split(y, f[x]);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const Frag<ET> q = row_frag(sh.Q + (16 * rt + li) * LK + 32 * T + 8 * g);
#pragma unroll
                for (int j = 0; j < NH; ++j)
#pragma unroll
                    for (int x = 0; x < NV; ++x) O[rt][x] = mma(f[x][j], q, O[rt][x]);
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float wo = sh.d.wo[16 * rt + li];
#pragma unroll
            for (int x = 0; x < NV; ++x) O[rt][x] *= wo;
        }
        const int col = c0 + 16 * NV * w + 4 * NV * g;  // the lane's first column of O
        const auto row_of = [&](int rt, float (&o)[4 * NV]) {
#pragma unroll
            for (int x = 0; x < NV; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[4 * x + e] = O[rt][x][e];
        };
        if constexpr (DOT) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int r = 16 * rt + li;
                float o[4 * NV], s = 0.f;
                row_of(rt, o);
                if (r < n) {
                    const int64_t at = a.X.at(b, t0 + r, h) + col;
                    if (a.X.vec && col + 4 * NV <= a.dv) {
                        float x[4 * NV];
                        ops::loadv<4 * NV>(a.X.p, at, a.dt, x);
#pragma unroll
                        for (int j = 0; j < 4 * NV; ++j) s = fmaf(x[j], o[j], s);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4 * NV; ++j)
                            if (col + j < a.dv) s = fmaf(load_as_f32(a.X.p, at + j, a.dt), o[j], s);
                    }
                }
                s += lane_xor16(s);
                s += lane_xor32(s);
                if (g == 0) sh.dot[w][r] = s;
            }
        }

        // P: blocks (rt, st) of 16 outputs by 16 sources with st <= rt (reverse: >=), one to a wave in turn; the blocks that
        // fill a product's 32 sources are zeros
        {
            ET *const sP = sh.p();
            f4 acc[3];
            int e = 0;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int st = REV ? rt : 0; st < (REV ? RT : rt + 1); ++st, ++e) {
                    if ((e & 3) != w) continue;
                    f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < D; k += 32)
                        x = mma(row_frag(sh.K + (16 * st + li) * LK + k + 8 * g),
                                row_frag(sh.Q + (16 * rt + li) * LK + k + 8 * g), x);
                    acc[e >> 2] = x;
                }
            if constexpr (TAKEN) __syncthreads();
            if constexpr (KIND == DV && TAKEN) {
                tx.fetch(a.X, a.X.at(b, t0, h) + c0, n, a.dv - c0, a.dt);
                tx.store(sh.x());
            }
            const auto put = [&](int rt, int st, const ET (&p)[4]) {
                ET *o = sP + (16 * rt + li) * LP + 16 * st + 4 * g;
                if constexpr (F32) *reinterpret_cast<float4 *>(o) = make_float4(p[0], p[1], p[2], p[3]);
                else *reinterpret_cast<uint2 *>(o) = *reinterpret_cast<const uint2 *>(p);
            };
            e = 0;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                for (int st = REV ? rt : 0; st < (REV ? RT : rt + 1); ++st, ++e) {
                    if ((e & 3) != w) continue;
                    const int r = 16 * rt + li, s0 = 16 * st + 4 * g;
                    const double gr = sh.d.G[r];
                    ET p[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float d = (float)(REV ? sh.d.G[s0 + j] - gr : gr - sh.d.G[s0 + j]);
                        const bool in = REV ? s0 + j >= r : s0 + j <= r;
                        acc[e >> 2][j] = in ? acc[e >> 2][j] * (a.scale * __builtin_amdgcn_exp2f(d)) : 0.f;
                        p[j] = (ET)acc[e >> 2][j];
                    }
                    put(rt, st, p);
                }
                const ET zero[4] = {(ET)0.f, (ET)0.f, (ET)0.f, (ET)0.f};
                if (w == rt && (rt & 1) == (REV ? 1 : 0)) put(rt, rt ^ 1, zero);
            }
            __syncthreads();
            // M of the same blocks, its sums over outputs and sources apart in 64 bits: their difference from a token on is
            // the sum of the pairs that cross it
            if constexpr (KIND == DV) {
                double *cross = sh.cross[w];
                cross[l] = 0.;
                e = 0;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int st = rt; st < RT; ++st, ++e) {
                        if ((e & 3) != w) continue;
                        f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int k = 0; k < 64 * NV; k += 32)
                            x = mma(row_frag(sh.V + (16 * st + li) * LV + k + 8 * g),
                                    row_frag(sh.x() + (16 * rt + li) * LV + k + 8 * g), x);
                        double out = 0.;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int s = 16 * st + 4 * g + j;
                            double m = s > 16 * rt + li ? (double)x[j] * (double)acc[e >> 2][j] : 0.;
                            out += m;
                            m += dpp_mov_f64<DPP_QUAD_1032>(m);
                            m += dpp_mov_f64<DPP_QUAD_2301>(m);
                            m += dpp_mov_f64<DPP_ROW_HALF_MIRROR>(m);
                            m += dpp_mov_f64<DPP_ROW_MIRROR>(m);
                            if (li == 0) cross[s] += m;
                        }
                        out += __shfl_xor(out, 16);
                        out += __shfl_xor(out, 32);
                        if (g == 0) cross[16 * rt + li] -= out;
                    }
            }
        }
        const float total = sh.d.total;
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int x = 0; x < NV; ++x) S.s[t][x] *= total;
#pragma unroll
        for (int k0 = 0; k0 < C; k0 += 32) {
            Frag<ET> v[NV], vw[NV][NS];
#pragma unroll
            for (int x = 0; x < NV; ++x) {
                v[x] = col_frag(sh.V, LV, k0, 16 * NV * w + 4 * x, 4 * NV);
                weigh<ET>(v[x], sh.d.ws + k0 + 8 * g, vw[x]);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (REV ? 16 * rt >= k0 + 32 : 16 * rt + 16 <= k0) continue;
                const Frag<ET> p = row_frag(sh.p() + (16 * rt + li) * LP + k0 + 8 * g);
#pragma unroll
                for (int x = 0; x < NV; ++x) O[rt][x] = mma(v[x], p, O[rt][x]);
            }
            S.template add<NS, ET>(sh.K, k0, vw);
        }

#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = 16 * rt + li;
            float o[4 * NV];
            row_of(rt, o);
            if (r < n) {
                const int64_t at = ((b * (int64_t)a.T + t0 + r) * a.Hv + h) * a.dv + col;
                if (a.o_vec && col + 4 * NV <= a.dv) {
                    ops::storev<4 * NV>(a.o, at, a.o_dt, o);
                } else {
#pragma unroll
                    for (int j = 0; j < 4 * NV; ++j)
                        if (col + j < a.dv) store_from_f32(a.o, at + j, o[j], a.o_dt);
                }
            }
        }
        const int64_t at = (((int64_t)slice * a.B + b) * a.Hv + h) * a.T + t0;
        if constexpr (DOT) {
            __syncthreads();
            if (tid < n) a.dot[at + tid] = (sh.dot[0][tid] + sh.dot[1][tid]) + (sh.dot[2][tid] + sh.dot[3][tid]);
            if (KIND == DK && tid == 0 && slice == 0) a.decay[head * a.nc + c] = total;
        }
        if constexpr (KIND == DV) {
            __syncthreads();
            if (w == 0) {
                const int t = C - 1 - l;
                const double x = (sh.cross[0][t] + sh.cross[1][t]) + (sh.cross[2][t] + sh.cross[3][t]);
                const double s = wave_prefix_sum(x);
                if (t < n) a.dot[at + t] = (float)s;
            }
        }
    }
    if (a.s_out && seg == (REV ? 0 : a.nseg - 1)) S.store(a.s_out + head * a.dk * a.dv, a.dk, a.dv, c0, a.s_t);
}

struct Seg {
    Ten K, V;
    Gate g;
    float *s;      // [B][Hv][nseg][dv][dk]
    float *decay;  // [B][Hv][nseg]
    int B, T, Hv, dk, dv, slices, nseg, cps, nc, dt;
    float scale;
};

// What a segment adds to a state that starts from nothing, and its decay.  The segment that the chain ends with is left out
// (the last; reverse: the first).
template <typename ET, int D, int NV, bool REV>
__global__ __launch_bounds__(NT) void seg_kernel(const Seg a) {
    constexpr int NS = std::is_same_v<ET, float> ? 1 : 3, LV = 64 * NV + pad<ET>();
    __shared__ __attribute__((aligned(16))) ET sK[C * (D + pad<ET>())];
    __shared__ __attribute__((aligned(16))) ET sV[C * LV];
    __shared__ Decays d;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4;
    int id = blockIdx.x;
    const int slice = id % a.slices;
    id /= a.slices;
    const int h = id % a.Hv;
    id /= a.Hv;
    const int b = id % a.B, seg = id / a.B + (REV ? 1 : 0), c0 = slice * 64 * NV;
    const int first = seg * a.cps, last = min(a.nc, first + a.cps) - 1;
    State<D, NV> S;
    S.load(nullptr, a.dk, a.dv, c0, 0);
    Tile<ET, C, D> tk;
    Tile<ET, C, 64 * NV> tv;
    float tg = 0.f, all = 1.f;
    const auto fetch = [&](int c) {
        const int64_t t0 = (int64_t)c * C;
        const int n = min((int64_t)C, a.T - t0);
        tk.fetch(a.K, a.K.at(b, t0, h), n, a.dk, a.dt);
        tv.fetch(a.V, a.V.at(b, t0, h) + c0, n, a.dv - c0, a.dt);
        if (w == 0) tg = l < n ? a.g.load(b, t0 + l, h) : 0.f;
    };
    for (int i = first - 1; i <= last; ++i) {
        if (i >= first) {
            __syncthreads();
            tk.store(sK);
            tv.store(sV);
            if (w == 0) d.template set<REV>(tg, a.scale);
            __syncthreads();
        }
        if (i < last) fetch(REV ? first + last - i - 1 : i + 1);
        if (i < first) continue;
        const float total = d.total;
        all *= total;
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int x = 0; x < NV; ++x) S.s[t][x] *= total;
#pragma unroll
        for (int k0 = 0; k0 < C; k0 += 32) {
            Frag<ET> vw[NV][NS];
#pragma unroll
            for (int x = 0; x < NV; ++x)
                weigh<ET>(col_frag(sV, LV, k0, 16 * NV * w + 4 * x, 4 * NV), d.ws + k0 + 8 * g, vw[x]);
            S.template add<NS, ET>(sK, k0, vw);
        }
    }
    const int64_t at = ((int64_t)b * a.Hv + h) * a.nseg + seg;
    S.store(a.s + at * a.dk * a.dv, a.dk, a.dv, c0, 0);
    if (tid == 0 && slice == 0) a.decay[at] = all;
}

// Columns of V' to a workgroup: 64, or 128 where the state of 128 fits the registers beside the tiles.
inline int cols_of(int dk, int dv) { return dv <= 64 || dk > 128 ? 64 : 128; }

// Launches for K' heads of up to 64, 128 and 256 channels; a.slices is set.
void pass_d64(const Pass &a, Kind kind, hipStream_t st);
void pass_d128(const Pass &a, Kind kind, hipStream_t st);
void pass_d256(const Pass &a, Kind kind, hipStream_t st);
void seg_d64(const Seg &a, bool rev, hipStream_t st);
void seg_d128(const Seg &a, bool rev, hipStream_t st);
void seg_d256(const Seg &a, bool rev, hipStream_t st);

template <typename ET, int D, int NV>
void launch_pass(const Pass &a, Kind kind, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.slices * a.Hv * a.B * a.nseg));
    if (kind == Y) hipLaunchKernelGGL((pass_kernel<ET, D, NV, Y>), grid, dim3(NT), 0, st, a);
    else if (kind == DQ) hipLaunchKernelGGL((pass_kernel<ET, D, NV, DQ>), grid, dim3(NT), 0, st, a);
    else if (kind == DK) hipLaunchKernelGGL((pass_kernel<ET, D, NV, DK>), grid, dim3(NT), 0, st, a);
    else hipLaunchKernelGGL((pass_kernel<ET, D, NV, DV>), grid, dim3(NT), 0, st, a);
}
template <typename ET, int D, int NV>
void launch_seg(const Seg &a, bool rev, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.slices * a.Hv * a.B * (a.nseg - 1)));
    if (rev) hipLaunchKernelGGL((seg_kernel<ET, D, NV, true>), grid, dim3(NT), 0, st, a);
    else hipLaunchKernelGGL((seg_kernel<ET, D, NV, false>), grid, dim3(NT), 0, st, a);
}

}  // namespace la
}  // namespace gdn
