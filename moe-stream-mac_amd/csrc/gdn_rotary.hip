// Rotary positions on q and k in one launch, for gfx950.
//
// Pair i of a head's first R channels turns by the angle p * inv_freq[i] of its token's position p:
//   (a, b) -> factor * (a cos - b sin, b cos + a sin),
// with the pair (i, i + R/2) in the half layout and (2i, 2i + 1) in the interleaved one; channels from R on pass through.
// The gradient of the inputs is the same turn backwards (the transposed 2x2 matrix): sign = -1.
//
// Angles of far positions lose everything in 32 bits (p = 10^6: half an ulp is 0.03 rad), so turns p * inv_freq / 2 pi
// are formed and reduced to [-1/2, 1/2] in 64 bits; sine and cosine of what is left are 32-bit.  That is R/2 pairs per
// token, shared by its heads through LDS.  The rest is a copy: 2 x 8192 tokens of 48 heads of 128 bf16 channels, 0.40 GB, in
// 87 us (4.6 TB/s; a plain copy 5.1).  One head and one vector at a time took 159 us, the type looked up per load 120.
//
// Loads are as wide as sizes, strides and addresses allow: 89 us a launch of that size with 8 channels each, 100 with 4 (rows of
// the projection 4 channels longer), 226 with one (an odd row, as of a projection of q, k, v and an odd number of decays).
#include "gdn_common.h"
#include "gdn_host.h"
#include "gdn_vec.h"
#include "../../include/gdn_mi355x.h"

namespace gdn {
namespace rope {

constexpr int NT = 256;
constexpr int MAX_R = 1024;  // channels that turn: 512 pairs per token in LDS
constexpr int MAX_TOK = 4;   // tokens to a workgroup

struct Args {
    const void *x[2];      // q, k
    void *y[2];            // contiguous [B][T][H][D]
    int64_t sb[2], st[2], sh[2];
    int H[2];
    const void *pos;
    int64_t psb, pst;
    int pos64;
    const double *inv;
    float factor, sign;
    int64_t tokens;        // B * T
    int T, D, R, interleaved, tok, units, lanes;
};

// A unit is 2 V channels: V pairs that turn, or as many that pass.  `lanes` (a power of two) lanes walk the units of one head;
// a workgroup takes `tok` tokens, whose places in memory are worked out once, and its groups of lanes two heads at a time,
// loads first: 16 bytes times four under way for each lane.
template <int V, int DT>
struct Unit {
    float p[V], q[V];
    int e0, e1;
    bool turns, second;
    __device__ __forceinline__ void load(const Args &a, const void *x, int64_t at, int u, int turning) {
        turns = u < turning;
        e0 = turns ? (a.interleaved ? 2 * V * u : V * u) : a.R + (u - turning) * 2 * V;
        e1 = turns && !a.interleaved ? e0 + a.R / 2 : e0 + V;
        second = e1 < a.D;
        ops::loadv<V>(x, at + e0, DT, p);
        ops::loadv<V>(x, at + (second ? e1 : e0), DT, q);
    }
    __device__ __forceinline__ void store(const Args &a, void *y, int64_t at, const float2 *c) {
        if (turns) {
            if (a.interleaved) {
                float z[2 * V];
#pragma unroll
                for (int i = 0; i < V; ++i) { z[i] = p[i]; z[V + i] = q[i]; }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float r = z[2 * i], s = z[2 * i + 1];
                    z[2 * i] = r * c[i].x - s * c[i].y;
                    z[2 * i + 1] = s * c[i].x + r * c[i].y;
                }
#pragma unroll
                for (int i = 0; i < V; ++i) { p[i] = z[i]; q[i] = z[V + i]; }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float r = p[i], s = q[i];
                    p[i] = r * c[i].x - s * c[i].y;
                    q[i] = s * c[i].x + r * c[i].y;
                }
            }
        }
        ops::storev<V>(y, at + e0, DT, p);
        if (second) ops::storev<V>(y, at + e1, DT, q);
    }
};

template <int V, int DT>
__global__ __launch_bounds__(NT) void rotary_kernel(const Args a) {
    extern __shared__ float2 cs[];  // [tok][R / 2]
    __shared__ int64_t from[MAX_TOK][2];
    const int tid = threadIdx.x, half = a.R / 2;
    const int64_t t0 = block_index() * a.tok;
    if (t0 >= a.tokens) return;
    const int ntok = (int)min((int64_t)a.tok, a.tokens - t0);
    if (tid < ntok) {
        const int64_t b = (t0 + tid) / a.T, t = (t0 + tid) % a.T;
        for (int w = 0; w < 2; ++w) from[tid][w] = b * a.sb[w] + t * a.st[w];
    }
    for (int i = tid; i < ntok * half; i += NT) {
        const int tk = i / half;
        const int64_t b = (t0 + tk) / a.T, at = b * a.psb + (t0 + tk - b * a.T) * a.pst;
        const double p = a.pos64 ? (double)static_cast<const int64_t *>(a.pos)[at]
                                 : (double)static_cast<const int32_t *>(a.pos)[at];
        const double turns = p * a.inv[i - tk * half] * 0.15915494309189533577;  // 1 / 2 pi
        const float f = 2.f * (float)(turns - rint(turns));
        cs[i] = make_float2(a.factor * cospif(f), a.sign * a.factor * sinpif(f));
    }
    __syncthreads();
    const int lane = tid & (a.lanes - 1), slots = NT / a.lanes;
    const int heads = a.H[0] + a.H[1], turning = a.R / (2 * V);
    int tk = 0, hh = tid / a.lanes;  // this group's next head
    const auto skip = [&] {
        while (hh >= heads && tk < ntok) { hh -= heads; ++tk; }
    };
    skip();
    while (tk < ntok) {
        int64_t in[2], out[2];
        int w[2], at[2], n = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // a group without a second head loads the first again
            const bool any = tk < ntok;
            const int k = any ? tk : at[0], g = any ? hh : -1;
            w[i] = any ? g >= a.H[0] : w[0];
            const int h = w[i] ? g - a.H[0] : g;
            in[i] = any ? from[k][w[i]] + h * a.sh[w[i]] : in[0];
            out[i] = any ? ((t0 + k) * a.H[w[i]] + h) * a.D : out[0];
            at[i] = k;
            n += any;
            hh += slots;
            skip();
        }
        for (int u = lane; u < a.units; u += a.lanes) {
            Unit<V, DT> x, y;
            x.load(a, a.x[w[0]], in[0], u, turning);
            y.load(a, a.x[w[1]], in[1], u, turning);
            x.store(a, a.y[w[0]], out[0], cs + at[0] * half + (u < turning ? V * u : 0));
            if (n == 2) y.store(a, a.y[w[1]], out[1], cs + at[1] * half + (u < turning ? V * u : 0));
        }
    }
}

}  // namespace rope
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_rotary(const void *q, const void *k, void *q_out, void *k_out, const void *positions,
                          const double *inv_freq, int64_t q_stride_b, int64_t q_stride_t, int64_t q_stride_h,
                          int64_t k_stride_b, int64_t k_stride_t, int64_t k_stride_h, int64_t pos_stride_b,
                          int64_t pos_stride_t, int B, int T, int Hq, int Hk, int D, int R, int interleaved,
                          int backward, int positions_64, float factor, int dtype, void *stream) {
    clear_error();
    if (B < 0 || T < 0 || Hq < 0 || Hk < 0 || D <= 0)
        return fail(GDN_ERR_INVALID, "B, T and the head counts must be >= 0 and D > 0");
    if (R <= 0 || R % 2 || R > D) return fail(GDN_ERR_INVALID, "the rotated part must be even, > 0 and <= D");
    if (R > rope::MAX_R) return fail(GDN_ERR_UNSUPPORTED, "more than %d rotated channels are not supported", rope::MAX_R);
    if (dtype != GDN_F32 && dtype != GDN_BF16 && dtype != GDN_F16) return fail(GDN_ERR_INVALID, "unknown dtype code");
    const int64_t tokens = (int64_t)B * T;
    if (tokens == 0 || Hq + Hk == 0) return GDN_OK;
    if ((int64_t)Hq + Hk > 65536) return fail(GDN_ERR_UNSUPPORTED, "more than 65536 heads are not supported");
    if (!positions || !inv_freq || (Hq && (!q || !q_out)) || (Hk && (!k || !k_out)))
        return fail(GDN_ERR_INVALID, "null pointer");
    rope::Args a{};
    a.x[0] = q; a.x[1] = k; a.y[0] = q_out; a.y[1] = k_out;
    a.sb[0] = q_stride_b; a.st[0] = q_stride_t; a.sh[0] = q_stride_h;
    a.sb[1] = k_stride_b; a.st[1] = k_stride_t; a.sh[1] = k_stride_h;
    a.H[0] = Hq; a.H[1] = Hk;
    a.pos = positions; a.psb = pos_stride_b; a.pst = pos_stride_t; a.pos64 = positions_64 != 0;
    a.inv = inv_freq; a.factor = factor; a.sign = backward ? -1.f : 1.f;
    a.tokens = tokens; a.T = T; a.D = D; a.R = R; a.interleaved = interleaved != 0;
    // channels per load: 16 bytes of 16-bit data where sizes, strides and addresses allow, else 4 channels, else 1
    int V = 8;
    for (; V > 1; V = V == 8 ? 4 : 1) {
        bool ok = R % (2 * V) == 0 && D % V == 0;
        for (int w = 0; w < 2; ++w)
            ok = ok && (!a.H[w] || (a.sb[w] % V == 0 && a.st[w] % V == 0 && a.sh[w] % V == 0 &&
                                    aligned_to(a.x[w], 16) && aligned_to(a.y[w], 16)));
        if (ok) break;
    }
    a.units = R / (2 * V) + (D - R + 2 * V - 1) / (2 * V);
    a.lanes = 1;
    while (a.lanes < a.units && a.lanes < 64) a.lanes *= 2;
    a.tok = tokens >= 2048 ? rope::MAX_TOK : 1;  // few tokens: a workgroup each, to fill 256 CUs several times over
    const int64_t blocks = (tokens + a.tok - 1) / a.tok;
    if (blocks > 0x7fffffff) return fail(GDN_ERR_UNSUPPORTED, "too many tokens");
    const size_t lds = (size_t)a.tok * (R / 2) * sizeof(float2);
    hipStream_t st = static_cast<hipStream_t>(stream);
    {
        Timed tm("rotary", st);
        const dim3 grid = grid_of(blocks), block(rope::NT);
#define GDN_ROTARY(DT)                                                                                      \
    if (V == 8) hipLaunchKernelGGL((rope::rotary_kernel<8, DT>), grid, block, lds, st, a);                   \
    else if (V == 4) hipLaunchKernelGGL((rope::rotary_kernel<4, DT>), grid, block, lds, st, a);              \
    else hipLaunchKernelGGL((rope::rotary_kernel<1, DT>), grid, block, lds, st, a)
        if (dtype == GDN_BF16) { GDN_ROTARY(DT_BF16); }
        else if (dtype == GDN_F32) { GDN_ROTARY(DT_F32); }
        else { GDN_ROTARY(DT_F16); }
#undef GDN_ROTARY
    }
    return check_launch(st, "gdn_rotary");
}
