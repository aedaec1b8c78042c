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
// sums without cancellation.  c comes by a chain, from D, the product <dS, S> of the states between two chunks: c = D - sum b of
// the chunk before it, c = D - sum a of the chunk after it, and D goes on as c + sum a backwards, c + sum b forwards.  Rounding
// errors of a chain stay while what they belong to fades, so every few chunks (mark_of) DQ leaves its state and DK multiplies
// its own with it: a chain runs at most that far, wherever the sequence is cut, and from the end whose terms are smaller.
// Through a chunk whose decay is below the errors of a and b nothing is passed on: c = 0.
// So one kernel, pass_kernel, computes all four.  Where there are few heads, the sequence is cut into segments: seg_kernel
// sums each segment's state from nothing, scan_kernel joins them to the states entering each segment, and the passes run all
// segments at once.
//
// Inputs in bf16 use v_mfma_f32_16x16x32_bf16, whose operands q, k, v and dy are exact; fp32 and fp16 inputs are held as fp32
// and use v_mfma_f32_16x16x4_f32.  Sums and states are fp32, decays' sums fp64.  What bf16 rounds besides is split into terms:
//   P and the state as operands of outputs and gradients, and of a and b, which a chain subtracts: two (2^-17).  In one term (2^-8)
//     Y and DV of 4 sequences of 4096 tokens were 1.4 times as far from 64 bits as sums of 32 bits rounded once, short ones up
//     to 1.6 times, now 1.0, for 6 % of a training step's time and 7 % of a prompt's;
//   e^{G_C - G_s} v_s: three (2^-26), as the final state is an fp32 output.
//
// What bounds the passes is the issue of instructions and the waits between them, not memory: 4 sequences of 4096 tokens, 16
// key and 32 value heads of 128 channels, bf16: Y 179 us, DQ 210, DK 217, DV 213, a segment sum 66 to 70 (medians of one run on
// one card; its shortest launches, and other cards, take 10 to 15 % less), for 0.3 to 0.6 GB of traffic each (60 to 110 us at the
// card's copy rate).  In a chunk of Y a wave has 200 matrix instructions of 16 cycles and some 970 vector instructions (decays,
// P, the state and V' split into bf16 terms, tiles to LDS), which take the SIMD's time one after the other.  Of the passes' wave
// cycles 27 to 36 % wait for an instruction's issue (SQ_WAIT_INST_ANY) and 24 to 40 % for anything else, loads, LDS or barriers,
// which no counter tells apart (SQ_WAIT_ANY); matrix units are busy 24 to 29 %.  Measured along the way, when P and the state of Y
// and DV were rounded to one term: loads under branches, each waited for where it stands, and one workgroup to a CU: Y 295 us, DQ
// 367.  LDS rows padded instead of permuted (three times the conflicts) and X loaded behind the next tiles: DQ 269, DV 245.  P in
// sixteen blocks instead of the twelve that count, weights formed ahead of all products instead of between them, and a chunk's
// loads all at one place: Y 161, DQ 208, DV 203, and without them 155, 186, 190.
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
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16;
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));

// x, unknown to the compiler from here on.
__device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

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

// A tile [rows][W] in LDS.  fp32 rows are padded by 16 bytes.  bf16 rows are not, their 16-byte chunks are permuted: chunk c of
// row r lies at c ^ swz(r), so that the 16 lanes of one cycle of a 16-byte read (0-3, 12-15, 20-23 and 24-27, ...) and the 4
// rows by 4 chunks of a transposing read lie in different banks.  swz depends on r mod 16 only and x, a multiple of 32 columns,
// enters by exclusive or: an offset is (lane part ^ x) + rows.
template <typename ET, int W>
struct Lds {
    static constexpr bool F32 = std::is_same_v<ET, float>;
    static constexpr int LD = W + (F32 ? 4 : 0);
    static __device__ __forceinline__ int quad(int r) {
        const int q = (r >> 2) & 3;
        return ((q ^ (q << 1)) & 2) | (q >> 1);  // 0, 2, 3, 1
    }
    static __device__ __forceinline__ int swz(int r) {
        const int low = quad(r);
        return W == 64 ? ((r & 2) << 1) | low : ((r & 3) << 2) | low;
    }
    static __device__ __forceinline__ int add(int o, int x) { return F32 ? o + x : o ^ x; }
    // 8 columns from c on, c a multiple of 8
    static __device__ __forceinline__ int at8(int r, int c) { return F32 ? r * LD + c : r * W + (c ^ (swz(r) << 3)); }
    // 4 columns from c on, c a multiple of 4
    static __device__ __forceinline__ int at4(int r, int c) { return F32 ? r * LD + c : r * W + (c ^ (swz(r) << 3)); }
    // the operand whose summed axis is contiguous: row li, 8 columns 8 g on of 32
    static __device__ __forceinline__ int row_lane(int li, int g) { return at8(li, 8 * g); }
    // the operand whose summed axis runs down the rows: what col_frag takes, for quads of columns CS apart
    template <int CS>
    static __device__ __forceinline__ int col_lane(int li, int g) {
        if constexpr (F32) return 8 * g * LD + (li >> 2) * CS + (li & 3);
        else return at4(8 * g + (li >> 2), (li & 3) * CS);
    }
};

// Row r0 (a multiple of 16) + the lane's, columns x (of 32) on.
template <typename L>
__device__ __forceinline__ bf8 row_frag(const bf16 *t, int lane, int r0, int x) {
    return *reinterpret_cast<const bf8 *>(t + L::add(lane, x) + r0 * L::LD);
}
template <typename L>
__device__ __forceinline__ F32Frag row_frag(const float *t, int lane, int r0, int x) {
    const float *p = t + L::add(lane, x) + r0 * L::LD;
    F32Frag f;
    const f4 a = *reinterpret_cast<const f4 *>(p), b = *reinterpret_cast<const f4 *>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f.v[j] = a[j];
        f.v[4 + j] = b[j];
    }
    return f;
}

// Rows k0 (of 32) on: lane 4 c + i of 16 holds column x + c CS + i (+ half, 0 or 4).  bf16: the LDS's transposing read, where
// the four lanes 4 j .. 4 j + 3 of 16 give the addresses of row j's four quads of columns and lane 4 c + i receives column i of
// quad c, rows 0 to 3; rows 4 on are a second read (their swz differs by 2).
template <typename L>
__device__ __forceinline__ bf8 col_frag(const bf16 *t, int lane, int k0, int x, int half) {
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const int o = L::add(lane, x);
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(t + o + k0 * L::LD + half));
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(t + (o ^ 16) + (k0 + 4) * L::LD + half));
    return __builtin_bit_cast(bf8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
template <typename L>
__device__ __forceinline__ F32Frag col_frag(const float *t, int lane, int k0, int x, int half) {
    const float *p = t + lane + x + half + k0 * L::LD;
    F32Frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = p[j * L::LD];
    return f;
}

// P in LDS, [outputs][sources].  fp32: a tile of C columns.  bf16: two terms of every element, of the six pieces of 16 outputs by
// 32 sources that hold pairs (whole tiles would leave no room for DV's second workgroup).  A term of a piece is 1 KB, its 16-byte
// chunks permuted so that reads of an operand and writes of a block of products meet no conflict.
template <typename ET, bool REV>
struct Pairs {
    static constexpr bool F32 = std::is_same_v<ET, float>;
    using L = Lds<ET, C>;
    static constexpr int TERMS = F32 ? 1 : 2, TERM = 512, SIZE = F32 ? C * L::LD : 6 * TERMS * TERM;
    // where the piece of outputs r0 (a multiple of 16) and sources s0 (of 32) begins
    static __device__ __forceinline__ int piece(int r0, int s0) {
        const int r = r0 >> 4;
        return ((s0 >> 5) == (REV ? 1 : 0) ? r : REV ? 4 + r : 2 + r) * TERMS * TERM;
    }
    // 4 sources from s on, a multiple of 4
    static __device__ __forceinline__ int at(int r, int s) {
        if constexpr (F32) return L::at4(r, s);
        else return piece(r & ~15, s & ~31) + (r & 15) * 32 + ((((s >> 3) & 3) ^ L::quad(r)) << 3) + (s & 7);
    }
    // the operand: row li, sources 8 g on
    static __device__ __forceinline__ int lane(int li, int g) {
        return F32 ? L::row_lane(li, g) : li * 32 + ((g ^ L::quad(li)) << 3);
    }
    static __device__ __forceinline__ Frag<ET> frag(const ET *p, int lane, int r0, int s0, int term) {
        if constexpr (F32) return row_frag<L>(p, lane, r0, s0);
        else return *reinterpret_cast<const bf8 *>(p + piece(r0, s0) + term * TERM + lane);
    }
};

// Two numbers rounded to bf16 by one instruction, and back.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, b2));
}
__device__ __forceinline__ float low_bf16(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high_bf16(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// x as the sum of N operands (fp32: itself).
template <int N>
__device__ __forceinline__ void split(const float (&x)[8], bf8 (&o)[N]) {
    u4 u[N];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a = x[2 * j], b = x[2 * j + 1];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            u[n][j] = pack_bf16(a, b);
            if (n + 1 < N) {
                a -= low_bf16(u[n][j]);
                b -= high_bf16(u[n][j]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) o[n] = __builtin_bit_cast(bf8, u[n]);
}
template <int N>
__device__ __forceinline__ void split(const float (&x)[8], F32Frag (&o)[N]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[0].v[j] = x[j];
}
// A tensor [B][T][heads][D], channels contiguous; value head h reads head h / div.
struct Ten {
    const void *p;
    int64_t sb, st, sh;
    int div;
    __device__ __forceinline__ int64_t at(int b, int64_t t, int h) const { return b * sb + t * st + (h / div) * sh; }
    template <typename ET>
    __device__ __forceinline__ const char *from(int b, int64_t t, int h, int c, int dt) const {
        return static_cast<const char *>(p) + (at(b, t, h) + c) * (std::is_same_v<ET, float> && dt == DT_F32 ? 4 : 2);
    }
};

// 16 bytes from an address that is a multiple of the element's size only
struct __attribute__((packed, aligned(2))) u4_any {
    u4 v;
};

// A [C][W] tile in registers on its way from memory to LDS, 8 channels to a piece, by N threads; rows >= n and columns >= w are
// zero.  VEC: w is a multiple of 8 (or none is left), pieces are loaded whole.  No load stands under a branch, where it would be waited
// for: rows and columns out of range load ones in range, and turn to zeros on the way to LDS.
template <typename ET, int W, bool VEC, int N = NT>
struct Tile {
    static constexpr bool F32 = std::is_same_v<ET, float>;
    static constexpr int PER = C * W / 8 / N, STEP = N / (W / 8);
    static_assert(PER * N * 8 == C * W, "a tile splits evenly");
    u4 x[PER][F32 ? 2 : 1];
    // t0: the tile's first row and channel; dt: its type; st: elements between rows
    __device__ __forceinline__ void fetch(const char *t0, int64_t st, int n, int w, int dt) {
        const int tid = opaque(threadIdx.x) & (N - 1), r0 = tid / (W / 8), c0 = (tid % (W / 8)) * 8;
        const unsigned size = F32 && dt == DT_F32 ? 4 : 2, row = (unsigned)st * size;
        if constexpr (VEC) {
            const unsigned c = (c0 < w ? c0 : 0) * size;
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                const char *s = t0 + (__umul24(min(r0 + p * STEP, n - 1), row) + c);
                x[p][0] = reinterpret_cast<const u4_any *>(s)->v;
                if constexpr (F32) x[p][1] = reinterpret_cast<const u4_any *>(s + (dt == DT_F32 ? 16 : 0))->v;
            }
        } else {
#pragma unroll
            for (int p = 0; p < PER; ++p) {
                const unsigned at = __umul24(min(r0 + p * STEP, n - 1), (unsigned)st);
                u4 y[2] = {};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const unsigned i = at + (c0 + j < w ? c0 + j : 0);
                    if (F32 && dt == DT_F32) {
                        const uint32_t v = reinterpret_cast<const uint32_t *>(t0)[i];
                        y[j / 4][j % 4] = c0 + j < w ? v : 0;
                    } else {
                        const uint32_t v = reinterpret_cast<const uint16_t *>(t0)[i];
                        y[0][j / 2] |= (c0 + j < w ? v : 0) << (16 * (j & 1));
                    }
                }
                x[p][0] = y[0];
                if constexpr (F32) x[p][1] = y[1];
            }
        }
    }
    __device__ __forceinline__ void store(ET *dst, int n, int w, int dt) const {
        if (n == C && w >= W) store_as<true>(dst, n, w, dt);
        else store_as<false>(dst, n, w, dt);
    }
    template <bool FULL>
    __device__ __forceinline__ void store_as(ET *dst, int n, int w, int dt) const {
        const int tid = opaque(threadIdx.x) & (N - 1), r0 = tid / (W / 8), c0 = (tid % (W / 8)) * 8;
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int r = r0 + p * STEP;
            // STEP rows on the permutation is the same where STEP is a multiple of 16
            ET *d = dst + (STEP % 16 == 0 ? Lds<ET, W>::at8(r0, c0) + p * STEP * Lds<ET, W>::LD : Lds<ET, W>::at8(r, c0));
            const bool in = FULL || (r < n && c0 < w);
            u4 a = x[p][0];
            if constexpr (F32) {
                u4 b = x[p][1];
                if (dt != DT_F32) {
                    const u4 h = a;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        a[j] = __float_as_uint(ops::half_bits_to_f32(h[j / 2] >> (16 * (j & 1))));
                        b[j] = __float_as_uint(ops::half_bits_to_f32(h[2 + j / 2] >> (16 * (j & 1))));
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = in ? b[j] : 0;
                *reinterpret_cast<u4 *>(d + 4) = b;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = in ? a[j] : 0;
            *reinterpret_cast<u4 *>(d) = a;
        }
    }
};

// 4 or 8 channels from element i on, at any alignment, in 16 bits or (two pieces a 4) fp32.
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
struct __attribute__((packed, aligned(2))) u2_any {
    u2 v;
};
template <int N, typename ET>
__device__ __forceinline__ void store_row(char *p, unsigned i, int dt, const float (&o)[N]) {
    if (dt == DT_F32) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const u4 a = {__float_as_uint(o[j]), __float_as_uint(o[j + 1]), __float_as_uint(o[j + 2]), __float_as_uint(o[j + 3])};
            reinterpret_cast<u4_any *>(p + 4 * (i + j))->v = a;
        }
    } else {
        uint32_t u[N / 2];
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            if constexpr (std::is_same_v<ET, bf16>) u[j] = pack_bf16(o[2 * j], o[2 * j + 1]);
            else u[j] = ops::pack2(o[2 * j], o[2 * j + 1], DT_F16);
        }
        if constexpr (N == 8) reinterpret_cast<u4_any *>(p + 2 * i)->v = u4{u[0], u[1], u[2], u[3]};
        else reinterpret_cast<u2_any *>(p + 2 * i)->v = u2{u[0], u[1]};
    }
}

// N channels of a row on their way to a sum: raw bits, turned to fp32 where they are used.
template <int N, typename ET, bool VEC>
struct Piece {
    static constexpr bool F32 = std::is_same_v<ET, float>;
    uint32_t u[F32 ? N : N / 2];
    // p: the tensor's type dt; elements from i on, w of them left
    __device__ __forceinline__ void fetch(const char *p, unsigned i, int w, int dt) {
        if constexpr (VEC) {
            const char *q = p + (w > 0 ? i : 0) * (F32 && dt == DT_F32 ? 4 : 2);
            if (N == 4 && !(F32 && dt == DT_F32)) {
                const u2 a = reinterpret_cast<const u2_any *>(q)->v;
                u[0] = a[0];
                u[1] = a[1];
            } else {
#pragma unroll
                for (int j = 0; j < (int)(sizeof(u) / 16); ++j) {
                    const u4 a = reinterpret_cast<const u4_any *>(q + (F32 && dt != DT_F32 ? 0 : 16 * j))->v;
#pragma unroll
                    for (int k = 0; k < 4; ++k) u[4 * j + k] = a[k];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const unsigned e = j < w ? i + j : 0;
                uint32_t v;
                if (F32 && dt == DT_F32) v = reinterpret_cast<const uint32_t *>(p)[e];
                else v = reinterpret_cast<const uint16_t *>(p)[e];
                if constexpr (F32) u[j] = v;
                else u[j / 2] = j & 1 ? u[j / 2] | (v << 16) : v;
            }
        }
    }
    __device__ __forceinline__ float get(int j, int dt) const {
        if constexpr (!F32) return __uint_as_float(j & 1 ? u[j / 2] & 0xffff0000u : u[j / 2] << 16);
        else if (dt == DT_F32) return __uint_as_float(u[j]);
        else return ops::half_bits_to_f32(VEC ? u[j / 2] >> (16 * (j & 1)) : u[j]);
    }
};

struct Gate {
    const void *p;
    int64_t sb, st, sh;
    int dt;
    // log decays below -1e4 (-inf: nothing is kept) run as -1e4, whose exponential is 0 and whose differences are finite
    __device__ __forceinline__ uint32_t fetch(int b, int64_t t, int h) const {
        const int64_t i = b * sb + t * st + h * sh;
        return dt == DT_F32 ? static_cast<const uint32_t *>(p)[i] : (uint32_t) static_cast<const uint16_t *>(p)[i];
    }
    __device__ __forceinline__ float value(uint32_t u) const {
        const float g = dt == DT_F32 ? __uint_as_float(u) : dt == DT_BF16 ? __uint_as_float(u << 16) : ops::half_bits_to_f32(u);
        return g < -1e4f ? -1e4f : g;
    }
    __device__ __forceinline__ float load(int b, int64_t t, int h) const { return value(fetch(b, t, h)); }
};

// Of one chunk, as decay_kernel writes them, 256 floats: G as powers of two, in two terms (differences hold where sums are
// large), e^{G_r}, and e^{G_C - G_s}.
struct Decays {
    float2 G[C];
    float in[C], out[C];
};
constexpr int DECAYS = sizeof(Decays) / sizeof(float);
static_assert(DECAYS == NT, "one float to a thread");

enum Kind { Y, DQ, DK, DV };  // what a pass computes

// Chunks between two products of the states.  Eight: 512 KB of states for 4096 tokens of a head of 128 x 128; four take 2.4 % of
// a bf16 step's time, whose a and b have 17 bits.  fp32 and fp16 inputs, whose a and b have more, take four: one decay for a
// head of 2047 tokens is 5e-7 off (8e-7 with eight; 32-bit chunks in plain form 7e-7), for 0.7 % of the time.
constexpr int mark_of(bool f32) { return f32 ? 4 : 8; }

struct Pass {
    Ten Q, K, V, X;
    const float *decays;  // [B][Hv][nc][DECAYS]
    const float *s_in;  // states entering the segments, head (b, h) at s_in + (b Hv + h) s_head, segment j at + j s_seg; or NULL
    float *s_out;       // the state leaving the last segment (reverse: the first), [B][Hv][..], or NULL
    int64_t s_head, s_seg;
    int s_t;            // states are [v'][k'] (0) or [k'][v'] (1)
    void *o;            // [B][T][heads][dv] contiguous
    float *marks;       // DQ writes, DK reads: the states entering every mark_of() chunks, from the first on, as the lanes hold
                        // them, [B][Hv][nm][slices][D / 16][NV][64 NW][4]
    double *ends;       // DK: their products with the cotangents there, [B][Hv][nm][slices][NW], a wave's part each
    int nm, mark0;      // marks of the sequence; the first that is taken (1 where the state before the first token is zero)
    float *dot;         // per token [slices][B][Hv][T]: DQ, DK X . (O from the state); DV the pairs that cross it, X = v
    int B, T, Hv, dk, dv, slices, nseg, cps, nc;  // cps: chunks of a segment, nc: of the sequence
    int dt, o_dt, pair;  // pair: two heads to a workgroup, whose outputs are added
    float scale;
};

// fp32 tiles of 256 channels leave no room for P and X, which then take the place of Q' once that is used.
template <typename ET, int D>
constexpr bool p_over_q() { return std::is_same_v<ET, float> && D > 128; }

// G: heads to a workgroup, NW waves each, that share V'.
template <typename ET, int D, int NV, int NW, int KIND, int G>
struct Shared {
    using LK = Lds<ET, D>;        // tiles Q' and K'
    using LV = Lds<ET, 16 * NV * NW>;  // V' and X
    using P = Pairs<ET, (KIND >= DK)>;
    static constexpr bool TAKEN = p_over_q<ET, D>(), DOT = KIND == DQ || KIND == DK;
    static constexpr int SUM = 4 * NV * 64 * NW;  // float4s of a head's outputs
    ET Q[G][C * LK::LD], K[G][C * LK::LD], V[C * LV::LD];
    ET own_p[G][TAKEN ? 8 : P::SIZE], own_x[KIND == DV && !TAKEN ? C * LV::LD : 8];
    Decays d[G];
    float total[G], dot[DOT ? G : 1][DOT ? NW : 1][DOT ? C : 1];
    static constexpr bool SUM_OVER_Q = SUM * sizeof(float4) <= G * C * LK::LD * sizeof(ET);
    float4 own_sum[G == 2 && !SUM_OVER_Q ? SUM : 1];
    // where Q' was, once it is used: the waves' sums of M for each token, [NW][C]
    using Cross = std::conditional_t<std::is_same_v<ET, float>, double, float>;
    __device__ __forceinline__ Cross *cross() { return reinterpret_cast<Cross *>(Q[0] + (TAKEN ? P::SIZE + C * LV::LD : 0)); }
    __device__ __forceinline__ ET *p(int i) { return TAKEN ? Q[0] : own_p[i]; }
    __device__ __forceinline__ ET *x() { return TAKEN ? Q[0] + P::SIZE : own_x; }
    __device__ __forceinline__ float4 *sum() { return SUM_OVER_Q ? reinterpret_cast<float4 *>(Q[0]) : own_sum; }
};

// 32 rows of a wave's V', and the same times their weights in NS terms, worked out two elements of a lane at a time: PARTS
// parts, to stand between matrix products, which leave the vector unit 12 of their 16 cycles.
template <typename ET, int NV, int NS>
struct Weighted {
    static constexpr int PARTS = 4 * NV;
    static constexpr bool F32 = std::is_same_v<ET, float>;
    Frag<ET> v[NV];
    std::conditional_t<F32, F32Frag, u4> t[NV][NS];
    float w[8];
    __device__ __forceinline__ Frag<ET> term(int x, int n) const { return __builtin_bit_cast(Frag<ET>, t[x][n]); }
    template <typename L>
    __device__ __forceinline__ void read(const ET *sV, int lane, int k0, int x0, const float *weights) {
#pragma unroll
        for (int x = 0; x < NV; ++x) v[x] = col_frag<L>(sV, lane, k0, x0, 4 * x);
        const f4 a = *reinterpret_cast<const f4 *>(weights), b = *reinterpret_cast<const f4 *>(weights + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = a[j];
            w[4 + j] = b[j];
        }
    }
    __device__ __forceinline__ void part(int i) {
        const int x = i / 4, j = 2 * (i % 4);
        if constexpr (F32) {
            t[x][0].v[j] = v[x].v[j] * w[j];
            t[x][0].v[j + 1] = v[x].v[j + 1] * w[j + 1];
        } else {
            const uint32_t u = __builtin_bit_cast(u4, v[x])[j / 2];
            float a = low_bf16(u) * w[j], b = high_bf16(u) * w[j + 1];
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                const uint32_t h = pack_bf16(a, b);
                t[x][n][j / 2] = h;
                a -= low_bf16(h);
                b -= high_bf16(h);
            }
        }
    }
    __device__ __forceinline__ void all() {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) part(i);
    }
};

// The state of a wave: K' rows 32 T + 8 (l / 16) + 4 (t & 1) + e of tile t = 2 T, 2 T + 1 by its columns 16 NV w + ...: what
// lane l holds of two tiles is 8 consecutive K' rows of one column, an operand as it stands.
template <int D, int NV, int NW>
struct State {
    f4 s[D / 16][NV];
    // the lane's column of tile n
    static __device__ __forceinline__ int col(int n) {
        const int l = threadIdx.x & 63, li = l & 15, w = (threadIdx.x >> 6) & (NW - 1);
        return 16 * NV * w + 4 * NV * (li >> 2) + 4 * n + (li & 3);
    }
    // p: [v'][k'], or with tr [k'][v']; out of range (and without p) zeros
    __device__ __forceinline__ void load(const float *p, int dk, int dv, int c0, int tr) {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int T = 0; T < D / 32; ++T)
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int k = 32 * T + 8 * g, v = c0 + col(n), vv = min(v, dv - 1);
                float x[8] = {};
                if (p) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int kk = min(k + e, dk - 1);
                        x[e] = p[tr ? kk * dv + vv : vv * dk + kk];
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) s[2 * T + e / 4][n][e % 4] = k + e < dk && v < dv ? x[e] : 0.f;
            }
    }
    __device__ __forceinline__ void store(float *p, int dk, int dv, int c0, int tr) const {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int T = 0; T < D / 32; ++T)
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int k = 32 * T + 8 * g, v = c0 + col(n);
                if (v >= dv) continue;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (k + e < dk) p[tr ? (k + e) * dv + v : v * dk + k + e] = s[2 * T + e / 4][n][e % 4];
            }
    }
    // the state as the lanes hold it, lane `tid` of the head's
    __device__ __forceinline__ void put(float *p, int tid) const {
        f4 *const m = reinterpret_cast<f4 *>(p) + tid;
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int n = 0; n < NV; ++n) m[(t * NV + n) * 64 * NW] = s[t][n];
    }
    // the lane's part of the product with a state put there, a few loads at a time (registers)
    __device__ __forceinline__ double product(const float *p, int tid) const {
        const f4 *const m = reinterpret_cast<const f4 *>(p) + tid;
        constexpr int STEP = 4 / NV;
        double x = 0.;
#pragma unroll
        for (int t0 = 0; t0 < D / 16; t0 += STEP) {
            f4 y[STEP][NV];
#pragma unroll
            for (int t = 0; t < STEP; ++t)
#pragma unroll
                for (int n = 0; n < NV; ++n) y[t][n] = m[((t0 + t) * NV + n) * 64 * NW];
#pragma unroll
            for (int t = 0; t < STEP; ++t)
#pragma unroll
                for (int n = 0; n < NV; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x = fma((double)s[t0 + t][n][e], (double)y[t][n][e], x);
            __builtin_amdgcn_sched_barrier(0);
        }
        return x;
    }
    // s += K'^T diag(weights) V' over 32 rows, tile by tile, between(t) behind the products of each
    template <int NS, typename ET, typename F>
    __device__ __forceinline__ void add(const ET *sK, int lane, int k0, const Weighted<ET, NV, NS> &v, F between) {
        Frag<ET> a = col_frag<Lds<ET, D>>(sK, lane, k0, 0, 0);
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
            Frag<ET> next = a;
            if (t + 1 < D / 16) next = col_frag<Lds<ET, D>>(sK, lane, k0, 32 * ((t + 1) >> 1), 4 * ((t + 1) & 1));
#pragma unroll
            for (int i = 0; i < NS; ++i)
#pragma unroll
                for (int n = 0; n < NV; ++n) s[t][n] = mma(a, v.term(n, i), s[t][n]);
            between(t);
            if constexpr (NS == 3) __builtin_amdgcn_sched_barrier(0);
            a = next;
        }
    }
    __device__ __forceinline__ void scale(int t, float f) {
#pragma unroll
        for (int n = 0; n < NV; ++n) s[t][n] *= f;
    }
};

// The e-th of twelve 16 x 16 blocks of P, its first output and source: the ten that hold pairs, and two that fill the products'
// 32 sources with zeros.  Blocks 0-7 are the four of two outputs (for the last of them all sources count; reverse: the first),
// so that a wave's blocks e and e + 4 share their sources.
struct Block {
    int r0, s0;
};
template <bool REV>
__device__ __forceinline__ Block block(int e) {
    const int r = e < 8 ? 2 + (e >> 2) : (e >> 1) & 1, s = e < 8 ? e & 3 : e & 1;
    return REV ? Block{48 - 16 * r, 48 - 16 * s} : Block{16 * r, 16 * s};
}

// Workgroups go to the 8 XCDs in turn, each with its own L2: an order in which neighbours, the heads that share a key head,
// stay on one.
__device__ __forceinline__ int xcd_order(int i, int n) { return n % 8 == 0 ? (i % 8) * (n / 8) + i / 8 : i; }

// The sum over 16 lanes.
__device__ __forceinline__ float sum16(float x) { return row16_allreduce(x); }
__device__ __forceinline__ double sum16(double x) {
    x += dpp_mov_f64<DPP_QUAD_1032>(x);
    x += dpp_mov_f64<DPP_QUAD_2301>(x);
    x += dpp_mov_f64<DPP_ROW_HALF_MIRROR>(x);
    return x + dpp_mov_f64<DPP_ROW_MIRROR>(x);
}
// Lane i of 16 receives lane i - 1 (lane 0: 0); the sum over the lanes up to its own.
__device__ __forceinline__ float row_shr1(float x) { return dpp_mov<0x111>(x); }
__device__ __forceinline__ double row_shr1(double x) { return dpp_mov_f64<0x111>(x); }
__device__ __forceinline__ float prefix16(float x) {
    x += dpp_mov<0x111>(x);
    x += dpp_mov<0x112>(x);
    x += dpp_mov<0x114>(x);
    return x + dpp_mov<0x118>(x);
}
__device__ __forceinline__ double prefix16(double x) {
    x += dpp_mov_f64<0x111>(x);
    x += dpp_mov_f64<0x112>(x);
    x += dpp_mov_f64<0x114>(x);
    return x + dpp_mov_f64<0x118>(x);
}
__device__ __forceinline__ float xor16(float x) { return lane_xor16(x); }
__device__ __forceinline__ float xor32(float x) { return lane_xor32(x); }
__device__ __forceinline__ double xor16(double x) { return __shfl_xor(x, 16); }
__device__ __forceinline__ double xor32(double x) { return __shfl_xor(x, 32); }

// Waves to a SIMD that the registers have to allow.
template <typename ET, int D>
constexpr int waves() { return std::is_same_v<ET, bf16> && D <= 128 ? 2 : 1; }

// One segment of G value heads, 16 NV NW columns of V'.  The state stays in the accumulators of the products that sum it, laid
// out so that it is an operand of the next chunk's O as it stands; tiles pass once from memory through registers, a chunk
// ahead, to LDS.  32 columns to a wave: every operand read from LDS serves two products (state, V') or is shared by all waves
// (P).  O is formed transposed, so that a lane stores consecutive channels.
template <typename ET, int D, int NV, int NW, int KIND, int G, bool VEC>
__global__ __launch_bounds__(64 * NW * G, (waves<ET, D>())) void pass_kernel(const Pass a) {
    constexpr bool F32 = std::is_same_v<ET, float>, REV = KIND >= DK, DOT = KIND == DQ || KIND == DK;
    constexpr int NS = F32 ? 1 : 3, NH = F32 ? 1 : 2;  // terms of the weighted V', of the state as an operand
    constexpr int RT = C / 16;
    using LK = Lds<ET, D>;
    using LV = Lds<ET, 16 * NV * NW>;
    using P = Pairs<ET, REV>;
    constexpr bool TAKEN = Shared<ET, D, NV, NW, KIND, G>::TAKEN;
    __shared__ __attribute__((aligned(16))) Shared<ET, D, NV, NW, KIND, G> sh;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & (NW - 1), grp = wave / NW;
    int id = xcd_order(blockIdx.x, gridDim.x);
    const int slice = id % a.slices;
    id /= a.slices;
    const int hg = id % (a.Hv / G), h = hg * G + grp;
    id /= a.Hv / G;
    const int b = id % a.B, seg = id / a.B, c0 = slice * 16 * NV * NW;
    const int first = seg * a.cps, last = min(a.nc, first + a.cps) - 1;
    const int64_t head = (int64_t)b * a.Hv + h;

    State<D, NV, NW> S;
    S.load(a.s_in ? a.s_in + head * a.s_head + seg * a.s_seg : nullptr, a.dk, a.dv, c0, a.s_t);

    Tile<ET, D, VEC, 64 * NW> tq, tk;
    Tile<ET, 16 * NV * NW, VEC, 64 * NW * G> tv;
    Tile<ET, 16 * NV * NW, VEC, 64 * NW> tx;
    float td = 0.f;
    // the next chunk's tiles, one by one between the phases of this one
    const auto fetch = [&](int c, int part) {
        const int64_t t0 = (int64_t)c * C;
        const int n = min((int64_t)C, a.T - t0);
        if (part == 0) {
            tq.fetch(a.Q.template from<ET>(b, t0, h, 0, a.dt), a.Q.st, n, a.dk, a.dt);
            td = a.decays[(head * a.nc + c) * DECAYS + (threadIdx.x & (NT - 1))];
        } else if (part == 1) {
            tk.fetch(a.K.template from<ET>(b, t0, h, 0, a.dt), a.K.st, n, a.dk, a.dt);
        } else {
            tv.fetch(a.V.template from<ET>(b, t0, h, c0, a.dt), a.V.st, n, a.dv - c0, a.dt);
        }
    };
    Piece<4 * NV, ET, VEC> px[RT];
    const auto fetch_x = [&](int c) {
        const int64_t t0 = (int64_t)c * C;
        const int n = min((int64_t)C, a.T - t0);
        const char *x0 = a.X.template from<ET>(b, t0, h, 0, a.dt);
        const int l = opaque(threadIdx.x & 63), li = l & 15, col = c0 + 16 * NV * w + 4 * NV * (l >> 4);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
            px[rt].fetch(x0, __umul24(min(16 * rt + li, n - 1), (unsigned)a.X.st) + col, a.dv - col, a.dt);
    };
    for (int part = 0; part < 3; ++part) fetch(REV ? last : first, part);
    for (int i = first; i <= last; ++i) {
        const int c = REV ? first + last - i : i;
        const int64_t t0 = (int64_t)c * C;
        const int n = min((int64_t)C, a.T - t0);
        // opaque: addresses in LDS are formed where they are used, not hoisted out of the loop and spilled
        const int tid = opaque(threadIdx.x), l = tid & 63, li = l & 15, g = l >> 4;
        const int col = c0 + 16 * NV * w + 4 * NV * g;  // the lane's first column of O
        constexpr int M = mark_of(F32);
        const bool marked = DOT && c % M == 0 && c / M >= a.mark0;
        const int64_t mark = marked ? (head * a.nm + c / M) * a.slices + slice : 0;
        if constexpr (KIND == DQ) {
            if (marked) S.put(a.marks + mark * (D * 16 * NV * NW), w * 64 + l);
        }
        __syncthreads();
        tq.store(sh.Q[grp], n, a.dk, a.dt);
        tk.store(sh.K[grp], n, a.dk, a.dt);
        tv.store(sh.V, n, a.dv - c0, a.dt);
        // the scale goes with e^{G_r}: into the outputs, reverse into the sources
        reinterpret_cast<float *>(&sh.d[grp])[tid & (NT - 1)] = (w & 3) == 2 ? td * a.scale : td;
        if (w == 2 && l == C - 1) sh.total[grp] = td;
        __syncthreads();
        // X before the next tiles: loads are waited for in their order
        if constexpr (DOT) fetch_x(c);
        if constexpr (KIND == DV) tx.fetch(a.X.template from<ET>(b, t0, h, c0, a.dt), a.X.st, n, a.dv - c0, a.dt);
        const int after = REV ? c - 1 : c + 1;
        if (i < last) fetch(after, 0);

        // O = diag(wo) S Q'^T, later + P V', transposed: a lane holds one token, 4 NV consecutive columns
        const int lk = LK::row_lane(li, g);
        f4 O[RT][NV];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int x = 0; x < NV; ++x) O[rt][x] = f4{0.f, 0.f, 0.f, 0.f};
        const int lvc = LV::template col_lane<4 * NV>(li, g);
        const float *const weights = (REV ? sh.d[grp].in : sh.d[grp].out) + 8 * g;
        Weighted<ET, NV, NS> v;
        v.template read<LV>(sh.V, lvc, 0, 16 * NV * w, weights);
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
                const Frag<ET> q = row_frag<LK>(sh.Q[grp], lk, 16 * rt, 32 * T);
#pragma unroll
                for (int j = 0; j < NH; ++j)
#pragma unroll
                    for (int x = 0; x < NV; ++x) O[rt][x] = mma(f[x][j], q, O[rt][x]);
            }
#pragma unroll
            for (int i = T * v.PARTS * 32 / D; i < (T + 1) * v.PARTS * 32 / D; ++i) v.part(i);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float wo = (REV ? sh.d[grp].out : sh.d[grp].in)[16 * rt + li];
#pragma unroll
            for (int x = 0; x < NV; ++x) O[rt][x] *= wo;
        }
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
#pragma unroll
                for (int j = 0; j < 4 * NV; ++j) s = fmaf(col + j < a.dv ? px[rt].get(j, a.dt) : 0.f, o[j], s);
                s = r < n ? s : 0.f;
                s += lane_xor16(s);
                s += lane_xor32(s);
                if (g == 0) sh.dot[grp][w][r] = s;
            }
        }

        if (i < last) fetch(after, 1);
        // P: its blocks to the waves in turn
        ET *const sP = sh.p(grp);
        constexpr int BLOCKS = (12 + NW - 1) / NW;
        const bool last_block = 12 % NW == 0 || w < 12 % NW;
        f4 acc[BLOCKS] = {};
        float2 gr[BLOCKS], gs[BLOCKS][4];
        const auto read_decays = [&] {
#pragma unroll
            for (int e = 0; e < BLOCKS; ++e) {
                const Block k = block<REV>(w + NW * e);
                gr[e] = sh.d[grp].G[(k.r0 + li) & (C - 1)];
#pragma unroll
                for (int j = 0; j < 4; ++j) gs[e][j] = sh.d[grp].G[(k.s0 + 4 * g + j) & (C - 1)];
            }
        };
        if constexpr (KIND != DV) read_decays();  // ahead of the products; DV has no registers left for it
#pragma unroll
        for (int x = 0; x < D; x += 32)
#pragma unroll
            for (int e = 0; e < BLOCKS; ++e) {
                if (e == BLOCKS - 1 && !last_block) continue;
                const Block k = block<REV>(w + NW * e);
                acc[e] = mma(row_frag<LK>(sh.K[grp], lk, k.s0, x), row_frag<LK>(sh.Q[grp], lk, k.r0, x), acc[e]);
            }
        if constexpr (TAKEN) {
            __syncthreads();
        }
        if constexpr (KIND == DV) tx.store(sh.x(), n, a.dv - c0, a.dt);
        if constexpr (KIND == DV) read_decays();
        const auto put = [&](int r, int s, const f4 &p) {
            ET *o = sP + P::at(r, s);
            if constexpr (F32) {
                *reinterpret_cast<f4 *>(o) = p;
            } else {
                const uint32_t a = pack_bf16(p[0], p[1]), b = pack_bf16(p[2], p[3]);
                *reinterpret_cast<uint2 *>(o) = make_uint2(a, b);
                *reinterpret_cast<uint2 *>(o + P::TERM) = make_uint2(pack_bf16(p[0] - low_bf16(a), p[1] - high_bf16(a)),
                                                                     pack_bf16(p[2] - low_bf16(b), p[3] - high_bf16(b)));
            }
        };
#pragma unroll
        for (int e = 0; e < BLOCKS; ++e) {
            if (e == BLOCKS - 1 && !last_block) continue;
            const Block k = block<REV>(w + NW * e);
            const int r = k.r0 + li, s0 = k.s0 + 4 * g;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float d = (gr[e].x - gs[e][j].x) + (gr[e].y - gs[e][j].y);
                const float x = acc[e][j] * (a.scale * __builtin_amdgcn_exp2f(REV ? -d : d));
                acc[e][j] = (REV ? s0 + j >= r : s0 + j <= r) ? x : 0.f;
            }
            put(r, s0, acc[e]);
        }
        __syncthreads();
        if (i < last) fetch(after, 2);
        // M of the same blocks, and for every token t the sum of the pairs that cross it, an output before t with a source from t
        // on (fp32 inputs: in 64 bits).  Only those are added, none is added and taken away again: what later pairs are, large
        // or NaN, has no part in it.  Lane t of a wave sums its blocks' part.
        if constexpr (KIND == DV) {
            using Cross = typename Shared<ET, D, NV, NW, KIND, G>::Cross;
            const int lv = LV::row_lane(li, g);
            Cross mine = 0;
#pragma unroll
            for (int e = 0; e < BLOCKS; ++e) {
                const Block k = block<REV>(w + NW * e);
                if ((e == BLOCKS - 1 && !last_block) || k.s0 < k.r0) continue;
                f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 16 * NV * NW; i += 32)
                    x = mma(row_frag<LV>(sh.V, lv, k.s0, i), row_frag<LV>(sh.x(), lv, k.r0, i), x);
                const bool diagonal = k.s0 == k.r0;
                // the lane's output (column li) with its sources from each of the lane's four on
                Cross from[4];
#pragma unroll
                for (int j = 3; j >= 0; --j) {
                    const Cross p = (Cross)x[j] * (Cross)acc[e][j];
                    from[j] = (!diagonal || 4 * g + j > li ? p : 0) + (j < 3 ? from[(j + 1) & 3] : 0);
                }
                const Cross beside = xor16(from[0]), two = from[0] + beside, others = xor32(two);
                const Cross after = (g & 1 ? 0 : beside) + (g < 2 ? others : 0);
                // t among the sources: their sums over all outputs (of its own block: those before t)
#pragma unroll
                for (int j = 0; j < 4; ++j) from[j] = sum16(!diagonal || li < 4 * g + j ? from[j] + after : (Cross)0);
                const Cross own = li & 2 ? (li & 1 ? from[3] : from[2]) : (li & 1 ? from[1] : from[0]);
                const Cross sources = __shfl(own, 16 * (li >> 2) + (li & 3));
                // t among the outputs: those before it with all sources; t in a block between: all of both
                const Cross outputs = prefix16(two + others), before = row_shr1(outputs), all = sum16(two + others);
                const int t0 = l & 48;
                mine += t0 == k.s0 ? sources : t0 == k.r0 ? before : t0 > k.r0 && t0 < k.s0 ? all : (Cross)0;
            }
            sh.cross()[w * C + l] = mine;
        }
        const float total = sh.total[grp];
        const int lp = P::lane(li, g), lkc = LK::template col_lane<8>(li, g);
        const auto pairs_of = [&](int k0, const Frag<ET> (&v)[NV]) {
            // an infinite or NaN source of a later token (reverse: an earlier one) must not reach an output through its weight
            // of 0: where a product with zeros shows one, the sum takes the pairs that count one by one (looking costs a pass
            // 1 to 2% of its time)
            f4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < NV; ++x) z = mma(v[x], Frag<ET>{}, z);
            if (__any((z[0] + z[1]) + (z[2] + z[3]) != 0.f)) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll 1
                    for (int s = k0; s < k0 + 32; ++s) {
                        if (REV ? s < 16 * rt + li : s > 16 * rt + li) continue;
                        const ET *const ps = sP + P::at(16 * rt + li, s & ~3) + (s & 3);
                        const float p = F32 ? (float)ps[0] : (float)ps[0] + (float)ps[P::TERM];
                        const ET *const vs = sh.V + LV::at4(s, col - c0);
#pragma unroll
                        for (int j = 0; j < 4 * NV; ++j) O[rt][j / 4][j % 4] = fmaf(p, (float)vs[j], O[rt][j / 4][j % 4]);
                    }
                return;
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (REV ? 16 * rt >= k0 + 32 : 16 * rt + 16 <= k0) continue;
#pragma unroll
                for (int n = 0; n < P::TERMS; ++n) {
                    const Frag<ET> p = P::frag(sP, lp, 16 * rt, k0, n);
#pragma unroll
                    for (int x = 0; x < NV; ++x) O[rt][x] = mma(v[x], p, O[rt][x]);
                }
            }
        };
        Weighted<ET, NV, NS> next;
        next.template read<LV>(sh.V, lvc, 32, 16 * NV * w, weights + 32);
        S.scale(0, total);
        pairs_of(0, v.v);
        S.template add<NS, ET>(
            sh.K[grp], lkc, 0, v,
            [&](int t) {
                if (t + 1 < D / 16) S.scale(t + 1, total);
#pragma unroll
                for (int i = t * next.PARTS * 16 / D; i < (t + 1) * next.PARTS * 16 / D; ++i) next.part(i);
            });
        pairs_of(32, next.v);
        S.template add<NS, ET>(sh.K[grp], lkc, 32, next, [](int) {});

        if constexpr (G == 2) {
            float4 *const sum = sh.sum() + w * 64 + l;
            if (grp == 1) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int x = 0; x < NV; ++x)
                        sum[(rt * NV + x) * 64 * NW] = make_float4(O[rt][x][0], O[rt][x][1], O[rt][x][2], O[rt][x][3]);
            }
            __syncthreads();
            if (grp == 0) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int x = 0; x < NV; ++x) {
                        const float4 y = sum[(rt * NV + x) * 64 * NW];
                        O[rt][x] += f4{y.x, y.y, y.z, y.w};
                    }
            }
        }
        const unsigned o_row = (a.Hv / G) * a.dv;
        char *const o0 = static_cast<char *>(a.o) + (((b * (int64_t)a.T + t0) * (a.Hv / G) + hg) * a.dv << (a.o_dt == DT_F32 ? 2 : 1));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = 16 * rt + li;
            float o[4 * NV];
            row_of(rt, o);
            if (r < n && grp == 0) {
                const unsigned at = __umul24(r, o_row) + col;
                if constexpr (VEC) {
                    if (col < a.dv) store_row<4 * NV, ET>(o0, at, a.o_dt, o);
                } else {
#pragma unroll
                    for (int j = 0; j < 4 * NV; ++j)
                        if (col + j < a.dv) store_from_f32(o0, at + j, o[j], a.o_dt);
                }
            }
        }
        if constexpr (KIND == DK) {
            if (marked) {
                const double x = wave_prefix_sum(S.product(a.marks + mark * (D * 16 * NV * NW), w * 64 + l));
                if (l == 63) a.ends[mark * NW + w] = x;
            }
        }
        const int64_t at = (((int64_t)slice * a.B + b) * a.Hv + h) * a.T + t0;
        if constexpr (DOT) {
            __syncthreads();
            if (w == 0 && l < n) {
                float d = 0.f;
#pragma unroll
                for (int i = 0; i < NW; ++i) d += sh.dot[grp][i][l];
                a.dot[at + l] = d;
            }
        }
        if constexpr (KIND == DV) {
            __syncthreads();
            if (w == 0) {
                double x = 0.;
#pragma unroll
                for (int i = 0; i < NW; ++i) x += (double)sh.cross()[i * C + l];
                if (l < n) a.dot[at + l] = (float)x;
            }
        }
    }
    if (a.s_out && seg == (REV ? 0 : a.nseg - 1)) S.store(a.s_out + head * a.dk * a.dv, a.dk, a.dv, c0, a.s_t);
}

struct Seg {
    Ten K, V;
    const float *decays;
    float *s;      // [B][Hv][nseg][dv][dk]
    float *decay;  // [B][Hv][nseg]
    int B, T, Hv, dk, dv, slices, nseg, cps, nc, dt;
    float scale;
};

// What a segment adds to a state that starts from nothing, and its decay.  The segment that the chain ends with is left out
// (the last; reverse: the first).  Three quarters of the sequence's state products once more (66 us at B=4, T=4096, Hv=32), for
// four times as many workgroups in every pass: unsplit, 128 heads leave half of 256 CUs without work.
template <typename ET, int D, int NV, int NW, bool REV, bool VEC>
__global__ __launch_bounds__(64 * NW, (waves<ET, D>())) void seg_kernel(const Seg a) {
    constexpr int NS = std::is_same_v<ET, float> ? 1 : 3;
    using LK = Lds<ET, D>;
    using LV = Lds<ET, 16 * NV * NW>;
    __shared__ __attribute__((aligned(16))) ET sK[C * LK::LD];
    __shared__ __attribute__((aligned(16))) ET sV[C * LV::LD];
    __shared__ Decays d;
    __shared__ float sum;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4;
    int id = xcd_order(blockIdx.x, gridDim.x);
    const int slice = id % a.slices;
    id /= a.slices;
    const int h = id % a.Hv;
    id /= a.Hv;
    const int b = id % a.B, seg = id / a.B + (REV ? 1 : 0), c0 = slice * 16 * NV * NW;
    const int first = seg * a.cps, last = min(a.nc, first + a.cps) - 1;
    State<D, NV, NW> S;
    S.load(nullptr, a.dk, a.dv, c0, 0);
    Tile<ET, D, VEC, 64 * NW> tk;
    Tile<ET, 16 * NV * NW, VEC, 64 * NW> tv;
    float td = 0.f, all = 1.f;
    const auto fetch = [&](int c) {
        const int64_t t0 = (int64_t)c * C;
        const int n = min((int64_t)C, a.T - t0);
        tk.fetch(a.K.template from<ET>(b, t0, h, 0, a.dt), a.K.st, n, a.dk, a.dt);
        tv.fetch(a.V.template from<ET>(b, t0, h, c0, a.dt), a.V.st, n, a.dv - c0, a.dt);
        td = a.decays[(((int64_t)b * a.Hv + h) * a.nc + c) * DECAYS + (tid & (NT - 1))];
    };
    fetch(REV ? last : first);
    for (int i = first; i <= last; ++i) {
        const int c = REV ? first + last - i : i, n = min((int64_t)C, a.T - (int64_t)c * C);
        __syncthreads();
        tk.store(sK, n, a.dk, a.dt);
        tv.store(sV, n, a.dv - c0, a.dt);
        reinterpret_cast<float *>(&d)[tid & (NT - 1)] = REV && (w & 3) == 2 ? td * a.scale : td;
        if (w == 2 && l == C - 1) sum = td;
        __syncthreads();
        if (i < last) fetch(REV ? c - 1 : c + 1);
        const float total = sum;
        all *= total;
        const int li = l & 15, lvc = LV::template col_lane<4 * NV>(li, g), lkc = LK::template col_lane<8>(li, g);
        const float *const weights = (REV ? d.in : d.out) + 8 * g;
        Weighted<ET, NV, NS> v, next;
        v.template read<LV>(sV, lvc, 0, 16 * NV * w, weights);
        v.all();
        next.template read<LV>(sV, lvc, 32, 16 * NV * w, weights + 32);
        S.scale(0, total);
        S.template add<NS, ET>(
            sK, lkc, 0, v,
            [&](int t) {
                if (t + 1 < D / 16) S.scale(t + 1, total);
#pragma unroll
                for (int i = t * next.PARTS * 16 / D; i < (t + 1) * next.PARTS * 16 / D; ++i) next.part(i);
            });
        S.template add<NS, ET>(sK, lkc, 32, next, [](int) {});
    }
    const int64_t at = ((int64_t)b * a.Hv + h) * a.nseg + seg;
    S.store(a.s + at * a.dk * a.dv, a.dk, a.dv, c0, 0);
    if (tid == 0 && slice == 0) a.decay[at] = all;
}

// Columns of V' to a workgroup: 64, or 128 where the state of 128 fits the registers beside the tiles.
inline int cols_of(int dk, int dv) { return dv <= 64 || dk > 128 ? 64 : 128; }
// Of a pass: K' channels that a kernel's tiles hold, and waves to a head.
inline int rows_of(int dk) { return dk <= 64 ? 64 : dk <= 128 ? 128 : 256; }
inline int waves_of(int dk, int dv, int dt) { return cols_of(dk, dv) == 128 && dt != DT_BF16 ? 8 : 4; }
// For segment sums in bf16 always 64: three quarters of two workgroups for each compute unit become three halves, which share
// out evenly, three waves to a SIMD (B=4, T=4096, Hv=32: 67 us against 79; two LDS buffers at 128 columns gained nothing).
inline int seg_cols(int dk, int dv, int dt) { return dt == DT_BF16 ? 64 : cols_of(dk, dv); }

// dq and dk of two value heads are added in one workgroup where its LDS holds both.
template <typename ET, int D>
constexpr bool pairs() { return std::is_same_v<ET, bf16> && D <= 128; }

// Launches for K' heads of up to 64, 128 and 256 channels, the second set for sizes that are no multiple of 8.
#define GDN_LINATT_DECLARE(NAME)                                  \
    void pass_##NAME(const Pass &a, Kind kind, hipStream_t st);   \
    void seg_##NAME(const Seg &a, bool rev, hipStream_t st);
GDN_LINATT_DECLARE(d64)
GDN_LINATT_DECLARE(d128)
GDN_LINATT_DECLARE(d256)
GDN_LINATT_DECLARE(odd64)
GDN_LINATT_DECLARE(odd128)
GDN_LINATT_DECLARE(odd256)

// VEC: all heads' channels are a multiple of 8.
template <typename ET, int D, int NV, int NW, bool VEC>
void launch_pass(const Pass &a, Kind kind, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.slices * a.Hv * a.B * a.nseg / (a.pair ? 2 : 1)));
    if constexpr (pairs<ET, D>()) {
        if (a.pair) {
            const dim3 block(128 * NW);
            if (kind == DQ) hipLaunchKernelGGL((pass_kernel<ET, D, NV, NW, DQ, 2, VEC>), grid, block, 0, st, a);
            else hipLaunchKernelGGL((pass_kernel<ET, D, NV, NW, DK, 2, VEC>), grid, block, 0, st, a);
            return;
        }
    }
    const dim3 block(64 * NW);
    if (kind == Y) hipLaunchKernelGGL((pass_kernel<ET, D, NV, NW, Y, 1, VEC>), grid, block, 0, st, a);
    else if (kind == DQ) hipLaunchKernelGGL((pass_kernel<ET, D, NV, NW, DQ, 1, VEC>), grid, block, 0, st, a);
    else if (kind == DK) hipLaunchKernelGGL((pass_kernel<ET, D, NV, NW, DK, 1, VEC>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((pass_kernel<ET, D, NV, NW, DV, 1, VEC>), grid, block, 0, st, a);
}
template <typename ET, int D, int NV, int NW, bool VEC>
void launch_seg(const Seg &a, bool rev, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.slices * a.Hv * a.B * (a.nseg - 1))), block(64 * NW);
    if (rev) hipLaunchKernelGGL((seg_kernel<ET, D, NV, NW, true, VEC>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((seg_kernel<ET, D, NV, NW, false, VEC>), grid, block, 0, st, a);
}
// 128 columns of V' go to four waves of 32 in bf16 (eight of 16 read the K' and Q' tiles twice as often: 171 us against 144
// for two sequences of 8100 tokens, 32 heads, when both were tried, with one term of P and the state), to eight of 16 in fp32
// (two waves to a SIMD: 83 us against 87 for 2047 tokens; now 80).
template <typename ET>
constexpr int wide_columns() { return std::is_same_v<ET, bf16> ? 2 : 1; }
template <typename ET, int D, bool VEC>
void launch_pass_cols(const Pass &a, Kind kind, hipStream_t st) {
    if constexpr (D <= 128) {
        constexpr int NV = wide_columns<ET>();
        if (cols_of(D, a.dv) == 128) return launch_pass<ET, D, NV, 8 / NV, VEC>(a, kind, st);
    }
    launch_pass<ET, D, 1, 4, VEC>(a, kind, st);
}
template <typename ET, int D, bool VEC>
void launch_seg_cols(const Seg &a, bool rev, hipStream_t st) {
    if constexpr (D <= 128 && std::is_same_v<ET, float>) {
        if (seg_cols(D, a.dv, a.dt) == 128) return launch_seg<ET, D, 1, 8, VEC>(a, rev, st);
    }
    launch_seg<ET, D, 1, 4, VEC>(a, rev, st);
}
#define GDN_LINATT(NAME, D, VEC)                                       \
    void pass_##NAME(const Pass &a, Kind kind, hipStream_t st) {        \
        if (a.dt == DT_BF16) launch_pass_cols<bf16, D, VEC>(a, kind, st); \
        else launch_pass_cols<float, D, VEC>(a, kind, st);             \
    }                                                                  \
    void seg_##NAME(const Seg &a, bool rev, hipStream_t st) {           \
        if (a.dt == DT_BF16) launch_seg_cols<bf16, D, VEC>(a, rev, st);  \
        else launch_seg_cols<float, D, VEC>(a, rev, st);               \
    }

}  // namespace la
}  // namespace gdn
