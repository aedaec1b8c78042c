// Log probabilities of given tokens with entropy and top alternatives, and the gradient of the logits, for gfx950.
//
// A row z of V logits: p_j = e^{z_j - M} / s, M = max z, s = sum e^{z_j - M};
//   logp = z_target - M - log s,   H = log s - t / s,  t = sum e^{z_j - M} (z_j - M).
// Rows are cut into pieces of PIECE logits, one workgroup each, that a thread holds in registers: every logit is read
// once, and a single row still spreads over V / PIECE workgroups.  A piece leaves (m, s, t) of its own maximum and its
// `top` largest; a second kernel joins the pieces of a row (factors e^{m - M}).
//
// Top alternatives are ordered by value, equal ones by index: a logit's key is its value as an ordered integer above
// the complement of its index, so keys are unique and no order of arrival can matter.  The `top` largest keys of a
// piece are held by at most `top` threads, those whose own largest key ranks among the first `top`: only these hand
// their keys on, and the few that remain are ranked by counting.
//
// Gradient: dz_j = d ([j = target] - p_j) - e p_j (log p_j + H) for the cotangents d of logp and e of H.  Streaming:
// logits in, gradient out.
//
// Measured: 8192 rows of 32000 bf16 logits (524 MB): pieces 126 us (4.2 TB/s; 136 with a group of 8 loaded after the other),
// join 6, gradient 159 (1.05 GB less what ignored rows need not read).  64 rows of 131072 with entropy and 20 alternatives
// 22.5 us: 26 with one lane to a key in the ranking, 30 with every thread's largest key ranked first.
#include "gdn_common.h"
#include "gdn_host.h"
#include "gdn_vec.h"
#include "../../include/gdn_mi355x.h"

namespace gdn {
namespace lp {

constexpr int NT = 256;
constexpr int E = 32;             // logits per thread
constexpr int PIECE = NT * E;
constexpr int MAX_TOP = 64;
constexpr int TURN = 32;
constexpr float LOG2E = 1.4426950408889634f;

struct Rows {  // row r of [outer][inner] rows of V logits
    const void *z;
    int64_t so, si;
    int inner, dt;
    int64_t V;
    __device__ __forceinline__ int64_t at(int64_t r) const { return (r / inner) * so + (r % inner) * si; }
};

// e^x by 2^(x log2 e) on v_exp_f32: x <= 0 here, relative error about 2^-23 (1 + |x|)
__device__ __forceinline__ float exp_(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// 16 bytes from an address that is a multiple of the element's size only: rows of an odd V start anywhere
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) u4_any {
    u4 v;
};
// Eight logits as they lie in memory.
template <int DT>
struct Raw8 {
    u4 a[DT == DT_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void *p, int64_t i) {
        const char *s = static_cast<const char *>(p) + i * (DT == DT_F32 ? 4 : 2);
        a[0] = reinterpret_cast<const u4_any *>(s)->v;
        if constexpr (DT == DT_F32) a[1] = reinterpret_cast<const u4_any *>(s + 16)->v;
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (DT == DT_F32) return __uint_as_float(a[j / 4][j % 4]);
        else if constexpr (DT == DT_BF16) return __uint_as_float(j & 1 ? a[0][j / 2] & 0xffff0000u : a[0][j / 2] << 16);
        else return ops::half_bits_to_f32(a[0][j / 2] >> (16 * (j & 1)));
    }
};
template <int DT>
__device__ __forceinline__ void store8(void *p, int64_t i, const float (&o)[8]) {
    if constexpr (DT == DT_F32) {
        const u4 a = {__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3])};
        const u4 b = {__float_as_uint(o[4]), __float_as_uint(o[5]), __float_as_uint(o[6]), __float_as_uint(o[7])};
        reinterpret_cast<u4_any *>(static_cast<float *>(p) + i)->v = a;
        reinterpret_cast<u4_any *>(static_cast<float *>(p) + i + 4)->v = b;
    } else {
        u4 a;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = ops::pack2_cvt(o[2 * j], o[2 * j + 1], DT);
        reinterpret_cast<u4_any *>(static_cast<uint16_t *>(p) + i)->v = a;
    }
}

// The E logits of thread tid of the piece that starts at v0: 8 at a time, NT * 8 apart; past the end `fill`.  All loads are
// issued before the first is used: none stands under a branch, those past the end read the piece's first logits.
template <int DT>
__device__ __forceinline__ void load_piece(const Rows &a, int64_t row, int64_t v0, float (&x)[E], float fill) {
    const int64_t base = a.at(row) + v0;
    const int left = (int)min((int64_t)PIECE, a.V - v0);
    if (left < 8) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = fill;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (threadIdx.x == 0 && i < left) x[i] = load_as_f32(a.z, base + i, DT);
        return;
    }
    Raw8<DT> raw[E / 8];
#pragma unroll
    for (int c = 0; c < E / 8; ++c) {
        const int j = (c * NT + threadIdx.x) * 8;
        raw[c].load(a.z, base + (j + 8 <= left ? j : 0));
    }
#pragma unroll
    for (int c = 0; c < E / 8; ++c) {
        const int j = (c * NT + threadIdx.x) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[c * 8 + i] = raw[c].get(i);
        if (j + 8 > left) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[c * 8 + i] = j + i < left ? load_as_f32(a.z, base + j + i, DT) : fill;
        }
    }
}

__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dpp_mov<DPP_QUAD_1032>(x));
    x = fmaxf(x, dpp_mov<DPP_QUAD_2301>(x));
    x = fmaxf(x, dpp_mov<DPP_ROW_HALF_MIRROR>(x));
    x = fmaxf(x, dpp_mov<DPP_ROW_MIRROR>(x));
    x = fmaxf(x, lane_xor16(x));
    return fmaxf(x, lane_xor32(x));
}

// Order of values as unsigned integers: -inf < ... < -0 = +0 < ... < +inf < NaN; every value is > 0.
__device__ __forceinline__ uint32_t ordered(float x) {
    x += 0.f;  // -0 is equal to +0
    const uint32_t u = __float_as_uint(x);
    if (x != x) return 0xffffffffu;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
    return o == 0xffffffffu ? __uint_as_float(0x7fc00000u)
                            : __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return ((uint64_t)ordered(x) << 32) | (uint32_t)~i; }

struct TopShared {
    uint64_t best[NT];
    __attribute__((aligned(16))) uint64_t list[MAX_TOP * E + TURN];  // at most `top` threads hand on at most E keys each
    uint64_t border;
    float group[NT / 4], least;
    int n, odd;
};

// The keys of the list by rank, the r-th to out[r]; places without a key get 0, as keys of 0 are none.  Four lanes count the
// larger ones for a key, 32 to a turn and all of a turn's reads under way at once (one by one their latency is the kernel's
// time: 15 us for 20 alternatives of 16 pieces).  Every thread calls it; it begins with a barrier.
__device__ __forceinline__ void rank_list(TopShared &sh, int n, int top, uint64_t *out) {
    const int tid = threadIdx.x;
    if (tid < TURN) sh.list[n + tid] = 0;
    for (int i = n + tid; i < top; i += NT) out[i] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += NT / 4) {
        const int i = i0 + tid / 4;
        const uint64_t k = i < n ? sh.list[i] : ~(uint64_t)0;
        int r = 0;
        for (int j = 2 * (tid & 3); j < n; j += TURN) {
            ulonglong2 v[TURN / 8];
#pragma unroll
            for (int e = 0; e < TURN / 8; ++e) v[e] = *reinterpret_cast<const ulonglong2 *>(sh.list + j + 8 * e);
#pragma unroll
            for (int e = 0; e < TURN / 8; ++e) r += (v[e].x > k) + (v[e].y > k);
        }
        r += __shfl_xor(r, 1);
        r += __shfl_xor(r, 2);
        if (i < n && k && r < top && (tid & 3) == 0) out[r] = k;
    }
}

// The `top` largest of the workgroup's keys (0: none), the r-th to out[r]; places without a key get 0.  Every thread
// calls it.
template <typename KEY>
__device__ __forceinline__ void select_top(TopShared &sh, KEY key, int top, uint64_t *out) {
    const int tid = threadIdx.x;
    uint64_t best = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint64_t k = key(e);
        best = k > best ? k : best;
    }
    sh.best[tid] = best;
    if (tid == 0) sh.n = 0;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < NT; ++i) before += sh.best[i] > best;
    // the top-th largest of the threads' best is at most the top-th largest of all
    if (tid == 0) sh.border = 0;
    __syncthreads();
    if (best && before == top - 1) sh.border = best;
    __syncthreads();
    const uint64_t b = sh.border;  // 0 where fewer than `top` threads hold a key: everything is handed on
    if (best && before < top) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint64_t k = key(e);
            if (k && k >= b) sh.list[atomicAdd(&sh.n, 1)] = k;  // ranks below do not depend on the order
        }
    }
    __syncthreads();
    rank_list(sh, sh.n, top, out);
}

// The same from the logits: those not below the top-th largest of 64 groups' maxima (at least `top` of them, seldom many
// more) are handed on.  False, and nothing written, where that gives more than the list holds (equal logits, most of them
// -inf) or a logit is NaN, whose order the maxima do not show.  mine: the thread's largest logit; index: a logit's place in
// the row, or < 0 past its end.
template <typename INDEX>
__device__ __forceinline__ bool select_values(TopShared &sh, const float (&x)[E], float mine, INDEX index, int top,
                                              uint64_t *out) {
    const int tid = threadIdx.x;
    float nan = 0.f, g = mine;
#pragma unroll
    for (int e = 0; e < E; ++e) nan += x[e] != x[e] ? 1.f : 0.f;
    g = fmaxf(g, dpp_mov<DPP_QUAD_1032>(g));
    g = fmaxf(g, dpp_mov<DPP_QUAD_2301>(g));
    if ((tid & 3) == 0) sh.group[tid / 4] = g;
    if (tid == 0) sh.n = sh.odd = 0;
    __syncthreads();
    if (nan != 0.f) sh.odd = 1;
    int above = 0, equal = 0;
#pragma unroll
    for (int i = 0; i < NT / 4; i += 4) {
        const float4 v = *reinterpret_cast<const float4 *>(sh.group + i);
        above += (v.x > g) + (v.y > g) + (v.z > g) + (v.w > g);
        equal += (v.x == g) + (v.y == g) + (v.z == g) + (v.w == g);
    }
    if (above < top && above + equal >= top) sh.least = g;  // the same value from every group that has it
    __syncthreads();
    if (sh.odd) return false;
    const float least = sh.least;
    if (mine >= least) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t j = index(e);
            if (j >= 0 && x[e] >= least) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < MAX_TOP * E) sh.list[at] = key_of(x[e], (uint32_t)j);
            }
        }
    }
    __syncthreads();
    if (sh.n > MAX_TOP * E) return false;
    rank_list(sh, sh.n, top, out);
    return true;
}

// One piece of one row: part[row][piece] = (m, s, t, -), keys[row][piece][top].
template <int DT, bool ENT, bool TOP>
__global__ __launch_bounds__(NT) void piece_kernel(Rows a, float4 *part, uint64_t *keys, int pieces, int top) {
    const int piece = blockIdx.x % pieces, tid = threadIdx.x;
    const int64_t row = blockIdx.x / pieces, v0 = (int64_t)piece * PIECE;
    float x[E];
    load_piece<DT>(a, row, v0, x, -__builtin_inff());
    __shared__ float red[3][NT / 64];
    float mine = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) mine = fmaxf(mine, x[e]);
    float m = wave_max(mine);
    if ((tid & 63) == 0) red[0][tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float mm = m == -__builtin_inff() ? 0.f : m;  // a piece with nothing left: s = 0
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float d = x[e] - mm, p = exp_(d);
        s += p;
        if constexpr (ENT) t = p > 0.f ? fmaf(p, d, t) : t;
    }
    s = ops::group_sum<64>(s);
    if constexpr (ENT) t = ops::group_sum<64>(t);
    if ((tid & 63) == 0) {
        red[1][tid >> 6] = s;
        if constexpr (ENT) red[2][tid >> 6] = t;
    }
    __syncthreads();
    if (tid == 0) {
        s = red[1][0] + red[1][1] + red[1][2] + red[1][3];
        t = ENT ? red[2][0] + red[2][1] + red[2][2] + red[2][3] : 0.f;
        part[row * pieces + piece] = make_float4(m, s, t, 0.f);
    }
    if constexpr (TOP) {
        __shared__ TopShared sh;
        const int64_t left = a.V - v0;
        const auto at = [&](int e) { return (int64_t)((e / 8) * NT + tid) * 8 + e % 8; };
        uint64_t *const out = keys + (row * pieces + piece) * top;
        if (!select_values(sh, x, mine, [&](int e) { return at(e) < left ? v0 + at(e) : (int64_t)-1; }, top, out)) {
            __syncthreads();
            select_top(sh, [&](int e) { return at(e) < left ? key_of(x[e], (uint32_t)(v0 + at(e))) : (uint64_t)0; }, top, out);
        }
    }
}

struct Join {
    Rows a;
    const int64_t *target;
    int64_t ignore;
    const float4 *part;
    const uint64_t *keys;
    float *logp, *entropy, *stat, *top_logp;  // stat [rows][2]: M, log s
    int64_t *top_ids;
    int64_t rows;
    int pieces, top;
};

// A row of -inf alone, from its statistics: no logit above -inf and the sum 0, for which join_row leaves log s = 0.  Maxima
// skip NaN, so that a row of NaN has M = -inf too, but its log s is NaN.
__device__ __forceinline__ bool nothing_left(float M, float ls) { return M == -__builtin_inff() && ls == 0.f; }

// Joins the pieces of a row in one wave; the lanes' sums are combined in a fixed order.
__device__ __forceinline__ void join_row(const Join &j, int64_t row, int lane, float &M, float &ls) {
    const float4 *p = j.part + row * j.pieces;
    M = -__builtin_inff();
    for (int i = lane; i < j.pieces; i += 64) M = fmaxf(M, p[i].x);
    M = wave_max(M);
    float s = 0.f, t = 0.f;
    for (int i = lane; i < j.pieces; i += 64) {
        const float4 v = p[i];
        if (v.y == 0.f) continue;  // nothing in it (NaN is not 0)
        const float d = v.x - M, f = exp_(d);
        s = fmaf(v.y, f, s);
        t = f > 0.f ? fmaf(f, fmaf(d, v.y, v.z), t) : t;
    }
    s = ops::group_sum<64>(s);
    t = ops::group_sum<64>(t);
    ls = s == 0.f ? 0.f : logf(s);
    if (lane == 0) {
        if (j.stat) {
            j.stat[2 * row] = M;
            j.stat[2 * row + 1] = ls;
        }
        if (j.entropy) j.entropy[row] = s == 0.f ? 0.f : ls - t / s;
        if (j.logp) {
            const int64_t y = j.target[row];
            float o = 0.f;
            if (y != j.ignore) {
                // a target outside the vocabulary has no probability
                o = y < 0 || y >= j.a.V ? __builtin_nanf("") : load_as_f32(j.a.z, j.a.at(row) + y, j.a.dt);
                if (!nothing_left(M, ls)) o = o - M - ls;
            }
            j.logp[row] = o;
        }
    }
}

__global__ __launch_bounds__(NT) void join_kernel(Join j) {
    const int64_t row = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
    float M, ls;
    if (row < j.rows) join_row(j, row, threadIdx.x & 63, M, ls);
}

// With top alternatives: a workgroup per row; its keys are the pieces' largest (at most PIECE of them).
__global__ __launch_bounds__(NT) void join_top_kernel(Join j) {
    __shared__ TopShared sh;
    __shared__ uint64_t best[MAX_TOP];
    const int64_t row = blockIdx.x;
    const int n = j.pieces * j.top, tid = threadIdx.x;
    const uint64_t *k = j.keys + row * n;
    if (n <= MAX_TOP * E) {  // all of them ranked; some may be 0, below every key
        for (int i = tid; i < n; i += NT) sh.list[i] = k[i];
        if (tid < j.top) best[tid] = 0;
        __syncthreads();
        rank_list(sh, n, j.top, best);
    } else {
        uint64_t mine[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = e * NT + tid;
            mine[e] = i < n ? k[i] : 0;
        }
        select_top(sh, [&](int e) { return mine[e]; }, j.top, best);
    }
    __syncthreads();
    float M, ls;
    if (tid < 64) {
        join_row(j, row, tid, M, ls);
        if (tid < j.top) {
            const uint64_t b = best[tid];
            const float v = unordered((uint32_t)(b >> 32));
            j.top_ids[row * j.top + tid] = (int64_t)(uint32_t)~(uint32_t)b;
            j.top_logp[row * j.top + tid] = nothing_left(M, ls) ? v : v - M - ls;
        }
    }
}

struct Bwd {
    Rows a;
    const int64_t *target;
    int64_t ignore;
    const float *stat, *entropy, *dlogp, *dent;
    void *dz;  // contiguous [rows][V]
    int pieces;
};

template <int DT, bool ENT>
__global__ __launch_bounds__(NT) void bwd_kernel(Bwd b) {
    const int64_t row = blockIdx.x / b.pieces, v0 = (int64_t)(blockIdx.x % b.pieces) * PIECE;
    const int64_t left = b.a.V - v0, y = b.target[row];
    const bool live = y != b.ignore;
    float d = live && b.dlogp ? b.dlogp[row] : 0.f;
    if (live && b.dlogp && (y < 0 || y >= b.a.V)) d = __builtin_nanf("");  // as its logp, where that is in the loss
    const float e = ENT ? b.dent[row] : 0.f;
    const int64_t out = row * b.a.V + v0;
    float x[E] = {};
    const bool zero = !live && (!ENT || e == 0.f);  // an ignored row: nothing to read
    if (!zero) load_piece<DT>(b.a, row, v0, x, 0.f);
    const float M = b.stat[2 * row], ls = b.stat[2 * row + 1], h = ENT ? b.entropy[row] : 0.f;
    const bool none = nothing_left(M, ls);  // no gradient
#pragma unroll
    for (int c = 0; c < E / 8; ++c) {
        const int64_t j = (int64_t)(c * NT + threadIdx.x) * 8;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float l = x[c * 8 + i] - M - ls, p = exp_(l);
            float w = d;
            if constexpr (ENT) w = p > 0.f ? fmaf(e, l + h, d) : 0.f;
            o[i] = zero || none ? 0.f : -p * w;
        }
        const int64_t hit = y - v0 - j;
        if (live && !none && hit >= 0 && hit < 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (hit == i) o[i] += d;
        }
        if (j + 8 <= left) {
            store8<DT>(b.dz, out + j, o);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j + i < left) store_from_f32(b.dz, out + j + i, o[i], DT);
        }
    }
}

static int64_t pieces_of(int64_t V) { return (V + PIECE - 1) / PIECE; }
static size_t part_bytes(int64_t rows, int64_t V) { return align_up256((size_t)rows * pieces_of(V) * sizeof(float4)); }

// The checks that the forward and the backward share; 1: nothing to do.
static int check(int64_t outer, int64_t inner, int64_t V, int dtype) {
    if (outer < 0 || inner < 0 || V <= 0) return fail(GDN_ERR_INVALID, "row counts must be >= 0 and V > 0");
    if (dtype != GDN_F32 && dtype != GDN_BF16 && dtype != GDN_F16) return fail(GDN_ERR_INVALID, "unknown dtype code");
    if (outer == 0 || inner == 0) return 1;
    constexpr int64_t MOST = (1 << 24) - 1;  // workgroups of 256 threads: a launch has less than 2^32
    if (V > 0x7fffffff || inner > MOST || outer > MOST / inner || pieces_of(V) > MOST / (outer * inner))
        return fail(GDN_ERR_UNSUPPORTED, "2^24 or more pieces of %d logits are not supported", PIECE);
    return 0;
}

}  // namespace lp
}  // namespace gdn

using namespace gdn;

extern "C" size_t gdn_logprobs_workspace_bytes(int64_t rows, int64_t V, int top) {
    if (rows <= 0 || V <= 0 || top < 0) return 0;
    return lp::part_bytes(rows, V) + align_up256((size_t)rows * lp::pieces_of(V) * top * sizeof(uint64_t));
}

extern "C" int gdn_logprobs_fwd(const void *logits, const int64_t *targets, float *logp, float *entropy, float *stat,
                                int64_t *top_ids, float *top_logp, void *workspace, size_t workspace_bytes,
                                int64_t outer, int64_t inner, int64_t V, int64_t stride_outer, int64_t stride_inner,
                                int64_t ignore_index, int top, int dtype, void *stream) {
    clear_error();
    if (top < 0 || top > V) return fail(GDN_ERR_INVALID, "top must be between 0 and V");
    const int rc = lp::check(outer, inner, V, dtype);
    if (rc) return rc < 0 ? rc : GDN_OK;
    const int64_t rows = outer * inner, pieces = lp::pieces_of(V);
    if (top > lp::MAX_TOP || pieces * top > lp::PIECE)
        return fail(GDN_ERR_UNSUPPORTED, "top alternatives: at most %d, and at most %d over all pieces of %d logits",
                    lp::MAX_TOP, lp::PIECE, lp::PIECE);
    if (!logits || !targets || !logp || (top && (!top_ids || !top_logp))) return fail(GDN_ERR_INVALID, "null pointer");
    const size_t need = gdn_logprobs_workspace_bytes(rows, V, top);
    if (!workspace || workspace_bytes < need)
        return fail(GDN_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %zu bytes required",
                    workspace_bytes, need);
    hipStream_t st = static_cast<hipStream_t>(stream);
    lp::Rows a{logits, stride_outer, stride_inner, (int)inner, dtype, V};
    float4 *part = static_cast<float4 *>(workspace);
    uint64_t *keys = reinterpret_cast<uint64_t *>(static_cast<char *>(workspace) + lp::part_bytes(rows, V));
    const dim3 grid((unsigned)(rows * pieces)), block(lp::NT);
    {
        Timed tm("logprobs_pieces", st);
#define GDN_LP(DT)                                                                                                    \
    if (top && entropy)                                                                                               \
        hipLaunchKernelGGL((lp::piece_kernel<DT, true, true>), grid, block, 0, st, a, part, keys, (int)pieces, top);  \
    else if (top)                                                                                                     \
        hipLaunchKernelGGL((lp::piece_kernel<DT, false, true>), grid, block, 0, st, a, part, keys, (int)pieces, top); \
    else if (entropy)                                                                                                 \
        hipLaunchKernelGGL((lp::piece_kernel<DT, true, false>), grid, block, 0, st, a, part, keys, (int)pieces, top); \
    else                                                                                                              \
        hipLaunchKernelGGL((lp::piece_kernel<DT, false, false>), grid, block, 0, st, a, part, keys, (int)pieces, top)
        if (dtype == GDN_BF16) { GDN_LP(DT_BF16); }
        else if (dtype == GDN_F32) { GDN_LP(DT_F32); }
        else { GDN_LP(DT_F16); }
#undef GDN_LP
    }
    int err = check_launch(st, "gdn_logprobs_fwd");
    if (err) return err;
    lp::Join j{a, targets, ignore_index, part, keys, logp, entropy, stat, top_logp, top_ids, rows, (int)pieces, top};
    {
        Timed tm("logprobs_join", st);
        if (top)
            hipLaunchKernelGGL(lp::join_top_kernel, dim3((unsigned)rows), block, 0, st, j);
        else
            hipLaunchKernelGGL(lp::join_kernel, dim3((unsigned)((rows + 3) / 4)), block, 0, st, j);
    }
    return check_launch(st, "gdn_logprobs_fwd");
}

extern "C" int gdn_logprobs_bwd(const void *logits, const int64_t *targets, const float *stat, const float *entropy,
                                const float *dlogp, const float *dentropy, void *dlogits, int64_t outer, int64_t inner,
                                int64_t V, int64_t stride_outer, int64_t stride_inner, int64_t ignore_index, int dtype,
                                void *stream) {
    clear_error();
    const int rc = lp::check(outer, inner, V, dtype);
    if (rc) return rc < 0 ? rc : GDN_OK;
    if (!logits || !targets || !stat || !dlogits || (dentropy && !entropy)) return fail(GDN_ERR_INVALID, "null pointer");
    const int64_t rows = outer * inner, pieces = lp::pieces_of(V);
    hipStream_t st = static_cast<hipStream_t>(stream);
    lp::Bwd b{{logits, stride_outer, stride_inner, (int)inner, dtype, V}, targets, ignore_index, stat, entropy, dlogp,
              dentropy, dlogits, (int)pieces};
    const dim3 grid((unsigned)(rows * pieces)), block(lp::NT);
    {
        Timed tm("logprobs_bwd", st);
#define GDN_LP(DT)                                                                                                    \
    if (dentropy)                                                                                                     \
        hipLaunchKernelGGL((lp::bwd_kernel<DT, true>), grid, block, 0, st, b);                                        \
    else                                                                                                              \
        hipLaunchKernelGGL((lp::bwd_kernel<DT, false>), grid, block, 0, st, b)
        if (dtype == GDN_BF16) { GDN_LP(DT_BF16); }
        else if (dtype == GDN_F32) { GDN_LP(DT_F32); }
        else { GDN_LP(DT_F16); }
#undef GDN_LP
    }
    return check_launch(st, "gdn_logprobs_bwd");
}
