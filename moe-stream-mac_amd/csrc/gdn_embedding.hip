// Rows of an embedding table, scaled, and the table's gradient by sorted tokens, for gfx950.
//
//   y_n = a W[id_n],     dW[v] = a sum_{n: id_n = v} dy_n   (64-bit sums, rounded to 32 bits and their type)
//
// Both stream: the forward reads and writes a row for each token; the backward reads a row of dy for each token and writes
// every row of dW, zeros where no token points.  Without an order of arrival that could matter: no atomics.
//
// Sorting.  A token's key is its id above its place, so keys are unique and every key's place in the order is a count of
// smaller keys.  Runs of 1024 keys are sorted by a workgroup each; then up to 32 runs at a time are joined by counting: a key's
// place is the sum of its lower bounds in all of them, looked up by bisection.  32768 tokens take two launches, a million three.
//
// Summing.  A word may have most of the tokens, so the sorted list is cut into chunks of 32.  A workgroup sums the
// runs in its chunk: it writes the rows of words that begin and end there, and leaves what it has of the others, whose rows are
// then the sums of what their chunks left; of long batches, groups of 64 chunks of one word are summed first.  Other workgroups
// write the zeros of words without a token meanwhile.  65536 tokens, two thirds of one word, 1024 bf16 channels: 202 us with the
// groups, 283 without.
//
// Measured, 16384 tokens, 32000 x 2048 bf16: rows 26 us (5 TB/s with what the caches hold), the order 20, chunks and zeros 46, the
// words over ends of chunks 7.
#include "gdn_common.h"
#include "gdn_host.h"
#include "gdn_vec.h"
#include "../../include/gdn_mi355x.h"

namespace gdn {
namespace emb {

constexpr int NT = 256;
constexpr int RUN = 1024;   // keys sorted by one workgroup
constexpr int RUN_BITS = 10;
constexpr int WAYS = 32;    // runs joined at a time
constexpr int CHUNK = 32;   // tokens summed together
constexpr int CT = 128;     // threads that do so
constexpr int WORDS = 32;   // words whose zeros a workgroup writes
constexpr int GROUP = 64;   // chunks of one word summed first
constexpr int64_t LONG = 1 << 16;  // tokens from which on they are

// ------------------------------------------------------------------------------------------------ forward

template <int DT>
struct Width { static constexpr int V = DT == DT_F32 ? 4 : 8; };  // elements to a thread: 16 bytes

// `per` vectors to a row.
template <int DT>
__global__ __launch_bounds__(NT) void rows_kernel(const int64_t *ids, const void *w, void *y, int64_t N, int64_t words, int H,
                                                  int64_t ld, double scale, uint32_t per) {
    constexpr int V = Width<DT>::V;
    const int64_t i = block_index() * NT + threadIdx.x;
    const int64_t n = i >> 32 ? i / per : (uint32_t)i / per;
    if (n >= N) return;
    const int64_t c = (i - n * per) * V, id = ids[n];
    float x[V];
    const bool in = id >= 0 && id < words;
    ops::load_first<V, DT>(w, (in ? id : 0) * ld + c, H - c, x);
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = in ? (float)(x[j] * scale) : NAN;
    ops::store_first<V, DT>(y, n * H + c, H - c, x);
}

// ------------------------------------------------------------------------------------------------ order

// Runs of RUN keys, sorted.  Tokens without a gradient get the id `words`, behind all others.  A key is sorted as 32 bits, its id
// above its place in the run: a network of compare-exchanges, over lanes of a wave by shuffles, over waves through LDS.
__global__ __launch_bounds__(RUN) void run_kernel(const int64_t *ids, uint64_t *keys, int64_t N, int64_t words, int64_t padding) {
    __shared__ uint32_t k[RUN];
    const int t = threadIdx.x;
    const int64_t n0 = block_index() * RUN, n = n0 + t;
    if (n0 >= N) return;
    uint32_t key = 0xffffffffu;
    if (n < N) {
        const int64_t id = ids[n];
        key = (uint32_t)(id >= 0 && id < words && id != padding ? id : words) << RUN_BITS | (uint32_t)t;
    }
#pragma unroll
    for (int size = 2; size <= RUN; size *= 2)
#pragma unroll
        for (int d = size / 2; d >= 1; d /= 2) {
            uint32_t o;
            if (d >= 64) {
                __syncthreads();
                k[t] = key;
                __syncthreads();
                o = k[t ^ d];
            } else {
                o = (uint32_t)__shfl_xor((int)key, d);
            }
            const bool least = ((t & d) == 0) == ((t & size) == 0);  // this thread keeps the smaller of the two
            key = least ? min(key, o) : max(key, o);
        }
    if (n < N) keys[n] = (uint64_t)(key >> RUN_BITS) << 32 | (uint64_t)(n0 + (key & (RUN - 1)));
}

// Joins WAYS runs of `run` keys: each key goes to the place that it has among all of them.  Eight lanes to a key, four runs to a
// lane.
__global__ __launch_bounds__(NT) void join_kernel(const uint64_t *in, uint64_t *out, int64_t N, int64_t run) {
    constexpr int LANES = 8, EACH = WAYS / LANES;
    const int64_t i = (block_index() * NT + threadIdx.x) / LANES;
    const int part = threadIdx.x % LANES;
    if (i >= N) return;  // all lanes of a key
    const uint64_t key = in[i];
    const int64_t first = i / (run * WAYS) * (run * WAYS);
    const int own = (int)((i - first) / run);
    int64_t lo[EACH], len[EACH];  // the number of keys below in each run, by bisection, side by side
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
        const int64_t a = first + (part * EACH + r) * run;
        lo[r] = a;
        len[r] = part * EACH + r == own ? 0 : max((int64_t)0, min(run, N - a));
    }
    for (int64_t left = run; left > 0; left >>= 1) {
#pragma unroll
        for (int r = 0; r < EACH; ++r) {
            const int64_t half = len[r] >> 1;
            const bool below = len[r] > 0 && in[min(lo[r] + half, N - 1)] < key;
            lo[r] = below ? lo[r] + half + 1 : lo[r];
            len[r] = below ? len[r] - half - 1 : half;
        }
    }
    int64_t place = 0;
#pragma unroll
    for (int r = 0; r < EACH; ++r) place += lo[r] - (first + (part * EACH + r) * run);
#pragma unroll
    for (int o = 1; o < LANES; o *= 2) place += __shfl_xor((int)place, o);
    if (part == 0) out[first + place + (i - first - own * run)] = key;
}

// ------------------------------------------------------------------------------------------------ sums

struct SumArgs {
    const uint64_t *keys;
    const void *dy;
    void *dw;
    double *part;   // [chunks][2][H]: of the word that began before the chunk, of the one that goes on behind it
    double *group;  // [groups][H] of GROUP chunks that began with, and are within, one word; of long batches
    int *starts;    // [words + 1] the first place of each word's run
    int64_t N, words, ld;
    int H;
    double scale;
};

__device__ __forceinline__ int64_t word(uint64_t key) { return (int64_t)(key >> 32); }
__device__ __forceinline__ int64_t token(uint64_t key) { return (int64_t)(key & 0xffffffffull); }

template <int DT, int V>
__device__ __forceinline__ void store_row(const SumArgs &s, int64_t v, int64_t c, const double (&x)[V]) {
    float y[V];
#pragma unroll
    for (int j = 0; j < V; ++j) y[j] = (float)(x[j] * s.scale);
    ops::store_first<V, DT>(s.dw, v * s.H + c, s.H - c, y);
}

// The first workgroups: sums of chunks, CT * V columns of one to each.  The others: the first places of WORDS words each, and the
// zeros of those that no token has.  Their stores fill the memory's time while the sums wait for loads: 16384 tokens of 2048 bf16
// channels, 32000 words (some 200 MB) 46 us, with the zeros in a pass of their own 35 and 38.
template <int DT>
__global__ __launch_bounds__(CT) void chunk_kernel(const SumArgs s, int64_t chunks, int parts) {
    constexpr int V = Width<DT>::V, U = 8;
    const int64_t g = block_index();
    if (g < chunks * parts) {
        const int64_t chunk = g / parts, a = chunk * CHUNK, c = ((g - chunk * parts) * CT + threadIdx.x) * V;
        const int n = (int)min((int64_t)CHUNK, s.N - a), lane = threadIdx.x & 63;
        // lane i of every wave: the chunk's token i, lane n the one behind it
        const bool any = lane <= n && a + lane < s.N;
        const uint64_t key = any ? s.keys[a + lane] : ~0ull;
        const int id = any ? (int)word(key) : -1;
        const int next = __shfl_down(id, 1);
        const int64_t row = any ? token(key) * s.ld : 0;
        const int first = __builtin_amdgcn_readlane(id, 0), last = __builtin_amdgcn_readlane(id, n - 1);
        const uint64_t ends = __ballot(lane < n && (id != next || lane == n - 1));
        const int live = __popcll(__ballot(lane < n && id != s.words));  // the rest of the list has no gradient
        bool before = a > 0 && word(s.keys[a - 1]) == first;
        const bool behind = __builtin_amdgcn_readlane(next, n - 1) == last;
        double x[V];
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = 0.;
        for (int i0 = 0; i0 < live; i0 += U) {
            float v[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = min(i0 + u, live - 1);  // the last one again behind the end
                const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)row, i);
                const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(row >> 32), i);
                ops::load_first<V, DT>(s.dy, (int64_t)((uint64_t)hi << 32 | lo) + c, s.H - c, v[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u;
                if (i < live) {
#pragma unroll
                    for (int j = 0; j < V; ++j) x[j] += v[u][j];
                    if (ends >> i & 1) {
                        const bool goes_on = behind && i == n - 1;
                        if (before || goes_on) {
                            double *to = s.part + (chunk * 2 + (before ? 0 : 1)) * s.H + c;
#pragma unroll
                            for (int j = 0; j < V; ++j)
                                if (c + j < s.H) to[j] = x[j];
                        } else {
                            store_row<DT>(s, __builtin_amdgcn_readlane(id, i), c, x);
                        }
#pragma unroll
                        for (int j = 0; j < V; ++j) x[j] = 0.;
                        before = false;
                    }
                }
            }
        }
        return;
    }
    __shared__ int64_t from[WORDS + 1];
    const int64_t v0 = (g - chunks * parts) * WORDS;
    if (v0 >= s.words) return;
    const int words = (int)min((int64_t)WORDS, s.words - v0);
    if ((int)threadIdx.x <= words) {
        const uint64_t key = (uint64_t)(v0 + threadIdx.x) << 32;
        int64_t lo = 0, len = s.N;
        while (len > 0) {
            const int64_t half = len >> 1;
            const bool below = s.keys[lo + half] < key;
            lo = below ? lo + half + 1 : lo;
            len = below ? len - half - 1 : half;
        }
        from[threadIdx.x] = lo;
        if ((int)threadIdx.x < words || v0 + words == s.words) s.starts[v0 + threadIdx.x] = (int)lo;
    }
    __syncthreads();
    const uint32_t per = (uint32_t)((s.H + V - 1) / V);
    double zero[V];
#pragma unroll
    for (int j = 0; j < V; ++j) zero[j] = 0.;
    for (uint32_t i = threadIdx.x; i < per * words; i += CT) {
        const uint32_t r = i / per;
        if (from[r] == from[r + 1]) store_row<DT>(s, v0 + r, (int64_t)(i - r * per) * V, zero);
    }
}

// x += `count` rows of sums, `step` numbers apart.
template <int V>
__device__ __forceinline__ void add_sums(const double *p, int64_t count, int64_t step, int64_t left, double (&x)[V]) {
#pragma unroll 4
    for (int64_t k = 0; k < count; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] += j < left ? p[k * step + j] : 0.;
}

// Groups of chunks: whole ones whose word is also that of the token before them.
__global__ __launch_bounds__(NT) void group_kernel(const SumArgs s) {
    constexpr int64_t TOKENS = (int64_t)GROUP * CHUNK;
    const int64_t g = blockIdx.x;
    if (g == 0) return;
    const int64_t id = word(s.keys[g * TOKENS - 1]);
    if (id == s.words || word(s.keys[(g + 1) * TOKENS - 1]) != id) return;
    for (int64_t c = threadIdx.x; c < s.H; c += NT) {
        double x[1] = {0.};
        add_sums<1>(s.part + g * GROUP * 2 * s.H + c, GROUP, 2 * s.H, 1, x);
        s.group[g * s.H + c] = x[0];
    }
}

// The words whose runs go over the end of a chunk: each by the workgroups of the second chunk that has it, two columns to a thread.
template <int DT>
__global__ __launch_bounds__(NT) void words_kernel(const SumArgs s, int parts) {
    const int64_t i = block_index(), chunk = i / parts + 1;
    if (chunk * CHUNK >= s.N) return;
    const int64_t id = word(s.keys[chunk * CHUNK]);
    if (id == s.words || word(s.keys[chunk * CHUNK - 1]) != id) return;
    const int64_t a = s.starts[id], b = s.starts[id + 1], c0 = a / CHUNK, c1 = (b - 1) / CHUNK;
    const int64_t c = ((i - (chunk - 1) * parts) * NT + threadIdx.x) * 2;
    if (c0 != chunk - 1 || c >= s.H) return;
    // what chunk c0 left of the run that goes on, then what chunks c0 + 1 to c1 did of the run that began before, whole groups of
    // them at once
    double x[2] = {0., 0.};
    const int64_t step = 2 * s.H, g0 = (c0 + GROUP) / GROUP, g1 = s.group ? b / CHUNK / GROUP : 0;
    const bool grouped = g0 < g1;
#pragma unroll 1
    for (int k = 0; k < 4; ++k) {
        const double *p = s.part + c;
        int64_t count, by = step;
        if (k == 0) {
            p += c0 * step + s.H;
            count = 1;
        } else if (k == 1) {
            p += (c0 + 1) * step;
            count = grouped ? g0 * GROUP - c0 - 1 : c1 - c0;
        } else if (k == 2) {
            p = s.group + g0 * s.H + c;
            count = grouped ? g1 - g0 : 0;
            by = s.H;
        } else {
            p += g1 * GROUP * step;
            count = grouped ? c1 + 1 - g1 * GROUP : 0;
        }
        add_sums<2>(p, count, by, s.H - c, x);
    }
    for (int j = 0; j < 2 && c + j < s.H; ++j) store_from_f32(s.dw, id * s.H + c + j, (float)(x[j] * s.scale), DT);
}

static int check(int64_t N, int64_t V, int64_t H, int dt) {
    if (N < 0 || V <= 0 || H <= 0) return fail(GDN_ERR_INVALID, "N must be >= 0, V and H > 0");
    if (dt != GDN_F32 && dt != GDN_BF16 && dt != GDN_F16) return fail(GDN_ERR_INVALID, "unknown dtype code");
    if (N > 1 << 26 || V >= 1 << 22 || H > 1 << 20)  // ids and places in a run in 32 bits
        return fail(GDN_ERR_UNSUPPORTED, "more than 2^26 tokens, 2^22 - 1 words or 2^20 channels are not supported");
    return GDN_OK;
}

#define GDN_BY_TYPE(dtype, call)                  \
    if (dtype == GDN_F32) { call(DT_F32); }       \
    else if (dtype == GDN_BF16) { call(DT_BF16); } \
    else { call(DT_F16); }

static int width(int dtype) { return dtype == GDN_F32 ? emb::Width<DT_F32>::V : emb::Width<DT_BF16>::V; }

}  // namespace emb
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_embedding_fwd(const int64_t *ids, const void *w, void *y, int64_t N, int64_t V, int64_t H, int64_t w_stride,
                                 double scale, int dtype, void *stream) {
    clear_error();
    if (const int rc = emb::check(N, V, H, dtype)) return rc;
    if (N == 0) return GDN_OK;
    if (!ids || !w || !y) return fail(GDN_ERR_INVALID, "null pointer");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t per = (H + emb::width(dtype) - 1) / emb::width(dtype);
    {
        Timed tm("embedding", st);
#define GDN_ROWS(DT)                                                                                                    \
    hipLaunchKernelGGL((emb::rows_kernel<DT>), grid_of((N * per + emb::NT - 1) / emb::NT), dim3(emb::NT), 0, st, ids, w, y, N, \
                       V, (int)H, w_stride, scale, (uint32_t)per)
        GDN_BY_TYPE(dtype, GDN_ROWS)
#undef GDN_ROWS
    }
    return check_launch(st, "gdn_embedding_fwd");
}

extern "C" size_t gdn_embedding_bwd_workspace_bytes(int64_t N, int64_t V, int64_t H) {
    if (N < 0 || V <= 0 || H <= 0 || N > 1 << 26 || V >= 1 << 22 || H > 1 << 20) return 0;
    const int64_t chunks = (N + emb::CHUNK - 1) / emb::CHUNK, groups = N >= emb::LONG ? N / emb::CHUNK / emb::GROUP : 0;
    return 2 * align_up256((size_t)N * 8) + align_up256((size_t)chunks * 2 * H * 8) + align_up256((size_t)groups * H * 8) +
           align_up256((size_t)(V + 1) * 4);
}

extern "C" int gdn_embedding_bwd(const int64_t *ids, const void *dy, void *dw, void *workspace, size_t workspace_bytes, int64_t N,
                                 int64_t V, int64_t H, int64_t dy_stride, int64_t padding_idx, double scale, int dtype,
                                 void *stream) {
    clear_error();
    if (const int rc = emb::check(N, V, H, dtype)) return rc;
    if (!dw || !workspace || (N > 0 && (!ids || !dy))) return fail(GDN_ERR_INVALID, "null pointer");
    const size_t bytes = gdn_embedding_bwd_workspace_bytes(N, V, H);
    if (workspace_bytes < bytes)
        return fail(GDN_ERR_WORKSPACE, "the workspace holds %zu bytes, %zu are needed", workspace_bytes, bytes);
    hipStream_t st = static_cast<hipStream_t>(stream);
    char *at = static_cast<char *>(workspace);
    uint64_t *keys = reinterpret_cast<uint64_t *>(at), *other = reinterpret_cast<uint64_t *>(at + align_up256((size_t)N * 8));
    at += 2 * align_up256((size_t)N * 8);
    emb::SumArgs s{};
    const int64_t chunks = (N + emb::CHUNK - 1) / emb::CHUNK, groups = N >= emb::LONG ? N / emb::CHUNK / emb::GROUP : 0;
    s.part = reinterpret_cast<double *>(at);
    at += align_up256((size_t)chunks * 2 * H * 8);
    s.group = groups ? reinterpret_cast<double *>(at) : nullptr;
    at += align_up256((size_t)groups * H * 8);
    s.starts = reinterpret_cast<int *>(at);
    if (N > 0) {
        Timed tm("embedding_order", st);
        hipLaunchKernelGGL(emb::run_kernel, grid_of((N + emb::RUN - 1) / emb::RUN), dim3(emb::RUN), 0, st, ids, keys, N, V,
                           padding_idx);
        for (int64_t run = emb::RUN; run < N; run *= emb::WAYS) {
            hipLaunchKernelGGL(emb::join_kernel, grid_of((N * 8 + emb::NT - 1) / emb::NT), dim3(emb::NT), 0, st, keys, other, N,
                               run);
            uint64_t *t = keys;
            keys = other;
            other = t;
        }
    }
    s.keys = keys; s.dy = dy; s.dw = dw;
    s.N = N; s.words = V; s.ld = dy_stride; s.H = (int)H; s.scale = scale;
    const int parts = (int)((H + emb::CT * emb::width(dtype) - 1) / (emb::CT * emb::width(dtype)));
    const int pairs = (int)((H + 2 * emb::NT - 1) / (2 * emb::NT));
    const dim3 block(emb::NT), some = grid_of(chunks * parts + (V + emb::WORDS - 1) / emb::WORDS);
    {
        Timed tm("embedding_sum", st);
#define GDN_SUMS(DT)                                                                  \
    hipLaunchKernelGGL((emb::chunk_kernel<DT>), some, dim3(emb::CT), 0, st, s, chunks, parts); \
    if (groups) hipLaunchKernelGGL(emb::group_kernel, dim3((unsigned)groups), block, 0, st, s); \
    if (chunks > 1) hipLaunchKernelGGL((emb::words_kernel<DT>), grid_of((chunks - 1) * pairs), block, 0, st, s, pairs)
        GDN_BY_TYPE(dtype, GDN_SUMS)
#undef GDN_SUMS
    }
    return check_launch(st, "gdn_embedding_bwd");
}
