// Rows of an embedding table, scaled, and the table's gradient by sorted tokens, for gfx950.
//
//   y_n = a W[id_n],     dW[v] = a sum_{n: id_n = v} dy_n   (64-bit sums in the order of n, rounded once)
//
// Both stream: the forward reads and writes a row for each token; the backward reads a row of dy for each token and writes
// every row of dW, zeros where no token points.  Without an order of arrival that could matter: no atomics.
//
// Sorting.  A token's key is its id above its place, so keys are unique and every key's place in the order is a count of
// smaller keys.  Runs of 1024 keys are sorted in LDS; then up to 32 runs at a time are joined by counting: a key's place is
// the sum of its lower bounds in all of them, looked up by bisection.  32768 tokens take two launches, a million three.
//
// Summing.  A word may have most of the tokens, so the sorted list is cut into chunks of 32: chunks that lie within one
// word's run are summed by a workgroup each, and a word's row is then the sum of its whole chunks and the tokens around them.
#include "gdn_common.h"
#include "gdn_host.h"
#include "gdn_vec.h"
#include "../../include/gdn_mi355x.h"

namespace gdn {
namespace emb {

constexpr int NT = 256;
constexpr int RUN = 1024;   // keys sorted in LDS
constexpr int WAYS = 32;    // runs joined at a time
constexpr int CHUNK = 32;   // tokens summed by one workgroup

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

// Runs of RUN keys, sorted.  Tokens without a gradient get the id `words`, behind all others.
__global__ __launch_bounds__(RUN) void run_kernel(const int64_t *ids, uint64_t *keys, int64_t N, int64_t words, int64_t padding) {
    __shared__ uint64_t k[RUN];
    const int t = threadIdx.x;
    const int64_t n = block_index() * RUN + t;
    if (block_index() * RUN >= N) return;
    uint64_t key = ~0ull;
    if (n < N) {
        const int64_t id = ids[n];
        key = (uint64_t)(id >= 0 && id < words && id != padding ? id : words) << 32 | (uint64_t)n;
    }
    k[t] = key;
    __syncthreads();
    for (int size = 2; size <= RUN; size *= 2)
        for (int d = size / 2; d >= 1; d /= 2) {
            const int o = t ^ d;
            if (o > t) {
                const uint64_t a = k[t], b = k[o];
                if ((a > b) == ((t & size) == 0)) { k[t] = b; k[o] = a; }
            }
            __syncthreads();
        }
    if (n < N) keys[n] = k[t];
}

// Joins WAYS runs of `run` keys: each key goes to the place that it has among all of them.
__global__ __launch_bounds__(NT) void join_kernel(const uint64_t *in, uint64_t *out, int64_t N, int64_t run) {
    const int64_t i = block_index() * NT + threadIdx.x;
    if (i >= N) return;
    const uint64_t key = in[i];
    const int64_t first = i / (run * WAYS) * (run * WAYS);
    const int own = (int)((i - first) / run);
    int64_t place = first + (i - first - own * run);
#pragma unroll 4
    for (int r = 0; r < WAYS; ++r) {
        const int64_t a = first + r * run, n = min(run, N - a);
        if (r == own || n <= 0) continue;
        int64_t lo = 0, len = n;  // the number of keys below
        while (len > 0) {
            const int64_t half = len >> 1;
            const bool below = in[a + lo + half] < key;
            lo = below ? lo + half + 1 : lo;
            len = below ? len - half - 1 : half;
        }
        place += lo;
    }
    out[place] = key;
}

// ------------------------------------------------------------------------------------------------ sums

struct SumArgs {
    const uint64_t *keys;
    const void *dy;
    void *dw;
    double *part;   // [chunks][H] of chunks within one word's run
    int *starts;    // [words + 1] the first place of each word's run
    int64_t N, words, ld;
    int H, lanes;  // lanes: threads to a row, a power of two
    double scale;
};

__device__ __forceinline__ int64_t word(uint64_t key) { return (int64_t)(key >> 32); }
__device__ __forceinline__ int64_t token(uint64_t key) { return (int64_t)(key & 0xffffffffull); }

// x += rows of the tokens [a, b) of the sorted list, U under way.
template <int DT, int U, int V>
__device__ __forceinline__ void add_tokens(const SumArgs &s, int64_t a, int64_t b, int64_t c, double (&x)[V]) {
    int64_t i = a;
    for (; i + U <= b; i += U) {
        float v[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) ops::load_first<V, DT>(s.dy, token(s.keys[i + u]) * s.ld + c, s.H - c, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] += v[u][j];
    }
    for (; i < b; ++i) {
        float v[V];
        ops::load_first<V, DT>(s.dy, token(s.keys[i]) * s.ld + c, s.H - c, v);
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] += v[j];
    }
}

// The first `chunks` workgroups: sums of whole chunks.  The others: the words' first places.
template <int DT>
__global__ __launch_bounds__(NT) void chunk_kernel(const SumArgs s, int64_t chunks) {
    constexpr int V = Width<DT>::V;
    const int64_t g = block_index();
    if (g < chunks) {
        const int64_t a = g * CHUNK, b = a + CHUNK;
        if (b > s.N) return;
        const int64_t id = word(s.keys[a]);
        if (id == s.words || word(s.keys[b - 1]) != id) return;
        for (int64_t c = (int64_t)threadIdx.x * V; c < s.H; c += NT * V) {
            double x[V];
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = 0.;
            add_tokens<DT, 8>(s, a, b, c, x);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < s.H) s.part[g * s.H + c + j] = x[j];
        }
        return;
    }
    const int64_t v = (g - chunks) * NT + threadIdx.x;
    if (v > s.words) return;
    const uint64_t key = (uint64_t)v << 32;
    int64_t lo = 0, len = s.N;
    while (len > 0) {
        const int64_t half = len >> 1;
        const bool below = s.keys[lo + half] < key;
        lo = below ? lo + half + 1 : lo;
        len = below ? len - half - 1 : half;
    }
    s.starts[v] = (int)lo;
}

template <int DT>
__global__ __launch_bounds__(NT) void words_kernel(const SumArgs s) {
    constexpr int V = Width<DT>::V;
    const int lane = threadIdx.x & (s.lanes - 1);
    const int64_t v = block_index() * (NT / s.lanes) + threadIdx.x / s.lanes;
    if (v >= s.words) return;
    const int64_t a = s.starts[v], b = s.starts[v + 1];
    for (int64_t c = (int64_t)lane * V; c < s.H; c += s.lanes * V) {
        double x[V];
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = 0.;
        // tokens up to the first whole chunk, whole chunks, tokens after them; or tokens alone
        const int64_t c0 = (a + CHUNK - 1) / CHUNK, c1 = b / CHUNK;
        int64_t from = a, to = c0 < c1 ? c0 * CHUNK : b;
        while (from < b) {
            add_tokens<DT, 4>(s, from, to, c, x);
            if (to == b) break;
#pragma unroll 2
            for (int64_t k = c0; k < c1; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) x[j] += c + j < s.H ? s.part[k * s.H + c + j] : 0.;
            from = c1 * CHUNK;
            to = b;
        }
        float y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = (float)(x[j] * s.scale);
        ops::store_first<V, DT>(s.dw, v * s.H + c, s.H - c, y);
    }
}

static int check(int64_t N, int64_t V, int64_t H, int dt) {
    if (N < 0 || V <= 0 || H <= 0) return fail(GDN_ERR_INVALID, "N must be >= 0, V and H > 0");
    if (dt != GDN_F32 && dt != GDN_BF16 && dt != GDN_F16) return fail(GDN_ERR_INVALID, "unknown dtype code");
    if (N > 1 << 26 || V > 1 << 26 || H > 1 << 20)
        return fail(GDN_ERR_UNSUPPORTED, "more than 2^26 tokens or words, or 2^20 channels are not supported");
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
    if (N < 0 || V <= 0 || H <= 0 || N > 1 << 26 || V > 1 << 26 || H > 1 << 20) return 0;
    return 2 * align_up256((size_t)N * 8) + align_up256((size_t)(N / emb::CHUNK) * H * 8) + align_up256((size_t)(V + 1) * 4);
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
    s.part = reinterpret_cast<double *>(at);
    s.starts = reinterpret_cast<int *>(at + align_up256((size_t)(N / emb::CHUNK) * H * 8));
    if (N > 0) {
        Timed tm("embedding_order", st);
        hipLaunchKernelGGL(emb::run_kernel, grid_of((N + emb::RUN - 1) / emb::RUN), dim3(emb::RUN), 0, st, ids, keys, N, V,
                           padding_idx);
        for (int64_t run = emb::RUN; run < N; run *= emb::WAYS) {
            hipLaunchKernelGGL(emb::join_kernel, grid_of((N + emb::NT - 1) / emb::NT), dim3(emb::NT), 0, st, keys, other, N, run);
            uint64_t *t = keys;
            keys = other;
            other = t;
        }
    }
    s.keys = keys; s.dy = dy; s.dw = dw;
    s.N = N; s.words = V; s.ld = dy_stride; s.H = (int)H; s.scale = scale;
    s.lanes = 1;
    while (s.lanes < emb::NT && s.lanes * emb::width(dtype) < H) s.lanes *= 2;
    const int64_t chunks = N / emb::CHUNK;
    const dim3 block(emb::NT), some = grid_of(chunks + (V + emb::NT) / emb::NT);
    const dim3 all = grid_of((V + emb::NT / s.lanes - 1) / (emb::NT / s.lanes));
    {
        Timed tm("embedding_sum", st);
#define GDN_SUMS(DT)                                                                  \
    hipLaunchKernelGGL((emb::chunk_kernel<DT>), some, block, 0, st, s, chunks);       \
    hipLaunchKernelGGL((emb::words_kernel<DT>), all, block, 0, st, s)
        GDN_BY_TYPE(dtype, GDN_SUMS)
#undef GDN_SUMS
    }
    return check_launch(st, "gdn_embedding_bwd");
}
