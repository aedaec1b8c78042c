// Linear attention: joining segments, heads and decays' gradients, the single token, and the C ABI.  The formulas and the
// kernels that walk the chunks are in gdn_linatt.h.
#include "gdn_linatt.h"

#include "../../include/gdn_mi355x.h"

namespace gdn {
namespace la {

constexpr int MAX_D = 256;

// The decays of every chunk, a wave to a chunk, once for the five or six kernels that use them (a wave of each pass would
// spend two 64-bit exponentials a chunk).  Sums run in 64 bits.  7 us at B=4, T=4096, Hv=32: latency.
__global__ __launch_bounds__(NT) void decay_kernel(Gate g, float *o, int B, int T, int Hv, int nc) {
    const int64_t id = block_index() * (NT / 64) + (threadIdx.x >> 6);
    const int l = threadIdx.x & 63;
    if (id >= (int64_t)B * Hv * nc) return;
    const int h = id % Hv, c = (id / Hv) % nc, b = id / Hv / nc;  // heads side by side: their decays are, in memory
    const int64_t t = (int64_t)c * C + l;
    const double s = wave_prefix_sum(t < T ? (double)g.load(b, t, h) * LOG2E : 0.), end = readlane_f64(s, C - 1);
    const float hi = (float)s;
    float *const p = o + (((int64_t)b * Hv + h) * nc + c) * DECAYS;
    reinterpret_cast<float2 *>(p)[l] = make_float2(hi, (float)(s - (double)hi));
    // rounded once: with one log decay for a whole head their errors repeat in every chunk
    p[2 * C + l] = (float)exp2(s);
    p[3 * C + l] = (float)exp2(end - s);
}

__device__ __forceinline__ double block_sum(double x, double *red, int waves) {
    x = readlane_f64(wave_prefix_sum(x), 63);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    double r = 0.;
    for (int i = 0; i < waves; ++i) r += red[i];
    __syncthreads();
    return r;
}

// The segments' sums become the states entering them (reverse: the cotangents, from the end): from s0 (or nothing) on, in
// place.  Streaming: 34 MB of states in and out, 10 us (128 heads of 128 x 128, four segments).
template <bool REV, int V>
__global__ __launch_bounds__(NT) void scan_kernel(float *s, const float *decay, const float *s0, int nseg, int64_t size) {
    const int64_t head = blockIdx.y, i = ((int64_t)blockIdx.x * NT + threadIdx.x) * V;
    if (i >= size) return;
    float cur[V] = {};
    if (s0)
        for (int e = 0; e < V; ++e) cur[e] = s0[head * size + i + e];  // at any alignment
    for (int j = 0; j < nseg; ++j) {
        const int seg = REV ? nseg - 1 - j : j;
        const int64_t p = (head * nseg + seg) * size + i;
        const float f = j < nseg - 1 ? decay[head * nseg + seg] : 0.f;
        float add[V] = {};
        if (j < nseg - 1) ops::loadv<V>(s, p, DT_F32, add);
        ops::storev<V>(s, p, DT_F32, cur);
#pragma unroll
        for (int e = 0; e < V; ++e) cur[e] = fmaf(f, cur[e], add[e]);
    }
}

// The heads of a group added in order: part [rows][group][D] to o [rows][D].  11 us for 2047 tokens of 2 x 16 heads of 128 in
// fp32 (50 MB).  Atomics into o would round and order the sums differently every time.
__global__ __launch_bounds__(NT) void group_kernel(const float *part, void *o, int64_t n, int group, int D, int dt) {
    const int64_t i = block_index() * NT + threadIdx.x;
    if (i >= n) return;
    const int64_t row = i / D;
    const float *p = part + row * group * D + i % D;
    float s = p[0];
    for (int j = 1; j < group; ++j) s += p[j * D];
    store_from_f32(o, i, s, dt);
}

struct DecayGrad {
    const float *a, *b, *cross;  // [slices][B][Hv][T]; cross: [cross_slices]
    const float *decays;         // [B][Hv][nc][DECAYS]
    const float *dlast, *last;   // [B][Hv][size], or dlast NULL
    const double *ends;          // <dS, S> before every mark_of() chunks, from mark0 on, [B][Hv][nm][parts]
    void *dg;                    // [B][T][Hv]
    double *sums;                // or with one decay per head [Hv][B][nm]
    int B, T, Hv, slices, cross_slices, per_head, dt, nc, nm, mark0, parts;
    float none;                  // a chunk's decay below which it passes nothing on
    int64_t size;
};

// dg between two marks, in 64 bits: a wave sums one chunk; c by the chain from either end.  Its errors are those of the numbers
// that it adds, so the end is taken whose magnitudes add up to less.  A NaN or infinite value or key makes the states after it
// odd, a query or cotangent those before it: of the two ends, and of the two sums over a chunk's tokens, each is formed from one
// side alone, so that gradients between a state and a cotangent that are both finite are, too.  grid (nm, Hv, B).  22 us at
// B=4, T=4096, Hv=32, 9 at B=1, T=2047 (and 5 for the sums of one decay per head): latency, a workgroup's loads, sums and one
// barrier after the other.
template <int MARK>
__global__ __launch_bounds__(64 * MARK) void dg_kernel(const DecayGrad a) {
    __shared__ double A[MARK], B[MARK], red[MARK], D0, D1;
    __shared__ float absA[MARK], absB[MARK];
    __shared__ int anew[MARK];
    const int m = blockIdx.x, h = blockIdx.y, b = blockIdx.z, l = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t heads = (int64_t)a.B * a.Hv, head = (int64_t)b * a.Hv + h;
    const int n = min(MARK, a.nc - m * MARK), c = m * MARK + w;  // chunks here, the wave's
    const int64_t t = (int64_t)c * C + l, last = (int64_t)c * C + C - 1 - l;
    const bool in = w < n && t < a.T;
    double xa = 0., xb = 0., x = 0.;  // a of token `last`, b and the pairs of token t
    if (w < n && last < a.T)
        for (int s = 0; s < a.slices; ++s) xa += (double)a.a[(s * heads + head) * a.T + last];
    if (in) {
        for (int s = 0; s < a.slices; ++s) xb += (double)a.b[(s * heads + head) * a.T + t];
        for (int s = 0; s < a.cross_slices; ++s) x += (double)a.cross[(s * heads + head) * a.T + t];
    }
    double end = 0.;
    if (m == a.nm - 1 && a.dlast) {
        const float *const p = a.dlast + head * a.size, *const q = a.last + head * a.size;
#pragma unroll 8
        for (int i = threadIdx.x; i < (int)a.size; i += 64 * MARK) end = fma((double)p[i], (double)q[i], end);
        end = block_sum(end, red, MARK);
    }
    if (w < 2) {
        const int at = m + w;
        double e = 0.;
        if (at >= a.mark0 && at < a.nm)
            for (int i = l; i < a.parts; i += 64) e += a.ends[(head * a.nm + at) * a.parts + i];
        e = wave_prefix_sum(e);
        if (l == 63) (w ? D1 : D0) = at < a.nm ? e : end;
    }
    const float fa = ops::group_sum<64>((float)fabs(xa)), fb = ops::group_sum<64>((float)fabs(xb));
    xa = wave_prefix_sum(xa);
    xb = wave_prefix_sum(xb);
    if (l == 63) {
        A[w] = xa;
        B[w] = xb;
        absA[w] = fa;
        absB[w] = fb;
        anew[w] = w < n && a.decays[(head * a.nc + c) * DECAYS + 3 * C - 1] < a.none;  // e^{G_C}
    }
    __syncthreads();
    double from_start = 0., from_end = 0., D = D0;
    float size_start = 0.f, size_end = 0.f, size = fabsf((float)D0);
    for (int i = 0; i < n && i <= w; ++i) {
        from_start = anew[i] ? 0. : D - A[i];
        size_start = anew[i] ? 0.f : size + absA[i];
        D = from_start + B[i];
        size = size_start + absB[i];
    }
    D = D1;
    size = fabsf((float)D1);
    for (int i = n - 1; i >= w; --i) {
        from_end = anew[i] ? 0. : D - B[i];
        size_end = anew[i] ? 0.f : size + absB[i];
        D = from_end + A[i];
        size = size_end + absA[i];
    }
    const bool start = isfinite(from_start) && (size_start <= size_end || !isfinite(from_end));
    // a from t on, b before t
    x += (start ? from_start : from_end) + __shfl(xa, C - 1 - l) + dpp_mov_f64<0x138>(xb);
    if (!a.per_head) {
        if (in) store_from_f32(a.dg, (b * (int64_t)a.T + t) * a.Hv + h, (float)x, a.dt);
        return;
    }
    x = block_sum(in ? x : 0., red, MARK);
    if (threadIdx.x == 0) a.sums[((int64_t)h * a.B + b) * a.nm + m] = x;
}

// One decay per head: the sums over n stretches of all sequences, in a fixed order.
__global__ __launch_bounds__(NT) void dg_head_kernel(const double *sums, void *dg, int64_t n, int dt) {
    __shared__ double red[NT / 64];
    double x = 0.;
    for (int64_t i = threadIdx.x; i < n; i += NT) x += sums[blockIdx.x * n + i];
    x = block_sum(x, red, NT / 64);
    if (threadIdx.x == 0) store_from_f32(dg, blockIdx.x, (float)x, dt);
}

// One token: y = scale S' q, S' = e^g S + v k^T, in place.  `lanes` lanes share a row of the state, V channels each at a time,
// and walk STEP_ROWS rows side by side, all of whose loads are under way before the first is used: the state, read and
// written once, is the kernel's traffic.  64 sequences of 32 states of 128 x 128: 268 MB in 52.8 us, 5.1 TB/s, what a copy
// reaches (44 us where the same states come again and part of them lies in the Infinity Cache).  One channel at a time, for states
// at any address: 66 us against 45.
constexpr int STEP_ROWS = 4;
struct Step {
    const void *q, *k, *v;
    Gate g;
    float *state;
    void *y;
    int Hk, Hv, Dk, Dv, dt, lanes;
    float scale;
};
template <int V>
__global__ __launch_bounds__(NT) void step_kernel(const Step a) {
    const int lanes = a.lanes, lane = threadIdx.x & (lanes - 1), rows = NT / lanes;
    const int row0 = blockIdx.x * rows * STEP_ROWS + threadIdx.x / lanes, h = blockIdx.y, b = blockIdx.z;
    const int64_t hv = (int64_t)b * a.Hv + h, hk = (int64_t)b * a.Hk + h / (a.Hv / a.Hk);
    const float f = __builtin_amdgcn_exp2f(a.g.load(b, 0, h) * (float)LOG2E);
    float *const s = a.state + hv * a.Dv * a.Dk;
    float y[STEP_ROWS] = {}, v[STEP_ROWS];
#pragma unroll
    for (int i = 0; i < STEP_ROWS; ++i) v[i] = load_as_f32(a.v, hv * a.Dv + min(row0 + i * rows, a.Dv - 1), a.dt);
    for (int c = lane * V; c < a.Dk; c += lanes * V) {
        float x[STEP_ROWS][V], q[V], k[V];
#pragma unroll
        for (int i = 0; i < STEP_ROWS; ++i) ops::loadv<V>(s, (int64_t)min(row0 + i * rows, a.Dv - 1) * a.Dk + c, DT_F32, x[i]);
        ops::loadv<V>(a.q, hk * a.Dk + c, a.dt, q);
        ops::loadv<V>(a.k, hk * a.Dk + c, a.dt, k);
#pragma unroll
        for (int i = 0; i < STEP_ROWS; ++i) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x[i][j] = fmaf(v[i], k[j], f * x[i][j]);
                y[i] = fmaf(x[i][j], q[j], y[i]);
            }
            if (row0 + i * rows < a.Dv) ops::storev<V>(s, (int64_t)(row0 + i * rows) * a.Dk + c, DT_F32, x[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < STEP_ROWS; ++i) {
        for (int m = 1; m < lanes; m <<= 1) y[i] += __shfl_xor(y[i], m);
        const int row = row0 + i * rows;
        if (lane == 0 && row < a.Dv) store_from_f32(a.y, hv * a.Dv + row, y[i] * a.scale, a.dt);
    }
}

// ---------------------------------------------------------------------------------------------------- host

static int slices_of(int dk, int dv) { return (dv + cols_of(dk, dv) - 1) / cols_of(dk, dv); }

struct Plan {
    int nseg, cps, nc;  // segments, chunks of each, chunks of the sequence
};
// Segments: two workgroups for each compute unit (their LDS leaves room for no more), and at least four chunks of work for
// each, as a segment costs its state's way through memory and its part of the sums (a single sequence of 2047 tokens, 32 fp32
// heads: eight segments, the forward pass 81 us).
static Plan plan(int B, int T, int Hv, int Dk, int Dv) {
    const int64_t wgs = (int64_t)B * Hv * slices_of(Dk, Dv), nc = ((int64_t)T + C - 1) / C;
    int64_t want = (512 + wgs - 1) / wgs;
    if (want > (nc + 3) / 4) want = (nc + 3) / 4;
    if (want < 1) want = 1;
    const int64_t cps = (nc + want - 1) / want;
    return {(int)((nc + cps - 1) / cps), (int)cps, (int)nc};
}

static Ten ten(const void *p, const int64_t *st, int div) { return {p, st[0], st[1], st[2], div}; }

static int slot(int dk, int dv) { return (dk <= 64 ? 0 : dk <= 128 ? 1 : 2) + (dk % 8 || dv % 8 ? 3 : 0); }

static int run_pass(Pass a, Kind kind, hipStream_t st) {
    static const char *const names[] = {"linatt_fwd", "linatt_dq", "linatt_dk", "linatt_dv"};
    a.slices = slices_of(a.dk, a.dv);
    {
        Timed tm(names[kind], st);
        constexpr decltype(&pass_d64) run[] = {pass_d64, pass_d128, pass_d256, pass_odd64, pass_odd128, pass_odd256};
        run[slot(a.dk, a.dv)](a, kind, st);
    }
    return check_launch(st, names[kind]);
}

// The states entering each segment (nseg > 1), from s0 on (reverse: the cotangents, from the end).
static int scan_width(int64_t size) { return size % 4 ? 1 : 4; }
template <bool REV>
static int run_segments(Seg a, const float *s0, hipStream_t st) {
    const int cols = seg_cols(a.dk, a.dv, a.dt);
    a.slices = (a.dv + cols - 1) / cols;
    {
        Timed tm(REV ? "linatt_segments_rev" : "linatt_segments", st);
        constexpr decltype(&seg_d64) run[] = {seg_d64, seg_d128, seg_d256, seg_odd64, seg_odd128, seg_odd256};
        run[slot(a.dk, a.dv)](a, REV, st);
    }
    const int rc = check_launch(st, "linear attention (segments)");
    if (rc) return rc;
    const int64_t size = (int64_t)a.dk * a.dv;
    {
        Timed tm("linatt_scan", st);
        const int per = NT * scan_width(size);
        const dim3 grid((unsigned)((size + per - 1) / per), (unsigned)(a.B * a.Hv));
        if (scan_width(size) == 4)
            hipLaunchKernelGGL((scan_kernel<REV, 4>), grid, dim3(NT), 0, st, a.s, a.decay, s0, a.nseg, size);
        else
            hipLaunchKernelGGL((scan_kernel<REV, 1>), grid, dim3(NT), 0, st, a.s, a.decay, s0, a.nseg, size);
    }
    return check_launch(st, "linear attention (scan)");
}

struct Sizes {
    size_t decays, state, decay, saved, part, dot, cross, marks, ends, sums, bwd;
    int nm, parts;
};
// value heads of a key head whose dq and dk are added after the passes: all, or the pairs of pair_heads()
static bool pair_heads(int r, int Dv, int dtype) { return dtype == DT_BF16 && Dv <= 128 && r % 2 == 0; }

static Sizes sizes(int B, int T, int Hk, int Hv, int Dk, int Dv, int dtype = DT_F32) {
    const Plan p = plan(B, T, Hv, Dk, Dv);
    Sizes s{};
    s.decays = align_up256((size_t)B * Hv * p.nc * DECAYS * sizeof(float));
    if (p.nseg > 1) {
        s.state = align_up256((size_t)B * Hv * p.nseg * Dk * Dv * sizeof(float));
        s.decay = align_up256((size_t)B * Hv * p.nseg * sizeof(float));
    }
    s.saved = s.decays + s.state;
    const int group = Hv / Hk / (pair_heads(Hv / Hk, Dv, dtype) ? 2 : 1);
    if (group > 1) s.part = align_up256((size_t)B * T * Hk * group * Dk * sizeof(float));
    const size_t rows = (size_t)B * Hv * T * sizeof(float);
    s.dot = align_up256(rows * slices_of(Dv, Dk));
    s.cross = align_up256(rows * slices_of(Dk, Dv));
    // of the passes that write dq and dk, whose K' are the value channels
    const int slices = slices_of(Dv, Dk);
    const int mark = mark_of(dtype != DT_BF16);
    s.nm = (p.nc + mark - 1) / mark;
    s.parts = slices * waves_of(Dv, Dk, dtype);
    const size_t marks = (size_t)B * Hv * s.nm;
    s.marks = align_up256(marks * slices * rows_of(Dv) * cols_of(Dv, Dk) * sizeof(float));
    s.ends = align_up256(marks * s.parts * sizeof(double));
    s.sums = align_up256(marks * sizeof(double));
    s.bwd = s.state + s.decay + s.part + 2 * s.dot + s.cross + s.marks + s.ends + s.sums;
    return s;
}

// What whole sequences and single tokens share.
static int check_sizes(int B, int T, int Hk, int Hv, int Dk, int Dv, int dtype, int g_dtype) {
    if (B < 0 || T < 0) return fail(GDN_ERR_INVALID, "B and T must be >= 0");
    if (Hk <= 0 || Hv <= 0 || Dk <= 0 || Dv <= 0) return fail(GDN_ERR_INVALID, "head counts and sizes must be positive");
    if (Hv % Hk) return fail(GDN_ERR_INVALID, "the key heads (%d) must divide the value heads (%d)", Hk, Hv);
    for (int d : {dtype, g_dtype})
        if (d != GDN_F32 && d != GDN_BF16 && d != GDN_F16) return fail(GDN_ERR_INVALID, "unknown dtype code");
    if (Dk > MAX_D || Dv > MAX_D) return fail(GDN_ERR_UNSUPPORTED, "heads of more than %d channels are not supported", MAX_D);
    return 0;
}

static int check(const int64_t *strides, int B, int T, int Hk, int Hv, int Dk, int Dv, int dtype, int g_dtype) {
    const int rc = check_sizes(B, T, Hk, Hv, Dk, Dv, dtype, g_dtype);
    if (rc) return rc;
    for (int i = 0; strides && i < 9; i += 3)
        if (strides[i + 1] < 0 || strides[i + 1] >= 1 << 22)  // a chunk's rows are addressed in 32 bits
            return fail(GDN_ERR_UNSUPPORTED, "tokens of q, k and v must be less than 2^22 elements apart");
    if ((int64_t)B * Hv > 65535) return fail(GDN_ERR_UNSUPPORTED, "more than 65535 heads over the batch");
    if ((int64_t)Hv * (Dk > Dv ? Dk : Dv) >= 1 << 22) return fail(GDN_ERR_UNSUPPORTED, "a token of more than 2^22 elements");
    if ((int64_t)B * Hv * T * (Dk > Dv ? Dk : Dv) >= (int64_t)1 << 39)  // grids of 2^31 workgroups
        return fail(GDN_ERR_UNSUPPORTED, "2^39 elements or more over the value heads");
    return 0;
}

}  // namespace la
}  // namespace gdn

using namespace gdn;

extern "C" size_t gdn_linatt_saved_bytes(int B, int T, int Hk, int Hv, int Dk, int Dv) {
    if (B <= 0 || T <= 0 || Hk <= 0 || Hv <= 0 || Dk <= 0 || Dv <= 0) return 0;
    const la::Sizes s = la::sizes(B, T, Hk, Hv, Dk, Dv);
    return s.saved + s.decay;
}
extern "C" size_t gdn_linatt_bwd_workspace_bytes(int B, int T, int Hk, int Hv, int Dk, int Dv, int dtype) {
    if (B <= 0 || T <= 0 || Hk <= 0 || Hv <= 0 || Dk <= 0 || Dv <= 0) return 0;
    return la::sizes(B, T, Hk, Hv, Dk, Dv, dtype).bwd;
}

extern "C" int gdn_linatt_fwd(const void *q, const void *k, const void *v, const void *g, const float *state0, void *y,
                              float *state_T, void *saved, size_t saved_bytes, const int64_t *strides, int B, int T, int Hk,
                              int Hv, int Dk, int Dv, float scale, int dtype, int g_dtype, void *stream) {
    clear_error();
    int rc = la::check(strides, B, T, Hk, Hv, Dk, Dv, dtype, g_dtype);
    if (rc) return rc;
    if (B == 0) return GDN_OK;
    if (T == 0) return fail(GDN_ERR_INVALID, "T must be positive");
    if (!q || !k || !v || !g || !y || !strides) return fail(GDN_ERR_INVALID, "null pointer");
    const la::Plan pl = la::plan(B, T, Hv, Dk, Dv);
    const la::Sizes sz = la::sizes(B, T, Hk, Hv, Dk, Dv);
    if (saved_bytes < sz.saved + sz.decay || !saved)
        return fail(GDN_ERR_WORKSPACE, "saved buffer of %zu bytes is smaller than the %zu bytes required", saved_bytes,
                    sz.saved + sz.decay);
    float *decays = static_cast<float *>(saved), *states = reinterpret_cast<float *>(static_cast<char *>(saved) + sz.decays);
    float *seg_decay = reinterpret_cast<float *>(static_cast<char *>(saved) + sz.saved);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int r = Hv / Hk;
    const la::Gate gate{g, strides[9], strides[10], strides[11], g_dtype};
    {
        Timed tm("linatt_decays", st);
        const int64_t waves = (int64_t)B * Hv * pl.nc;
        hipLaunchKernelGGL(la::decay_kernel, grid_of((waves + 3) / 4), dim3(la::NT), 0, st, gate, decays, B, T, Hv, pl.nc);
    }
    rc = check_launch(st, "linear attention (decays)");
    if (rc) return rc;
    la::Pass p{};
    p.Q = la::ten(q, strides, r);
    p.K = la::ten(k, strides + 3, r);
    p.V = la::ten(v, strides + 6, 1);
    p.decays = decays;
    p.B = B; p.T = T; p.Hv = Hv; p.dk = Dk; p.dv = Dv; p.nseg = pl.nseg; p.cps = pl.cps; p.nc = pl.nc;
    p.dt = p.o_dt = dtype;
    p.scale = scale;
    p.o = y;
    p.s_in = state0;
    p.s_head = (int64_t)Dk * Dv;
    p.s_out = state_T;
    if (pl.nseg > 1) {
        const la::Seg a{p.K, p.V, decays, states, seg_decay, B, T, Hv, Dk, Dv, 0, pl.nseg, pl.cps, pl.nc, dtype, scale};
        rc = la::run_segments<false>(a, state0, st);
        if (rc) return rc;
        p.s_in = states;
        p.s_seg = p.s_head;
        p.s_head *= pl.nseg;
    }
    return la::run_pass(p, la::Y, st);
}

extern "C" int gdn_linatt_bwd(const void *q, const void *k, const void *v, const void *g, const float *state0,
                              const float *state_T, const void *saved, size_t saved_bytes, const void *dy,
                              const float *dstate_T, void *dq, void *dk, void *dv, void *dg, float *dstate0, void *workspace,
                              size_t workspace_bytes, const int64_t *strides, int B, int T, int Hk, int Hv, int Dk, int Dv,
                              float scale, int g_per_head, int dtype, int g_dtype, void *stream) {
    clear_error();
    int rc = la::check(strides, B, T, Hk, Hv, Dk, Dv, dtype, g_dtype);
    if (rc) return rc;
    if (B == 0) return GDN_OK;
    if (T == 0) return fail(GDN_ERR_INVALID, "T must be positive");
    if (!q || !k || !v || !g || !dy || !dq || !dk || !dv || !dg || !strides || (dstate_T && !state_T))
        return fail(GDN_ERR_INVALID, "null pointer");
    const la::Plan pl = la::plan(B, T, Hv, Dk, Dv);
    const la::Sizes sz = la::sizes(B, T, Hk, Hv, Dk, Dv, dtype);
    if (!saved || saved_bytes < sz.saved + sz.decay)
        return fail(GDN_ERR_INVALID, "the saved buffer written by gdn_linatt_fwd (%zu bytes) is required", sz.saved + sz.decay);
    const float *decays = static_cast<const float *>(saved);
    const float *states = reinterpret_cast<const float *>(static_cast<const char *>(saved) + sz.decays);
    if (!workspace || workspace_bytes < sz.bwd)
        return fail(GDN_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %zu bytes required", workspace_bytes, sz.bwd);
    char *ws = static_cast<char *>(workspace);
    const auto take = [&ws](size_t bytes) {
        float *p = reinterpret_cast<float *>(ws);
        ws += bytes;
        return p;
    };
    float *ds = take(sz.state), *decay = take(sz.decay), *part = take(sz.part);
    float *sa = take(sz.dot), *sb = take(sz.dot), *cross = take(sz.cross);
    float *marks = take(sz.marks);
    double *ends = reinterpret_cast<double *>(take(sz.ends)), *sums = reinterpret_cast<double *>(take(sz.sums));
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int r = Hv / Hk;
    const int64_t dys[3] = {(int64_t)T * Hv * Dv, (int64_t)Hv * Dv, Dv}, size = (int64_t)Dk * Dv;
    const la::Ten tq = la::ten(q, strides, r), tk = la::ten(k, strides + 3, r);
    const la::Ten tv = la::ten(v, strides + 6, 1), tdy = la::ten(dy, dys, 1);
    la::Pass p{};
    p.decays = decays;
    p.B = B; p.T = T; p.Hv = Hv; p.nseg = pl.nseg; p.cps = pl.cps; p.nc = pl.nc;
    p.dt = dtype;
    p.scale = scale;
    p.marks = marks;
    p.ends = ends;
    p.nm = sz.nm;
    p.mark0 = state0 ? 0 : 1;
    const int64_t n = (int64_t)B * T * Hk * Dk;
    // value heads that share a key head: two to a workgroup, or each for itself, the rest added afterwards
    const int pair = la::pair_heads(r, Dv, dtype), group = pair ? r / 2 : r;
    const auto grouped = [&](void *out, la::Kind kind) {
        p.pair = pair;
        p.o = group > 1 ? part : out;
        p.o_dt = group > 1 ? GDN_F32 : dtype;
        const int e = la::run_pass(p, kind, st);
        if (e || group == 1) return e;
        {
            Timed tm("linatt_group", st);
            hipLaunchKernelGGL(la::group_kernel, grid_of((n + la::NT - 1) / la::NT), dim3(la::NT), 0, st, part, out, n, group, Dk,
                               dtype);
        }
        return check_launch(st, "linear attention (groups)");
    };
    // dq = LA(dy, v, k): the forward's states, read as [k' = value channel][v' = key channel]
    p.Q = tdy; p.K = tv; p.V = tk; p.X = tq;
    p.dk = Dv; p.dv = Dk;
    p.s_t = 1;
    p.s_head = size * (pl.nseg > 1 ? pl.nseg : 1);
    p.s_seg = size;
    p.s_in = pl.nseg > 1 ? states : state0;
    p.dot = sa;
    rc = grouped(dq, la::DQ);
    if (rc) return rc;
    const float *s_in = dstate_T;
    if (pl.nseg > 1) {
        const la::Seg a{tq, tdy, decays, ds, decay, B, T, Hv, Dk, Dv, 0, pl.nseg, pl.cps, pl.nc, dtype, scale};
        rc = la::run_segments<true>(a, dstate_T, st);
        if (rc) return rc;
        s_in = ds;
    }
    // dk = RLA(v, dy, q)
    p.Q = tv; p.K = tdy; p.V = tq; p.X = tk;
    p.s_in = s_in;
    p.dot = sb;
    rc = grouped(dk, la::DK);
    if (rc) return rc;
    // dv = RLA(k, q, dy)
    p.Q = tk; p.K = tq; p.V = tdy; p.X = tv;
    p.pair = 0;
    p.dk = Dk; p.dv = Dv;
    p.s_t = 0;
    p.dot = cross;
    p.o = dv;
    p.o_dt = dtype;
    p.s_out = dstate0;
    rc = la::run_pass(p, la::DV, st);
    if (rc) return rc;
    const la::DecayGrad d{sa, sb, cross, decays, dstate_T, state_T, ends, dg, sums, B, T, Hv, la::slices_of(Dv, Dk),
                          la::slices_of(Dk, Dv), g_per_head != 0, g_dtype, pl.nc, sz.nm, p.mark0, sz.parts,
                          // an eighth of the relative errors of a and b
                          dtype == GDN_BF16 ? 0x1p-20f : 0x1p-26f, size};
    {
        Timed tm("linatt_dg", st);
        const dim3 grid((unsigned)sz.nm, (unsigned)Hv, (unsigned)B);
        constexpr int M16 = la::mark_of(false), M32 = la::mark_of(true);
        if (dtype == GDN_BF16) hipLaunchKernelGGL(la::dg_kernel<M16>, grid, dim3(64 * M16), 0, st, d);
        else hipLaunchKernelGGL(la::dg_kernel<M32>, grid, dim3(64 * M32), 0, st, d);
        if (g_per_head)
            hipLaunchKernelGGL(la::dg_head_kernel, dim3((unsigned)Hv), dim3(la::NT), 0, st, sums, dg, (int64_t)B * sz.nm, g_dtype);
    }
    return check_launch(st, "linear attention (dg)");
}

extern "C" int gdn_linatt_step(const void *q, const void *k, const void *v, const void *g, float *state, void *y, int64_t gs_b,
                               int64_t gs_h, int B, int Hk, int Hv, int Dk, int Dv, float scale, int dtype, int g_dtype,
                               void *stream) {
    clear_error();
    const int rc = la::check_sizes(B, 1, Hk, Hv, Dk, Dv, dtype, g_dtype);
    if (rc) return rc;
    if (B > 65535 || Hv > 65535) return fail(GDN_ERR_UNSUPPORTED, "more than 65535 sequences or heads");
    if (B == 0) return GDN_OK;
    if (!q || !k || !v || !g || !state || !y) return fail(GDN_ERR_INVALID, "null pointer");
    const bool vec = Dk % 4 == 0 && aligned_to(q, 16) && aligned_to(k, 16) && aligned_to(state, 16);
    la::Step a{q, k, v, {g, gs_b, 0, gs_h, g_dtype}, state, y, Hk, Hv, Dk, Dv, dtype, 1, scale};
    while (a.lanes < 64 && a.lanes * (vec ? 4 : 1) < Dk) a.lanes *= 2;
    const int rows = la::NT / a.lanes * la::STEP_ROWS;
    const dim3 grid((unsigned)((Dv + rows - 1) / rows), (unsigned)Hv, (unsigned)B);
    hipStream_t st = static_cast<hipStream_t>(stream);
    {
        Timed tm("linatt_step", st);
        if (vec) hipLaunchKernelGGL(la::step_kernel<4>, grid, dim3(la::NT), 0, st, a);
        else hipLaunchKernelGGL(la::step_kernel<1>, grid, dim3(la::NT), 0, st, a);
    }
    return check_launch(st, "gdn_linatt_step");
}
