// Operands of the matrix products laid out in 16-bit terms along the contraction, straight or transposed, for gfx950.
//
// A number of more bits than a 16-bit type holds is a sum of terms, each the rounding of what the earlier ones leave:
// fp32 = 2 fp16 terms up to 2^-22 of it, or 3 bf16 terms.  fp16 has 5 bits of exponent, so a whole matrix is first
// multiplied by the power of two that takes its largest magnitude to 2^14: a number is then off by 2^-39 of the largest at most.
#include "gdn_common.h"
#include "gdn_terms.h"
#include "gdn_vec.h"

namespace gdn {
namespace mm {

constexpr int NT = 256;

// The caller's row for row r, or -1 where it counts as zeros.
__device__ __forceinline__ int64_t row_of(const Source &s, int64_t r) {
    if (s.index) return r < *s.count ? s.index[r] : -1;
    return s.targets && s.targets[r] == s.ignore ? -1 : r;
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}

__device__ __forceinline__ float magnitude(float x) {
    const float a = fabsf(x);
    return a <= 3.4028234e38f ? a : 0.f;  // neither infinite nor NaN
}

struct Pair { Source s[2]; };

// A wave to a row, 2048 elements at a time; the first PARTS workgroups for the first matrix.
template <int DT>
__global__ __launch_bounds__(1024) void maxima_kernel(const Pair both, float *part) {
    constexpr int WAVES = 16, U = 4;
    __shared__ float red[WAVES];
    const int which = blockIdx.x / PARTS, block = blockIdx.x % PARTS;
    const Source &s = both.s[which];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float m = 0.f;
    for (int64_t r = block * WAVES + w; r < s.rows; r += PARTS * WAVES) {
        const int64_t at = row_of(s, r);
        if (at < 0) continue;
        for (int64_t c = lane * 8; c < s.cols; c += U * 512) {
            float x[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) ops::load_first<8, DT>(s.p, at * s.ld + c + u * 512, s.cols - c - u * 512, x[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, magnitude(x[u][j]));
        }
    }
    m = wave_max(m);
    if (lane == 0) red[w] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 1; i < WAVES; ++i) m = fmaxf(m, red[i]);
        part[blockIdx.x] = m;
    }
}

// The exponent that takes m to [2^top, 2^(top + 1)), 0 for 0.
__device__ __forceinline__ int exponent_to(float m, int top) {
    int e = 0;
    if (m > 0.f) (void)frexpf(m, &e);  // m in [2^(e - 1), 2^e)
    return m > 0.f ? top + 1 - e : 0;
}

__global__ __launch_bounds__(64) void exponents_kernel(const float *part, int top, int *exps, float *most) {
    const int i = blockIdx.x;
    if (i < 2 && !exps) return;
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < PARTS / 64; ++k) m = fmaxf(m, part[i * PARTS + k * 64 + threadIdx.x]);
    m = wave_max(m);
    if (threadIdx.x == 0) {
        if (i < 2) exps[i] = exponent_to(m, top);
        else most[0] = m;
    }
}

// A wave to a row of fp32 numbers.
__global__ __launch_bounds__(NT) void row_exponents_kernel(const Source s, int top, int *exps) {
    const int lane = threadIdx.x & 63;
    const int64_t r = block_index() * (NT / 64) + (threadIdx.x >> 6);
    if (r >= s.rows) return;
    const int64_t at = row_of(s, r);
    float m = 0.f;
    if (at >= 0)
        for (int64_t c = lane * 8; c < s.cols; c += 512) {
            float x[8];
            ops::load_first<8, DT_F32>(s.p, at * s.ld + c, s.cols - c, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, magnitude(x[j]));
        }
    m = wave_max(m);
    if (lane == 0) exps[r] = exponent_to(m, top);
}

// The next term of y, which keeps the rest: rounded (fp16) or cut off (bf16: three take the 24 bits of an fp32 number as they
// are, and none becomes infinite).  An infinite or NaN number is its first term.
template <bool F16>
__device__ __forceinline__ uint16_t next_term(float &y) {
    uint16_t b;
    float back;
    if constexpr (F16) {
        const __half h = __float2half(y);
        b = __half_as_ushort(h);
        back = __half2float(h);
    } else {
        b = (uint16_t)(__float_as_uint(y) >> 16 | (y != y ? 0x40u : 0u));
        back = bf16_to_f32(b);
    }
    y = fabsf(back) <= 3.4028234e38f ? y - back : 0.f;
    return b;
}

__device__ __forceinline__ uint4 pack8(const uint16_t (&b)[8]) {
    return make_uint4(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16, b[4] | (uint32_t)b[5] << 16,
                      b[6] | (uint32_t)b[7] << 16);
}

// Eight elements of a row to a thread.
template <bool F16, int DT>
__global__ __launch_bounds__(NT) void terms_kernel(const Source s, int slots, const int *exps, int which, uint16_t *dst,
                                                   int64_t kp) {
    const int64_t i = block_index() * NT + threadIdx.x;
    const uint32_t per = (uint32_t)(kp / 8);
    const int64_t r = i >> 32 ? i / per : (uint32_t)i / per, c = (i - r * per) * 8;
    if (r >= s.rows) return;
    const int e = !exps ? 0 : exps[which == EACH_ROW ? r : which];
    float x[8], whole[8];
    const int64_t at = row_of(s, r);
    ops::load_first<8, DT>(s.p, at * s.ld + c, at < 0 ? 0 : s.cols - c, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = whole[j] = ldexpf(x[j], e);
    for (int t = 0; t < slots; ++t) {
        uint16_t b[8];
        if (F16 && t == 2) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = ldexpf(whole[j], -LOW);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = next_term<F16>(x[j]);
        *reinterpret_cast<uint4 *>(dst + r * (kp * slots) + t * kp + c) = pack8(b);
    }
}

// 64 x 64 elements to a workgroup, turned over in LDS.
template <bool F16, int DT>
__global__ __launch_bounds__(NT) void across_kernel(const Source s, int slots, const int *exps, int which, const Factors f,
                                                    uint16_t *dst, int64_t kp, int64_t tiles_c, int64_t tiles) {
    __shared__ float tile[64][65];
    const int64_t t0 = block_index();
    if (t0 >= tiles) return;
    const int64_t r0 = t0 / tiles_c * 64, c0 = t0 % tiles_c * 64;
    const int e = exps ? exps[which] : 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int rl = h * 32 + threadIdx.x / 8, cl = threadIdx.x % 8 * 8;
        const int64_t r = r0 + rl, c = c0 + cl;
        float x[8];
        const int64_t at = r < s.rows ? row_of(s, r) : -1;
        ops::load_first<8, DT>(s.p, at * s.ld + c, at < 0 ? 0 : s.cols - c, x);
        float by = 1.f;
        if (f.row && at >= 0) {
            const float most = f.by[0];
            by = most > 0.f ? f.row[r] / most : f.row[r];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) tile[rl][cl + j] = at < 0 ? 0.f : ldexpf(x[j] * by, e);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int cl = h * 32 + threadIdx.x / 8, rl = threadIdx.x % 8 * 8;
        if (c0 + cl >= s.cols) continue;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = tile[rl + j][cl];
        uint16_t *to = dst + (c0 + cl) * (kp * slots) + r0 + rl;
        for (int t = 0; t < slots; ++t) {
            uint16_t b[8];
            if (F16 && t == 2) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = ldexpf(tile[rl + j][cl], -LOW);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = next_term<F16>(x[j]);
            *reinterpret_cast<uint4 *>(to + t * kp) = pack8(b);
        }
    }
}

void maxima(const Source (&s)[2], float *part, hipStream_t st) {
    Timed tm("maxima", st);
    constexpr int64_t LONG = 8192;
    Pair p{{s[0], s[1]}};
    for (Source &m : p.s)
        if (m.ld == m.cols && !m.targets && !m.index && m.rows * m.cols % LONG == 0) {  // rows in one piece: of any length
            m.rows = m.rows * m.cols / LONG;
            m.ld = m.cols = LONG;
        }
    const dim3 grid(2 * PARTS), block(1024);
    if (s[0].dt == DT_F32) hipLaunchKernelGGL((maxima_kernel<DT_F32>), grid, block, 0, st, p, part);
    else if (s[0].dt == DT_BF16) hipLaunchKernelGGL((maxima_kernel<DT_BF16>), grid, block, 0, st, p, part);
    else hipLaunchKernelGGL((maxima_kernel<DT_F16>), grid, block, 0, st, p, part);
}

void exponents(const float *part, int top, int *exps, float *most, hipStream_t st) {
    hipLaunchKernelGGL(exponents_kernel, dim3(3), dim3(64), 0, st, part, top, exps, most);
}

void row_exponents(const Source &s, int top, int *exps, hipStream_t st) {
    Timed tm("row_exponents", st);
    hipLaunchKernelGGL(row_exponents_kernel, grid_of((s.rows + NT / 64 - 1) / (NT / 64)), dim3(NT), 0, st, s, top, exps);
}

#define GDN_TERMS(KERNEL, F16, DT, ...) hipLaunchKernelGGL((KERNEL<F16, DT>), grid, dim3(NT), 0, st, __VA_ARGS__)

void terms(const Source &s, int slots, bool f16, const int *exps, int which, void *dst, hipStream_t st) {
    Timed tm("terms", st);
    const int64_t kp = padded(s.cols);
    const dim3 grid = grid_of((s.rows * (kp / 8) + NT - 1) / NT);
#define GDN_STRAIGHT(F16, DT) GDN_TERMS(terms_kernel, F16, DT, s, slots, exps, which, static_cast<uint16_t *>(dst), kp)
    if (s.dt == DT_BF16) GDN_STRAIGHT(false, DT_BF16);  // never in fp16
    else if (s.dt == DT_F16 && f16) GDN_STRAIGHT(true, DT_F16);
    else if (s.dt == DT_F16) GDN_STRAIGHT(false, DT_F16);
    else if (f16) GDN_STRAIGHT(true, DT_F32);
    else GDN_STRAIGHT(false, DT_F32);
#undef GDN_STRAIGHT
}

void terms_across(const Source &s, int slots, bool f16, const int *exps, int which, const Factors &f, void *dst, hipStream_t st) {
    Timed tm("terms_across", st);
    const int64_t kp = padded(s.rows), tc = (s.cols + 63) / 64, tiles = kp / 64 * tc;
    const dim3 grid = grid_of(tiles);
#define GDN_ACROSS(F16, DT) GDN_TERMS(across_kernel, F16, DT, s, slots, exps, which, f, static_cast<uint16_t *>(dst), kp, tc, tiles)
    if (s.dt == DT_BF16) GDN_ACROSS(false, DT_BF16);
    else if (s.dt == DT_F16) GDN_ACROSS(true, DT_F16);
    else if (f16) GDN_ACROSS(true, DT_F32);
    else GDN_ACROSS(false, DT_F32);
#undef GDN_ACROSS
}
#undef GDN_TERMS

}  // namespace mm
}  // namespace gdn
