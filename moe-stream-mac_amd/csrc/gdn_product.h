// The matrix product of the operators that are not bound by memory: C[n][m] = sum_k B[n][k] A[m][k] with 16-bit operands
// that lie along the contraction, or one of them across it, 32-bit sums on the matrix cores, for gfx950.
//
// Whoever has another type or an odd size lays its operand out in a pass of its own (gdn_terms.h), which costs a percent or two
// of a large product and leaves one loop to make fast.  fp32 operands become sums of 16-bit terms, side by side along the
// contraction; the product then walks pairs of terms ("segments").
//
// A workgroup forms a BM x BN tile, BK = 64 at a time: rows of 128 bytes go from memory to LDS without passing through
// registers, two stages deep.  Chunk c of 16 bytes of row r lies in place c ^ (r / 2 & 7): sixteen rows of one chunk, which an
// LDS read serves at once, fill all 64 banks (with r & 7 half of the read cycles were conflicts).  The global addresses are
// permuted to that end, since LDS is filled in order.
//
// The barrier of a stage stands in its middle: by then all of its fragments are in registers, so after it the stage's LDS may be
// overwritten, and the next stage's fragments are read under the second half's products.  Loads thus have a whole stage to
// arrive, and no product waits for LDS.
//
// Lanes hold the columns of a matrix instruction's result and registers its rows: A's rows (m) run over registers, B's (n) over
// lanes.  Sums over m, such as those of a softmax over words, stay within a lane and its three partners 16 lanes apart.
//
// Measured, bf16: 8192 x 2048 x 8192 1.48 PFLOP/s, 8192 x 8192 x 2048 1.40 (a large library product 1.53).  The card lowers its
// clock under this load, to 1.9 GHz: with 32 x 32 x 16 instructions, which move twice the sums through registers, to 1.7 and
// 1.39 PFLOP/s.
#pragma once

#include "gdn_common.h"
#include "gdn_host.h"
#include "gdn_vec.h"

namespace gdn {
namespace mm {

typedef float acc_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 hf8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int BK = 64;

template <bool F16>
__device__ __forceinline__ acc_t mfma(u4 a, u4 b, acc_t c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hf8, a), __builtin_bit_cast(hf8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}

constexpr int PAIRS = 6;  // of terms, at most
// A matrix of `rows` rows, `ld` bytes apart, of `off[s]` bytes to the term that segment s takes.
struct Operand {
    const char *p;
    int64_t ld, rows;
    int64_t off[PAIRS];
    int64_t width;  // across the contraction: bytes of a row that may be read, a multiple of 16
};
struct Args {
    Operand a, b;
    int kit;     // BK-blocks of a term
    int nseg;    // 1 to PAIRS
    int splits;  // the nseg * kit blocks in this many parts (grid.z)
    int mt, nt;  // tiles
    // Sizes that only the device knows: `live` tokens count, of which these are those from live0 on.  They are b's rows, or with
    // live_k the length of the contraction; tiles and blocks behind them are not formed.
    const int *live;
    int64_t live0;
    int live_k;
    int across;    // the operand that lies across the contraction: 0, DOWN_A or DOWN_B
    int64_t down;  // its rows; its `rows` are columns then
};
struct Extent {
    int64_t rows_b, down;
    int nt, kit;
};
template <class S>
__device__ __forceinline__ Extent extent_of(const Args &g) {
    Extent x{g.b.rows, g.down, g.nt, g.kit};
    if (g.live) {
        const int64_t n = max((int64_t)0, (int64_t)*g.live - g.live0);
        if (g.live_k) {
            x.kit = (int)min((int64_t)g.kit, (n + BK - 1) / BK);
            x.down = min(g.down, n);
        } else {
            x.rows_b = min(g.b.rows, n);
            x.nt = (int)((x.rows_b + S::BN - 1) / S::BN);
        }
    }
    return x;
}

// BM x BN tile of WM x WN waves.
template <int BM_, int BN_, int WM_, int WN_, int PER_CU_>
struct Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NT = 64 * WM_ * WN_;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    static constexpr int A_BYTES = BM * BK * 2, STAGE = (BM + BN) * BK * 2, LDS = 2 * STAGE;
    static constexpr int STORE = WM * WN * 4096;  // LDS through which a wave's results leave, 4 KB each
    static constexpr int RA = BM * 8 / NT, RB = BN * 8 / NT;  // 16-byte loads of a thread for a stage
    static constexpr int PER_CU = PER_CU_;
    static constexpr int WAVES_EU = PER_CU_ * NT / 256;
    static_assert(RA >= 1 && RB >= 1 && TM % 4 == 0 && TN % 2 == 0 && TN >= 1, "tile");
};
// The lane, as a value that is worked out where it stands: what an epilogue derives from it would otherwise be kept in registers
// through the whole product, which has none to spare.
__device__ __forceinline__ int lane_here() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

// This wave's number, known to be the same for all its lanes.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

typedef Shape<256, 256, 2, 4, 1> Big;
typedef Shape<128, 128, 2, 2, 2> Mid;
typedef Shape<128, 64, 2, 2, 2> Few;
typedef Shape<128, 32, 2, 1, 3> One;

typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

// Workgroups go round the 8 XCDs in turn, and each XCD has an L2 of its own: it takes a run of neighbouring pieces of work.
__device__ __forceinline__ int run_of(int id, int total) {
    const int xcd = id & 7;
    return xcd * (total >> 3) + min(xcd, total & 7) + (id >> 3);
}

// A workgroup's first tile and its part of the contraction.  Where each workgroup has one tile of one part, the tiles of a part go
// to one XCD, or a few (`runs`): they share rows of both operands, which the parts do not.  513 x 1001 sums over 50001 words in 16
// parts, three pairs of terms: 232 us, 254 with the tiles of each part on all XCDs.
struct Part {
    int tile, z;
    bool runs;  // tiles are in order already
};
__device__ __forceinline__ Part part_of(const Args &g) {
    const int tiles = gridDim.x;
    if (g.splits == 1 || tiles != g.mt * g.nt) return {(int)blockIdx.x, (int)blockIdx.z, false};
    const int t = run_of(blockIdx.x + blockIdx.z * tiles, tiles * g.splits), z = t / tiles;
    return {t - z * tiles, z, true};
}

// Tile number id.  A run walks groups of 8 tiles along m, so that the tiles under way on an XCD share rows of both operands.
__device__ __forceinline__ void tile_of(int id, bool runs, int mt, int nt, int &tm, int &tn) {
    const int t = runs ? id : run_of(id, mt * nt);
    const int per = 8 * nt, g = t / per, first = g * 8, width = min(8, mt - first), r = t - g * per;
    tm = first + r % width;
    tn = r / width;
}

// An operand may also lie across the contraction (DOWN_A, DOWN_B): rows of m or n, one for each k, read as they are and turned by
// LDS reads that transpose 4 x 16 numbers.  32 bytes, what such a read takes of a row, lie in place (pair ^ down_swizzle(row)) of
// the row's, so that the 16 rows of one read fill all banks twice.  Rows behind the last (Extent::down of them) read as zeros;
// columns behind the last are whatever follows them, and nothing of them is stored.  2048 x 8192 x 8192: 1.44 PFLOP/s with A so.
enum : int { DOWN_A = 1, DOWN_B = 2 };
__device__ __forceinline__ int down_swizzle(int row) { return (row & 3) | (row >> 3 & 1) << 2; }
// The chunk of 16 bytes of a row that lies in place p.
__device__ __forceinline__ int down_chunk(int p, int row) { return ((p >> 1) ^ down_swizzle(row)) << 1 | (p & 1); }

// One operand's share of a workgroup's loads: ROWS rows of the tile (of m or n), or with DOWN their columns.
template <class S, int ROWS, bool DOWN>
struct Side {
    static constexpr int LOADS = ROWS * 8 / S::NT;                      // of a thread for a block
    static constexpr int LANES = ROWS / 8, ROUND = S::NT / (DOWN ? LANES : 8);  // DOWN: lanes to a row; rows to a load
    const char *p;       // of the block to load next
    int64_t rest;        // DOWN: bytes from p to the operand's end
    uint32_t at, at_odd; // this thread's offset in a block, DOWN also of odd loads
    uint32_t size, step; // bytes that loads may reach, none behind the last row; from one load's rows to the next one's

    // The tile's row (or column) r0 on of `rows`, block kk of a term at `off`; `down` rows along the contraction.
    __device__ __forceinline__ void start(const Operand &o, int64_t off, int64_t r0, int64_t rows, int kk, int64_t down) {
        const uint32_t ld = (uint32_t)o.ld;
        step = ROUND * ld;
        if constexpr (DOWN) {
            const int r = threadIdx.x / LANES, c = threadIdx.x % LANES;
            at = r * ld + down_chunk(c, r) * 16;
            at_odd = r * ld + down_chunk(c, r + ROUND) * 16;
            const int64_t from = (int64_t)kk * BK * o.ld + r0 * 2;
            p = o.p + off + from;
            rest = (down - 1) * o.ld + o.width - from;
        } else {
            const int r = threadIdx.x >> 3, c = threadIdx.x & 7;
            at = r * ld + ((c ^ (r >> 1 & 7)) << 4);
            p = o.p + off + r0 * o.ld + (int64_t)kk * (BK * 2);
            size = (uint32_t)(min((int64_t)ROWS, rows - r0) - 1) * ld + BK * 2;
        }
    }
    __device__ __forceinline__ void next(const Operand &o) {
        if constexpr (DOWN) {
            p += BK * o.ld;
            rest -= BK * o.ld;
        } else {
            p += BK * 2;
        }
    }
    // From the end of a term of kit blocks to the start of another, `off` bytes on.
    __device__ __forceinline__ void turn(const Operand &o, int64_t off, int kit) {
        if constexpr (DOWN) {
            p += off - (int64_t)kit * BK * o.ld;
            rest += (int64_t)kit * BK * o.ld;
        } else {
            p += off - (int64_t)kit * (BK * 2);
        }
    }
    // Load r of a block.
    __device__ __forceinline__ void load(char *__restrict__ dst, int r, int w) const {
#ifdef __HIP_DEVICE_COMPILE__  // the host's pass does not know buffer resources
        constexpr int RAW = 0x00020000;
        const uint32_t n = DOWN ? (uint32_t)min(max(rest, (int64_t)0), (int64_t)1 << 31) : size;
        const auto res = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), 0, n, RAW);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(res, (lvoid *)(dst + r * (S::NT * 16) + w * 1024), 16,
                                                 (DOWN && r % 2 ? at_odd : at) + r * step, 0, 0, 0);
#endif
    }
};

// A workgroup's walk over its tiles and their blocks: every gridDim.x-th tile from its first one on, each from block `first`
// to `end`.  It runs two blocks ahead of the products, over the border between two tiles too, so that the next tile's first
// loads are under way while results are written.
template <class S, int DOWN>
struct Loader {
    Side<S, S::BM, (DOWN & DOWN_A) != 0> a;
    Side<S, S::BN, (DOWN & DOWN_B) != 0> b;
    int left, seg_left, seg, tile, tiles, w;  // blocks left of the tile and of the segment
    bool runs;

    __device__ __forceinline__ void start(const Args &g, const Extent &x, int first, int end) {  // of a tile
        int tm, tn;
        tile_of(tile, runs, g.mt, x.nt, tm, tn);
        left = end - first;
        seg = first / x.kit;
        const int kk = first - seg * x.kit;
        seg_left = x.kit - kk;
        a.start(g.a, g.a.off[seg], (int64_t)tm * S::BM, g.a.rows, kk, x.down);
        b.start(g.b, g.b.off[seg], (int64_t)tn * S::BN, x.rows_b, kk, x.down);
    }
    // Loads [R0, R1) of a block's RA + RB.
    template <int R0, int R1>
    __device__ __forceinline__ void load(char *__restrict__ dst) const {
#pragma unroll
        for (int r = R0; r < R1; ++r) {
            if (r < S::RA) a.load(dst, r, w);
            else b.load(dst + S::A_BYTES, r - S::RA, w);
        }
    }
    // On to the next block; after the very last one it stays there, so that loads need no branch around them.
    __device__ __forceinline__ void next(const Args &g, const Extent &x, int first, int end) {
        if (left > 1) {
            a.next(g.a);
            b.next(g.b);
            --left;
            if (--seg_left == 0) {
                seg_left = x.kit;
                a.turn(g.a, g.a.off[seg + 1] - g.a.off[seg], x.kit);
                b.turn(g.b, g.b.off[seg + 1] - g.b.off[seg], x.kit);
                ++seg;
            }
        } else if (tile + (int)gridDim.x < tiles) {
            tile += gridDim.x;
            start(g, x, first, end);
        }
    }
};

// Every load into LDS has landed and every fragment read has returned, of all waves.
__device__ __forceinline__ void stage_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Tile i of 16 rows of an operand, 8 numbers along the contraction to a lane: 16 bytes of a row of the operand (at[k] for step k);
// or DOWN two reads of four rows each, at[0] the lane's place in a row of tile 0 and at[1] its swizzle, PITCH bytes a row.
template <bool DOWN, int PITCH>
__device__ __forceinline__ u4 fragment(const char *__restrict__ lds, const uint32_t (&at)[2], int k, int i) {
    if constexpr (DOWN) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) s4 lds_s4;
        const char *p = lds + at[0] + k * 32 * PITCH + ((uint32_t)(i * 32) ^ at[1]);
        const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)p);
        const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + 4 * PITCH));
        return __builtin_bit_cast(u4, (s8)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
        return *reinterpret_cast<const u4 *>(lds + at[k] + i * 16 * BK * 2);
    }
}

// A lane's places for `fragment`, from the operand's LDS on, for a wave whose rows begin at tile `first` (a multiple of `tiles`, 2,
// 4 or 8, that it has).
template <bool DOWN, int PITCH>
__device__ __forceinline__ void places(uint32_t (&at)[2], int lane, uint32_t base, int first) {
    if constexpr (DOWN) {
        const int row = 8 * (lane >> 4) + (lane >> 2 & 3);
        at[0] = base + row * PITCH + (lane & 3) * 8 + (first & ~7) * 32;
        at[1] = (uint32_t)(down_swizzle(row) ^ (first & 7)) * 32;
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            at[k] = base + (first * 16 + (lane & 15)) * BK * 2 + (((k * 4 + (lane >> 4)) ^ (lane >> 1 & 7)) << 4);
    }
}

// The fragments of a block: two steps of 32 along the contraction; A's rows in two halves.
template <class S, int DOWN>
struct Frags {
    static constexpr int H = S::TM / 2;
    static constexpr bool DA = (DOWN & DOWN_A) != 0, DB = (DOWN & DOWN_B) != 0;
    static constexpr int READ_A = DA ? 2 : 1, READ_B = DB ? 2 : 1;  // reads from LDS for a tile
    u4 lo[2][H], hi[2][H], b[2][S::TN];
    __device__ __forceinline__ void read_lo(const char *__restrict__ lds, const uint32_t (&at_a)[2], int k) {
#pragma unroll
        for (int i = 0; i < H; ++i) lo[k][i] = fragment<DA, S::BM * 2>(lds, at_a, k, i);
    }
    __device__ __forceinline__ void read_hi(const char *__restrict__ lds, const uint32_t (&at_a)[2], int k) {
#pragma unroll
        for (int i = 0; i < H; ++i) hi[k][i] = fragment<DA, S::BM * 2>(lds, at_a, k, H + i);
    }
    __device__ __forceinline__ void read_b(const char *__restrict__ lds, const uint32_t (&at_b)[2], int k) {
#pragma unroll
        for (int j = 0; j < S::TN; ++j) b[k][j] = fragment<DB, S::BN * 2>(lds, at_b, k, j);
    }
    template <bool F16>
    __device__ __forceinline__ void mul_lo(acc_t (&acc)[S::TM][S::TN], int k) const {
#pragma unroll
        for (int i = 0; i < H; ++i)
#pragma unroll
            for (int j = 0; j < S::TN; ++j) acc[i][j] = mfma<F16>(lo[k][i], b[k][j], acc[i][j]);
    }
    template <bool F16>
    __device__ __forceinline__ void mul_hi(acc_t (&acc)[S::TM][S::TN], int k) const {
#pragma unroll
        for (int i = 0; i < H; ++i)
#pragma unroll
            for (int j = 0; j < S::TN; ++j) acc[H + i][j] = mfma<F16>(hi[k][i], b[k][j], acc[H + i][j]);
    }
};

// First half of a block: the products of A's lower rows, while the rest of the block's fragments are read, one between two
// products, and the first product before them (its wait is for what the last half has read).
template <class S, bool F16, int DOWN>
__device__ __forceinline__ void first_half(const char *__restrict__ rd, const uint32_t (&at_a)[2], const uint32_t (&at_b)[2],
                                           Frags<S, DOWN> &f, acc_t (&acc)[S::TM][S::TN]) {
    constexpr int H = S::TM / 2, PRODUCTS = H * S::TN;
    constexpr int READS = S::TN * Frags<S, DOWN>::READ_B + 2 * H * Frags<S, DOWN>::READ_A;
    f.template mul_lo<F16>(acc, 0);
    f.read_b(rd, at_b, 1);
    f.read_hi(rd, at_a, 0);
    f.read_hi(rd, at_a, 1);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
#pragma unroll
    for (int i = 0; i < READS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        if (i < PRODUCTS - 1) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS, 0);
    __builtin_amdgcn_sched_barrier(0);
    f.template mul_lo<F16>(acc, 1);
    __builtin_amdgcn_sched_barrier(0);
}

// Second half: the products of A's upper rows, while the block after the next is loaded into this one's LDS and the next
// one's fragments are read in the place of those that no product needs any more.  A load takes the memory pipe 16 cycles for
// each of the workgroup's waves, so loads stand between products: in one run they held the products up.
template <class S, bool F16, int DOWN>
__device__ __forceinline__ void second_half(const char *__restrict__ rd, char *__restrict__ wr, const Loader<S, DOWN> &ld,
                                            const uint32_t (&at_a)[2], const uint32_t (&at_b)[2], Frags<S, DOWN> &f,
                                            acc_t (&acc)[S::TM][S::TN]) {
    constexpr int R = S::RA + S::RB, P = S::TM / 2 * S::TN;
    constexpr int READS = S::TM * Frags<S, DOWN>::READ_A, READS_B = S::TN * Frags<S, DOWN>::READ_B;
    ld.template load<0, R / 2>(wr);
    f.template mul_hi<F16>(acc, 0);
    f.read_lo(rd, at_a, 0);
    f.read_lo(rd, at_a, 1);
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x020, (R / 2 + P / 2 - 1) / (P / 2), 0);
        __builtin_amdgcn_sched_group_barrier(0x100, (READS + P / 2 - 1) / (P / 2), 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    ld.template load<R / 2, R>(wr);
    f.read_b(rd, at_b, 0);
    f.template mul_hi<F16>(acc, 1);
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, (READS_B + P / 2 - 1) / (P / 2), 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x020, (R - R / 2 + P / 2 - 1) / (P / 2), 0);
    }
    __builtin_amdgcn_sched_barrier(0);
}

template <class S>
__device__ __forceinline__ void clear(acc_t (&acc)[S::TM][S::TN]) {
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc[i][j] = acc_t{0.f, 0.f, 0.f, 0.f};
}

// Forms the workgroup's tiles and hands each to epilogue(tm, tn, acc).
// acc[i][j]: rows m = 16 i + 4 (lane / 16) + q of this wave's part for register q, column n = 16 j + lane % 16.
template <class S, bool F16, int DOWN = 0, class E>
__device__ __forceinline__ void products(const Args &g, const Extent &x, char *lds, E &&epilogue) {
    const int lane = threadIdx.x & 63, w = wave_index(), wm = w / S::WN, wn = w % S::WN;
    const int total = x.kit * g.nseg;
    const Part part = part_of(g);
    const int first = (int)((int64_t)total * part.z / g.splits), end = (int)((int64_t)total * (part.z + 1) / g.splits);
    const int blocks = end - first, mt = g.mt, nt = x.nt;
    Loader<S, DOWN> ld;
    ld.tile = part.tile;
    ld.runs = part.runs;
    ld.tiles = mt * nt;
    ld.w = w;
    if (ld.tile >= ld.tiles) return;
    uint32_t at_a[2], at_b[2];
    places<(DOWN & DOWN_A) != 0, S::BM * 2>(at_a, lane, 0, wm * S::TM);
    places<(DOWN & DOWN_B) != 0, S::BN * 2>(at_b, lane, S::A_BYTES, wn * S::TN);
    char *cur = lds, *other = lds + S::STAGE;
    if (blocks > 0) {  // else empty sums
        ld.start(g, x, first, end);
        ld.template load<0, S::RA + S::RB>(cur);
        ld.next(g, x, first, end);
        stage_barrier();
        ld.template load<0, S::RA + S::RB>(other);
        ld.next(g, x, first, end);
    }
    for (int t = part.tile; t < mt * nt; t += gridDim.x) {
        acc_t acc[S::TM][S::TN];
        clear<S>(acc);
        // read anew for each tile, so that their registers are free while results are written
        Frags<S, DOWN> f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            f.read_lo(cur, at_a, k);
            if (k < 1) f.read_b(cur, at_b, k);
        }
        for (int n = 0; n < blocks; ++n) {
            first_half<S, F16, DOWN>(cur, at_a, at_b, f, acc);
            stage_barrier();
            // after a tile's last block no product uses what this reads
            second_half<S, F16, DOWN>(other, cur, ld, at_a, at_b, f, acc);
            ld.next(g, x, first, end);
            char *c = cur;
            cur = other;
            other = c;
        }
        int tm, tn;
        tile_of(t, part.runs, mt, nt, tm, tn);
        epilogue(tm, tn, acc);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): no load into this LDS outlives the workgroup
}

// A wave's results leave through 4 KB of LDS, 32 rows of 128 bytes at a time (chunk c of 16 bytes of row r in place c ^ (r & 7)):
// eight lanes then store 128 bytes of one row, where registers hold 8 or 16 bytes of 32 rows.  At 8192 x 8192 x 2048 the
// product takes 215 us so, 231 to 280 with stores from registers.
__device__ __forceinline__ char *store_chunk(char *st, int row, int chunk) { return st + row * 128 + ((chunk ^ (row & 7)) << 4); }

// Rows [0, rows) of the 32 in LDS to memory, ld bytes apart (32 of them less than 2^32 bytes), of which the first `bytes` of
// each count.  to, ld, rows and bytes are the same for the whole wave.
__device__ __forceinline__ void store_rows(int lane, const char *st, char *to, uint32_t ld, int64_t rows, int64_t bytes,
                                           int elem) {
    typedef u4 any4 __attribute__((aligned(2)));
    const int c = lane & 7;
    asm volatile("" ::: "memory");  // what other lanes have put there: LDS keeps a wave's order, the compiler has to
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int r = t * 8 + (lane >> 3);
        const u4 v = *reinterpret_cast<const u4 *>(store_chunk(const_cast<char *>(st), r, c));
        if (r >= rows) continue;
        char *at = to + ((uint32_t)r * ld + (uint32_t)c * 16);
        if (c * 16 + 16 <= bytes) {
            *reinterpret_cast<any4 *>(at) = v;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // by 16 bits; an fp32 element is two
                const uint16_t h = (uint16_t)(v[j / 2] >> (16 * (j % 2)));
                if (c * 16 + j / (elem / 2) * elem + elem <= bytes) reinterpret_cast<uint16_t *>(at)[j] = h;
            }
        }
    }
    asm volatile("" ::: "memory");
}

// Adds the 32 rows in memory, ld bytes apart and padded to 16, to the fp32 numbers in LDS.
__device__ __forceinline__ void add_rows(int lane, char *st, const char *from, uint32_t ld, int64_t rows, int64_t bytes) {
    const int c = lane & 7;
    asm volatile("" ::: "memory");
    float4 v[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int r = t * 8 + (lane >> 3);
        v[t] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows && c * 16 < bytes) v[t] = *reinterpret_cast<const float4 *>(from + ((uint32_t)r * ld + (uint32_t)c * 16));
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        float4 &x = *reinterpret_cast<float4 *>(store_chunk(st, t * 8 + (lane >> 3), c));
        x = make_float4(x.x + v[t].x, x.y + v[t].y, x.z + v[t].z, x.w + v[t].w);
    }
}

// The registers of tile (ii, jj) of 4 x 2 tiles, 64 columns (m) of 32 rows (n), as 16-bit numbers.
__device__ __forceinline__ void put16(int lane, char *st, int ii, int jj, uint32_t lo, uint32_t hi) {
    char *at = store_chunk(st, 16 * jj + (lane & 15), 2 * ii + (lane >> 5));
    *reinterpret_cast<uint2 *>(at + 8 * (lane >> 4 & 1)) = make_uint2(lo, hi);
}
// The same of 2 x 2 tiles as fp32 numbers.
__device__ __forceinline__ void put32(int lane, char *st, int ii, int jj, const float (&x)[4]) {
    char *at = store_chunk(st, 16 * jj + (lane & 15), 4 * ii + (lane >> 4));
    *reinterpret_cast<float4 *>(at) = make_float4(x[0], x[1], x[2], x[3]);
}

// Whether a product takes operands with this row pitch: offsets within a tile of 256 rows stay below 2^31.
inline bool pitch_fits(int64_t ld_bytes) { return ld_bytes > 0 && ld_bytes <= (1 << 23); }

// What becomes of a product: C[n][m] -> 2^e row[n] C[n][m], rounded to dt, y rows ldy elements apart.  e = base + sum of
// sign[i] exps[i]; a row factor of 0 makes zeros of whatever the row holds.  With acc (fp32 [splits][rows][ldp], ldp columns_of
// the columns) the parts of a split contraction go there as they are, added to what is there with `add`; finish() turns them
// into y.
struct Result {
    void *y;
    int64_t ldy;
    int dt;
    const float *row;
    const int *exps;
    int base, sign[2];
    float *acc;
    int64_t ldp;
    int add;
    const float *by;   // y times by[0], where given
    const int *place;  // for finish(): the row of acc (and of `row`) that y's row n is, or -1 for zeros; NULL: row n
};
inline int64_t columns_of(int64_t cols) { return (cols + 3) / 4 * 4; }  // whole 16 bytes

enum : int { BIG = 0, MID = 1, FEW = 2, ONE = 3 };
struct Plan {
    int shape, splits;
};
// The tile and the split of the contraction (at most max_splits) for rows x cols results of `blocks` BK-blocks.  large: not the
// tiles for few rows (an operand across the contraction has wide rows in LDS).
Plan plan(int64_t rows, int64_t cols, int64_t blocks, int max_splits, bool large = false);

// Fills in the tiles of g and the grid of a launch.
template <class S>
inline dim3 tiles_of(Args &g, int splits) {
    g.mt = (int)((g.a.rows + S::BM - 1) / S::BM);
    g.nt = (int)((g.b.rows + S::BN - 1) / S::BN);
    g.splits = splits;
    const int64_t tiles = (int64_t)g.mt * g.nt;
    int64_t most = 256 * S::PER_CU / splits / 8 * 8;  // whole rounds of the XCDs
    if (most < 8) most = 8;
    return dim3((unsigned)(tiles < most ? tiles : most), 1, (unsigned)splits);
}

void multiply(Args g, bool f16, const Plan &p, const Result &r, hipStream_t st);
void finish(const Result &r, int splits, int64_t rows, int64_t cols, hipStream_t st);

__device__ __forceinline__ int exponent_of(const Result &r) {
    int e = r.base;
    if (r.exps) e += r.sign[0] * r.exps[0] + r.sign[1] * r.exps[1];
    return e;
}

}  // namespace mm
}  // namespace gdn
