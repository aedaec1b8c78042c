// Operands of the matrix products (gdn_product.h) in the order and type that these take: 16-bit terms along the contraction.
#pragma once

#include "gdn_host.h"

namespace gdn {
namespace mm {

// A matrix as the caller has it: rows of `cols` elements of type dt, ld elements apart.  With targets, rows whose target is
// `ignore` count as zeros, whatever they hold.  With index and count, row r is the caller's row index[r], and rows from *count
// on count as zeros (rows: how many there may be).
struct Source {
    const void *p;
    int dt;
    int64_t rows, cols, ld;
    const int64_t *targets;
    int64_t ignore;
    const int *index, *count;
};
// Factors on the rows, powers of two, each relative to the largest of them, by[0].
struct Factors {
    const float *row, *by;
};

constexpr int PARTS = 512;  // partial maxima of one matrix

// Elements of a row of `cols`, filled up to whole blocks of the contraction.
inline int64_t padded(int64_t cols) { return (cols + 63) / 64 * 64; }

// part[i][PARTS] = partial maxima of the finite magnitudes of s[i], i < 2, matrices of one type; without rows: zeros.
void maxima(const Source (&s)[2], float *part, hipStream_t st);

// exps[i] = the exponent e_i that takes the largest of part[i][PARTS] to [2^top, 2^(top + 1)), for i < 2, 0 for zeros;
// most[0] = the largest of part[2][PARTS].  exps NULL: only that.
void exponents(const float *part, int top, int *exps, float *most, hipStream_t st);

// exps[r] = the same for the finite magnitudes of row r alone.
void row_exponents(const Source &s, int top, int *exps, hipStream_t st);

// dst[r][t * padded(cols) + c] = term t < slots of 2^e s[r][c], e = exps[which], or exps[r] with which = EACH_ROW (0 without exps),
// zeros behind the last column: x is the sum of its terms up to the last one's rounding.  f16 or bf16 terms; the third of three
// fp16 slots holds the first term times 2^-LOW, the partner of a second term that is stored times 2^LOW.
constexpr int LOW = 11, EACH_ROW = -1;
void terms(const Source &s, int slots, bool f16, const int *exps, int which, void *dst, hipStream_t st);

// The same transposed, times f's factors (where f.row is not NULL): dst[c][t * padded(rows) + r].
void terms_across(const Source &s, int slots, bool f16, const int *exps, int which, const Factors &f, void *dst, hipStream_t st);

}  // namespace mm
}  // namespace gdn
