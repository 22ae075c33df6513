// Operands of a call that may lie in one buffer: columns of the rows of a product, for instance.  (No device code.)
#pragma once
#include <stdint.h>

namespace cacti {

// Whether `rows` rows of wa halves, lda from one to the next, and as many of wb and ldb share memory.  (Of different pitches: where what lies
// between their ends does.)
inline bool rows_share(int64_t rows, const void *a, int64_t lda, int64_t wa, const void *b, int64_t ldb, int64_t wb)
{
    const int64_t d = ((int64_t)reinterpret_cast<intptr_t>(b) - (int64_t)reinterpret_cast<intptr_t>(a)) / 2;
    if (d >= (rows - 1) * lda + wa || -d >= (rows - 1) * ldb + wb) return false;
    if (rows == 1 || lda != ldb) return true;
    const int64_t r = (d % lda + lda) % lda;       // where a row of b begins, from a row of a on
    return r < wa || r + wb > lda;
}

}  // namespace cacti
