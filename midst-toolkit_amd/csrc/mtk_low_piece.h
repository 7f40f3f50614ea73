// mtk_low_piece.h — where a lane of the adapter kernels takes its piece of a low-rank factor from.  Plain C++: the bounds are tested on the host.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define MTK_HD __host__ __device__
#else
#define MTK_HD
#endif

// B_e is N rows of `ld` values, whole 16-byte pieces, of which `values` are the rank's.  The offset of the piece that starts at value j of
// feature n's row (the last one's for n behind it); for a lane behind the rank, whose piece is cleared after the load, the first of the model:
// the one place that every B_e has.
MTK_HD constexpr int64_t mtk_low_piece(int n, int N, int ld, int values, int j) { return j < values ? (int64_t)(n < N ? n : N - 1) * ld + j : 0; }
