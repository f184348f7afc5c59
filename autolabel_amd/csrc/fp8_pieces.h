// Where the weight gradient of 8-bit blocks (k_fp8_tn, fp8.hip) reads a 16-bit tensor of M rows of C columns, ld >= C elements apart: steps of 128 rows,
// strips of 32 columns from `col` (a multiple of 32, col < C), pieces of eight consecutive values from column col + c8 of a row of the step.  Plain
// arithmetic, for the device and for tests on the host.
#pragma once
#include <stdint.h>
#ifdef __HIPCC__
#define ALN_HD __host__ __device__
#else
#define ALN_HD
#endif

// Whether some step needs more than tn_whole's loads
ALN_HD static inline bool tn_has_tail(int64_t M, int N, int K) { return M % 128 || N % 32 || K % 32; }

// Columns stand alone, so what a lane reads behind the last one does not matter as long as it is memory of the tensor: pieces that begin behind it read
// the last piece instead, and the last piece's seven values too many lie in the rows behind (ld >= C).
ALN_HD static inline int tn_column(int C, int col, int c8) { const int last = (C - 1 - col) & ~7; return c8 < last ? c8 : last; }
// True where every piece of the step is memory of the tensor: row r's begins at element r * ld + tn_column of the step's first row and column `col`
ALN_HD static inline bool tn_whole(int64_t M, int64_t ld, int C, int64_t step, int col) {
  const int64_t left = M - (step + 1) * 128;              // rows behind this step
  return left >= 0 && (col + 32 <= C || left * ld >= 7);
}
// The tensor's end: rows behind the last one read that one (and count as zeros), and a piece that would reach over the end begins earlier, by `over`, and
// is shifted down.  The tensor has eight values or more.
struct TnEnd { int last, end; };                          // the step's last row; where the last piece may begin (it may lie before the base)
ALN_HD static inline TnEnd tn_end(int64_t M, int64_t ld, int C, int64_t step, int col) {
  const int64_t rows = M - 1 - step * 128, size = rows * ld + C - col;
  return {(int)(rows < 127 ? rows : 127), (int)(size < 0x7fffffff ? size : 0x7fffffff) - 8};
}
struct TnPiece { int at, over; };                         // its first value, counted from the step's first row and column `col`; values to shift out
ALN_HD static inline TnPiece tn_piece(const TnEnd& e, int ld, int row, int c) {
  const int at = (row < e.last ? row : e.last) * ld + c, over = at > e.end ? at - e.end : 0;
  return {at - over, over};
}
