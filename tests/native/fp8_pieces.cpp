// Every address that k_fp8_tn (autolabel_amd/csrc/fp8.hip) reads, from the arithmetic that it uses (fp8_pieces.h), over small tensors and the ends of large
// ones: inside the tensor, and, where it counts, the value that belongs there.
#include <stdio.h>
#include <stdlib.h>
#include <initializer_list>
#include "../../autolabel_amd/csrc/fp8_pieces.h"

static long long checked = 0;

// one strip of one step; ld, C: pitch and columns; tail: the kernel's variant
static void strip(int64_t M, int64_t ld, int C, int64_t step, int col, bool tail) {
  const int64_t size = (M - 1) * ld + C, base = step * 128 * ld + col;     // the tensor's elements; the step's first
  auto fail = [&](const char* what, int row, int c8, int64_t at) {
    printf("%s: M %lld ld %lld C %d step %lld col %d row %d piece %d reads element %lld of %lld\n", what, (long long)M, (long long)ld, C, (long long)step, col, row, c8, (long long)at,
           (long long)size);
    exit(1);
  };
  for (int c8 = 0; c8 < 32; c8 += 8)
    for (int row = 0; row < 128; ++row) {
      const int c = tn_column(C, col, c8);
      int64_t at;
      int over = 0, last = 127;
      if (!tail || tn_whole(M, ld, C, step, col)) {
        const uint32_t off = 2 * ((uint32_t)(row & 15) * (uint32_t)ld + (uint32_t)c);
        at = base + (int64_t)(row & ~15) * ld + off / 2;
      } else {
        const TnEnd e = tn_end(M, ld, C, step, col);
        const TnPiece q = tn_piece(e, (int)ld, row, c);
        at = base + q.at, over = q.over, last = e.last;
      }
      if (at < 0 || at + 8 > size || over < 0 || over > 7) fail("out of the tensor", row, c8, at);
      // value k of the piece counts where its column exists: (rows behind the last are made zero)
      const int64_t real = step * 128 + row;
      if ((real < M) != (row <= last)) fail("a row too many or too few", row, c8, at);
      for (int k = 0; k < 8 && real < M; ++k) {
        const int column = col + c8 + k;
        if (column >= C) continue;
        if (k + over >= 8 || at + over + k != real * ld + column) fail("another value", row, c8, at + over + k);
      }
      ++checked;
    }
}

static void tensor(int64_t M, int64_t ld, int C, bool tail, int64_t first_step) {
  if (M * C < 8) return;                                   // (the entry point takes another way)
  for (int64_t step = first_step; step < (M + 127) / 128; ++step)
    for (int col = 0; col < C; col += 32) strip(M, ld, C, step, col, tail);
}

int main() {
  const int64_t rows[] = {1, 2, 3, 7, 8, 15, 16, 127, 128, 129, 130, 134, 135, 255, 256, 257, 260, 384};
  for (int64_t M : rows)
    for (int C = 1; C <= 70; ++C)
      for (int64_t ld : {(int64_t)C, (int64_t)C + 1, (int64_t)C + 2, (int64_t)C + 7, (int64_t)C + 8, (int64_t)3 * C + 5}) {
        // the other operand decides with this one whether the kernel knows the tensors' end
        tensor(M, ld, C, true, 0);
        if (!tn_has_tail(M, C, 32)) tensor(M, ld, C, false, 0);
      }
  // the largest pitches, 32-bit offsets at their ends, and the last steps of many rows
  for (int64_t ld : {(int64_t)(1 << 24) - 1, (int64_t)(1 << 24) - 8, (int64_t)5000001})
    for (int C : {1, 31, 40, 4097})
      for (int64_t M : {(int64_t)128, (int64_t)129, (int64_t)200, (int64_t)256, ((int64_t)1 << 31) - 257, ((int64_t)1 << 31) - 256})
        tensor(M, ld, C, true, M / 128 > 2 ? M / 128 - 2 : 0);
  for (int64_t M : {((int64_t)1 << 31) - 256, ((int64_t)1 << 30) + 5})
    for (int C : {1, 3, 33})
      for (int64_t ld : {(int64_t)C, (int64_t)C + 3}) tensor(M, ld, C, true, M / 128 - 2);
  // pieces of 32 bits: a step's offset in bytes stays under 2^32 for the largest pitch (16 rows of it)
  if (2 * (15 * (((uint64_t)1 << 24) - 1) + 24) >= (uint64_t)1 << 32) { printf("offsets run over\n"); return 1; }
  printf("%lld pieces inside their tensors\n", checked);
  return 0;
}
