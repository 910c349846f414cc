// The 1 x 128 quantiser's index arithmetic (csrc/block_kernels.h row_block),
// for every block a launch forms: the matrix's own and those past its end.
#include "block_kernels.h"

#include <climits>
#include <cstdio>

namespace {
int failures = 0;

void check(long rows, long cols, int blocks_a_cta) {
  const long kb = ngb::scale_blocks(cols), blocks = rows * kb;
  const long formed = (blocks + blocks_a_cta - 1) / blocks_a_cta * blocks_a_cta;
  const auto one = [&](long b) {
    const ngb::RowBlock at = ngb::row_block(b, blocks, int(kb), cols);
    bool ok;
    if (b < blocks) {
      const long row = b / kb, block = b % kb;
      ok = at.row == row && at.block == block && at.cols == cols && at.whole == ((block + 1) * 128 <= cols);
    } else { // nothing of it may be read: no column, and not taken for a whole block
      ok = at.row == 0 && at.block == 0 && at.cols == 0 && !at.whole;
    }
    if (!ok && ++failures < 10)
      std::printf("%ld x %ld, block %ld of %ld: row %d block %d cols %d whole %d\n", rows, cols, b, blocks, at.row,
                  at.block, at.cols, at.whole);
  };
  for (long b = 0; b < 300 && b < formed; ++b) one(b);
  for (long b = blocks > 300 ? blocks - 300 : 0; b < formed; ++b) one(b);
  for (long b = 0; b < blocks; b += blocks / 1000 + 1) one(b);
}
} // namespace

int main() {
  for (int blocks_a_cta : {32, 64}) {
    check(1, 1, blocks_a_cta);
    check(37, 389, blocks_a_cta);
    check(8192, 8192, blocks_a_cta);
    check(16777217, 16, blocks_a_cta);            // 2^24 + 1 blocks
    check(335545, 6400, blocks_a_cta);            // 2^24 + 34
    check(3, (1L << 30) - 1, blocks_a_cta);       // the longest rows
    check(1, INT_MAX / 2, blocks_a_cta);
    for (long n : {1L << 25, 1L << 26, (1L << 29) + 3, (1L << 30) + 7, 0x7FFFFFFFL}) check(n, 128, blocks_a_cta);
    check(0x7FFFFFFFL / 2, 129, blocks_a_cta);
  }
  std::printf(failures ? "FAILED %d\n" : "ok\n", failures);
  return failures != 0;
}
