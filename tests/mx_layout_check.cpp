// Every block of an operand has sixteen bytes of codes and a scale byte of its own, inside the operand, where the MMA looks for
// them (swizzled atoms of eight rows), and runs of rows that start at a multiple of 128 are contiguous stage by stage.
#include <cstdio>
#include <vector>

#include "../tensorfold_b200/csrc/mx_layout.h"

using namespace tf;

static int check(int rows, int k) {
  const int steps = mx_steps(k), blocks = 2 * steps;
  std::vector<char> used(static_cast<size_t>(mx_operand_bytes(rows, steps)), 0);
  int bad = 0;
  for (int r = 0; r < rows; ++r)
    for (int b = 0; b < blocks; ++b) {
      const int64_t c = mx_code_offset(rows, steps, r, b), s = mx_scale_offset(rows, steps, r, b);
      if (c < 0 || c % 16 || c + 16 > static_cast<int64_t>(used.size()) || s < 0 || s >= static_cast<int64_t>(used.size())) {
        ++bad;
        continue;
      }
      for (int i = 0; i < 16; ++i) bad += used[c + i]++ != 0;
      bad += used[s]++ != 0;
      // the stage, the row's atom and line inside it, and the exclusive-or of the swizzle on address bits
      const int u = b / 8;
      const int64_t base = u * mx_stage_bytes(rows);
      if (u < steps / 4) {
        const int64_t plain = base + (r / 8) * 1024 + (r % 8) * 128 + (b % 8) * 16;
        bad += (plain - base) != ((c - base) ^ (((c - base) >> 3) & 0x70));
        bad += s != base + rows * 128 + (r / 128) * 1024 + (b % 8) / 4 * 512 + (r % 32) * 16 + (r % 128) / 32 * 4 + b % 4;
      } else {
        const int64_t from = base + (b % 8) / 2 * rows * 32, plain = from + (r / 8) * 256 + (r % 8) * 32 + (b % 2) * 16;
        bad += (plain - from) != ((c - from) ^ (((c - from) >> 3) & 0x10));
      }
    }
  return bad;
}

int main() {
  int bad = 0;
  const int ks[] = {32, 64, 96, 128, 160, 224, 256, 288, 512, 736, 1856, 2688};
  const int rows[] = {8, 16, 24, 64, 120, 128, 256, 384};
  for (int k : ks)
    for (int r : rows) {
      const int here = check(r, k);
      if (here) std::printf("rows %d k %d: %d\n", r, k, here);
      bad += here;
    }
  if (mx_stage_bytes(128) != MX_UNIT || mx_operand_bytes(128, 4) != MX_UNIT || mx_operand_bytes(128, 1) != 4096 + 512) ++bad;
  for (int r = 0; r < 64; ++r) bad += mx_pair_row(r) != (r / 32) * 16 + r % 16 || mx_pair_second(r) != (r % 32 >= 16);
  std::printf("%s\n", bad ? "FAIL" : "OK");
  return bad ? 1 : 0;
}
