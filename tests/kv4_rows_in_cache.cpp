// Whether the 4-bit cache's writers take the rows of a position for the cache's
// (rows_in_cache of csrc/dip_kv4.h), on the CPU, for tests/test_kv4_host.py: the
// answer must be that of whole numbers without an end, at the ends of int64 too.
// Prints the number of wrong answers.
#include <cstdio>
#include <cstdint>

#include "dip_kv4.h"

int main() {
  const int64_t firsts[] = {INT64_MIN, INT64_MIN + 1, -(1ll << 40), -1, 0, 1, 30, 31, 32, 33,
                            (1ll << 31) - 1, 1ll << 31, 1ll << 32, 1ll << 40, INT64_MAX - 32,
                            INT64_MAX - 1, INT64_MAX};
  const int lens[] = {32, 64, 1 << 30};
  int bad = 0;
  for (int64_t first : firsts)
    for (int len : lens)
      for (int tokens : {0, 1, 2, 31, 32}) {
        const bool want = first >= 0 && (__int128)first + tokens <= len;
        if (dip::rows_in_cache(first, tokens, len) != want) {
          std::printf("first %lld tokens %d max_len %d\n", (long long)first, tokens, len);
          ++bad;
        }
      }
  std::printf("bad %d\n", bad);
  return bad != 0;
}
