// Checks on the CPU that what the sequence-cache kernels form addresses from
// (kernel.h_amd/csrc/kernels/kh_paged.h) stays inside the arrays it is for,
// whatever device memory holds. Prints "paged_bounds_check ok", or the first
// failure and exits 1.
#include "kh_paged.h"

#include <cstdio>
#include <cstdlib>
#include <initializer_list>

static void expect(bool ok, const char *what, long a = 0, long b = 0, long c = 0) {
  if (ok) return;
  std::printf("FAIL: %s (%ld, %ld, %ld)\n", what, a, b, c);
  std::exit(1);
}

// Rows of q and lse: those of tokens that exist, and none of a sequence without new tokens, wherever it starts.
static void queries() {
  for (int32_t tokens : {1, 2, 50})
    for (int32_t group : {1, 3, 4, 64}) {
      const KhDiv by = kh_div_by(static_cast<uint32_t>(group));
      for (int32_t a : {INT32_MIN, -1, 0, 1, 3, 49, 50, 51, INT32_MAX})
        for (int32_t b : {INT32_MIN, -1, 0, 1, 3, 7, 49, 50, 51, INT32_MAX}) {
          const KhSeq s = kh_seq(100, a, b, 100, tokens);
          for (int32_t R = 0; R < 64; ++R) {
            const KhQuery q = kh_query(s, group, by, R);
            if (s.m == 0) {
              expect(q.token < 0, "no new tokens, nothing to read", a, b, tokens);
              continue;
            }
            expect(q.token >= s.start && q.token < s.start + s.m && q.token < tokens, "a token of the sequence", a, b, R);
            expect(q.head >= 0 && q.head < group, "a head of the group", a, b, R);
            if (R < s.m * group) expect((q.token - s.start) * group + q.head == R, "the row's own", a, b, R);
          }
        }
    }
}

int main() {
  queries();
  std::printf("paged_bounds_check ok\n");
  return 0;
}
