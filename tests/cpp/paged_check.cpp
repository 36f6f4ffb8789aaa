// Checks the index arithmetic that the sequence-cache kernels and their
// launcher share (kernel.h_amd/csrc/kernels/kh_paged.h) on the CPU: division by
// multiplication, page walks with absent and out-of-range pages, clamped
// lengths and starts, what each token sees, and how entries are split.
// Prints "paged_check ok", or the first failure and exits 1.
#include "kh_paged.h"

#include <cstdio>
#include <cstdlib>
#include <vector>

static void expect(bool ok, const char *what, long a = 0, long b = 0, long c = 0) {
  if (ok) return;
  std::printf("FAIL: %s (%ld, %ld, %ld)\n", what, a, b, c);
  std::exit(1);
}

int main() {
  const uint32_t top = 0x7fffffffu;
  std::vector<uint32_t> bys;
  for (uint32_t by = 1; by <= 4200; ++by) bys.push_back(by);
  for (uint32_t by : {65535u, 65536u, 65537u, 1u << 20, (1u << 20) - 1, (1u << 30) - 1, 1u << 30, (1u << 30) + 1, top}) bys.push_back(by);
  for (uint32_t by : bys) {
    const KhDiv d = kh_div_by(by);
    for (uint32_t j = 0; j < 300; ++j) expect(kh_div(j, d) == j / by, "division", j, by);
    for (uint64_t q = 1; q * by <= top; q = q * 3 + 1) {
      for (int64_t e = -1; e <= 1; ++e) {
        const uint32_t j = static_cast<uint32_t>(q * by + e);
        if (j <= top) expect(kh_div(j, d) == j / by, "division near a multiple", j, by);
      }
    }
    for (uint32_t j = top; j > top - 300; --j) expect(kh_div(j, d) == j / by, "division", j, by);
    uint32_t x = by * 2654435761u;
    for (int i = 0; i < 200; ++i) {
      x = x * 1664525u + 1013904223u;
      expect(kh_div(x >> 1, d) == (x >> 1) / by, "division", x >> 1, by);
    }
  }

  // A row of five pages, of which some do not exist.
  const int32_t row[5] = {3, -1, 7, 8, INT32_MIN};
  for (uint32_t ps : {1u, 3u, 16u, 24u}) {
    const KhDiv by = kh_div_by(ps);
    for (uint32_t j = 0; j < 8 * ps; ++j) {
      const KhSlot s = kh_slot(row, 5, 8, by, j);
      const uint32_t i = j / ps;
      const bool there = i == 0 || i == 2;
      expect((s.page >= 0) == there, "an entry is there where its page is", j, ps, s.page);
      if (there) expect(s.page == row[i] && s.slot == static_cast<int32_t>(j % ps), "page and slot", j, ps);
    }
    expect(kh_slot(row, 5, 8, by, top).page < 0, "far past the row");
  }

  // Lengths and starts from device memory, whatever they hold.
  for (int64_t len : {INT32_MIN, -1, 0, 1, 99, 100, 101, INT32_MAX})
    for (int64_t a : {INT32_MIN, -1, 0, 3, 50, 51, INT32_MAX})
      for (int64_t b : {INT32_MIN, -1, 0, 3, 49, 50, INT32_MAX}) {
        const KhSeq s = kh_seq(static_cast<int32_t>(len), static_cast<int32_t>(a), static_cast<int32_t>(b), 100, 50);
        expect(s.n >= 0 && s.n <= 100 && s.start >= 0 && s.m >= 0 && s.start + s.m <= 50, "in range", len, a, b);
      }

  // What token i sees, entry by entry.
  for (int n = 0; n <= 40; ++n)
    for (int m = 0; m <= 45; ++m)
      for (int w : {0, 1, 2, 7, 40, 1000, INT32_MAX}) {
        const KhSeq s{n, m, 0};
        for (int i = 0; i < m; ++i) {
          const KhSpan r = kh_seen(s, i, w);
          const int at = n - m + i;
          expect(r.end <= n && r.first >= 0, "a span inside the sequence", n, m, i);
          for (int j = 0; j < n; ++j) {
            const bool sees = j <= at && (w == 0 || j > static_cast<long>(at) - w);
            expect((j >= r.first && j < r.end) == sees, "what a token sees", n, m, i);
          }
        }
        // The splits cover all that any token sees once, in order.
        for (int splits : {1, 2, 5})
          for (int keys : {1, 4, 16}) {
            int used = 0, next = -1;
            for (int k = 0; k < splits; ++k) {
              const KhSplit p = kh_split(s, w, splits, keys, k);
              if (k == 0) used = p.used, next = m > 0 ? (kh_seen(s, 0, w).first < n ? kh_seen(s, 0, w).first : n) : p.first;
              expect(p.used == used && used >= 1 && used <= splits, "how many splits are used", n, m, k);
              if (k >= used) {
                expect(p.first == p.end, "an unused split is empty", n, m, k);
              } else {
                expect(p.first == next || (n == 0 && p.first == p.end), "splits follow each other", n, m, k);
                expect(p.first <= p.end || p.first >= n, "a split is not turned round", n, m, k);
                next = p.end;
              }
            }
            expect(next == n || next >= n, "the splits reach the end", n, m, next);
          }
      }
  // Near the top of the range nothing overflows (this file is built with -fsanitize=undefined).
  const int32_t big = INT32_MAX - 65536;
  const KhSeq s{big, 5, 0};
  for (int w : {0, 1, big, INT32_MAX})
    for (int k : {0, 1, 100, 127}) {
      const KhSplit p = kh_split(s, w, 128, (big / 128 + 128) / 128 * 128, k);
      expect(p.first >= 0 && p.first <= p.end && p.end <= big, "a long sequence's split", w, k, p.first);
      expect(kh_seen(s, 4, w).end == big, "the last token's own entry");
    }
  std::printf("paged_check ok\n");
  return 0;
}
