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
        // The units' blocks cover all that any token sees.
        for (int whole : {0, 1}) {
          const KhUnits u = kh_units(s, 3, w, whole);
          expect(u.tiles == (m * 3 + 15) / 16 && u.blocks >= 1 && (whole == 0 || u.blocks == 1), "units", n, m, w);
          int first = n;
          for (int i = 0; i < m; ++i) first = kh_seen(s, i, w).first < first ? kh_seen(s, i, w).first : first;
          if (m > 0) expect(u.first <= first && (whole != 0 || u.first + u.blocks * KH_STRETCH >= n), "they cover", n, m, w);
        }
      }
  // Near the top of the range nothing overflows (this file is built with -fsanitize=undefined).
  const int32_t big = INT32_MAX - 65536;
  const KhSeq s{big, 5, 0};
  for (int w : {0, 1, big, INT32_MAX}) {
    const KhUnits u = kh_units(s, 7, w, 0);
    expect(u.first >= 0 && u.first + int64_t(u.blocks) * KH_STRETCH >= big, "a long sequence's blocks", w, u.first);
    expect(kh_seen(s, 4, w).end == big, "the last token's own entry");
  }

  // Parts of the wide form's units: whole tiles, in order, all of them.
  for (int first : {0, 1, 100})
    for (int keys : {0, 1, 63, 64, 255, 256, 257, 511, 512, 513, 5000, 100000})
      for (int splits : {1, 2, 3, 64}) {
        int next = first, used = 0;
        for (int k = 0; k < splits; ++k) {
          const KhPart p = kh_part(first, first + keys, splits, k);
          if (k == 0) used = p.used;
          expect(p.used == used && used >= 1 && used <= splits, "parts", keys, splits, k);
          if (k >= used) {
            expect(p.first >= p.end, "an unused part is empty", keys, splits, k);
            continue;
          }
          expect(p.first == next && (p.end > p.first || keys == 0), "parts follow each other", keys, splits, k);
          expect((p.first - first) % 64 == 0 && (k == used - 1 || p.end - p.first >= 256), "whole tiles", keys, splits, k);
          next = p.end;
        }
        expect(next == first + keys, "parts reach the end", keys, splits, next);
      }
  expect(kh_part(0, big, 1, 0).end == big && kh_part(5, 3, 7, 0).used == 1, "parts at the limits");

  // Shares follow each other, differ by a block at most, and know their owner.
  for (int work : {0, 1, 2, 7, 511, 512, 513, 100000, (1 << 30) - 1})
    for (int most : {1, 2, 3, 64, 511, 512, 4095}) {
      const KhShares s = kh_shares(work, most);
      expect(s.groups <= most && s.groups <= work && (work == 0 || s.groups >= 1), "workgroups with a share", work, most);
      expect(kh_share(s, 0) == 0 && kh_share(s, s.groups) == work, "shares cover all", work, most);
      for (int g = 0; g < s.groups; ++g) {
        const int a = kh_share(s, g), b = kh_share(s, g + 1);
        expect(b > a && b - a <= work / s.groups + 1, "a share", work, most, g);
        expect(kh_owner(s, a) == g && kh_owner(s, b - 1) == g && kh_owner(s, a + (b - a) / 2) == g, "its owner", work, most, g);
      }
    }
  std::printf("paged_check ok\n");
  return 0;
}
