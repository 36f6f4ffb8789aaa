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

// Sequences that claim the same tokens: counts of blocks past 32 bits, as the
// kernels add them up. The place in a sequence stays in it, and the owners of a
// unit's parts are workgroups that there are.
static void walks() {
  uint32_t seed = 1;
  auto random = [&seed](uint32_t below) {
    seed = seed * 1664525u + 1013904223u;
    return static_cast<int32_t>((static_cast<uint64_t>(seed) * below) >> 32);
  };
  int past = 0;
  for (int run = 0; run < 3000; ++run) {
    const int32_t blocks = 1 + random(1 << 20), seqs = 2 + random(30);
    int32_t work[32];
    uint32_t all = 0;
    int64_t real = 0;
    for (int i = 0; i < seqs; ++i) {
      work[i] = random((1 << 30) / blocks) * blocks;
      all += static_cast<uint32_t>(work[i]);
      real += work[i];
    }
    past += real > INT32_MAX;
    const int32_t line = static_cast<int32_t>(all);
    const KhShares s = kh_shares(line, 512);
    for (int32_t g = 0; g < s.groups; g += 1 + random(64)) {
      const int32_t start = kh_share(s, g), end = kh_share(s, g + 1);
      // The first sequence whose wrapped count passes the start.
      uint32_t upto = 0;
      int seq = -1;
      int32_t in = 0;
      for (int i = 0; i < seqs && seq < 0; ++i) {
        const uint32_t before = upto;
        upto += static_cast<uint32_t>(work[i]);
        if (static_cast<int32_t>(upto) > start) {
          seq = i;
          in = start - static_cast<int32_t>(before);
          const int32_t unit = in / blocks, begin = static_cast<int32_t>(before) + unit * blocks;
          const KhOwners o = kh_owners(s, line, begin, blocks);
          expect(o.first >= 0 && o.count >= 1 && o.first + o.count <= s.groups, "owners", run, g, o.first);
          expect(o.first <= g && g < o.first + o.count, "the workgroup is one of them", run, g, o.first);
        }
      }
      for (int32_t at = start; at < end && seq >= 0 && seq < seqs;) {
        while (seq < seqs && kh_passed(in, work[seq])) ++seq;
        if (seq == seqs) break;
        expect(in >= 0 && in < work[seq], "a place in the sequence", run, g, in);
        const int32_t left = blocks - in % blocks, step = end - at < left ? end - at : left;
        at += step, in += step;
      }
    }
  }
  expect(past > 1000, "counts past 32 bits");
}

// A chunk's older entries, in a sequence of up to the longest there may be.
static void older() {
  const int32_t top = INT32_MAX - 65536;
  for (int32_t n : {0, 1, 40, 1000, (1 << 30) + 100, top})
    for (int32_t m : {0, 1, 7, 50, 2000})
      for (int64_t first : {int64_t(0), int64_t(1024), int64_t(n) - m - 3, int64_t(n) - m, int64_t(n) - 5}) {
        if (first < 0 || first >= n) continue;
        const int64_t end = first + 1024 < n ? first + 1024 : n;
        int64_t want = 0;
        for (int64_t j = first; j < end; ++j) want += j < int64_t(n) - m;
        expect(kh_older(KhSeq{n, m, 0}, static_cast<int32_t>(first), static_cast<int32_t>(end)) == want, "older entries", n, m, first);
      }
}

// Which steps the narrow form has alone: single tokens and few each, not a batch
// that may have a long chunk among them.
static void forms() {
  expect(kh_narrow_only(64, 64, 4, 0, 32, 256), "single tokens");
  expect(kh_narrow_only(1, 1, 32, 0, 32, 256) && !kh_narrow_only(9, 1, 4, 0, 32, 256), "one sequence by its rows");
  expect(kh_narrow_only(64, 8, 4, 0, 32, 256), "a few tokens each");
  expect(!kh_narrow_only(127 + 128, 128, 4, 0, 32, 256) && !kh_narrow_only(127 + 896, 128, 4, 0, 32, 256), "a chunk among single tokens");
  expect(kh_narrow_only(127 + 33, 128, 4, 0, 32, 256), "a short one");
  expect(!kh_narrow_only(320, 64, 4, 0, 32, 256) && kh_narrow_only(320, 64, 4, 5, 32, 256), "five tokens each, said and not");
  expect(!kh_narrow_only(320, 64, 4, 100, 32, 256) && !kh_narrow_only(320, 64, 4, INT64_MAX, 32, 256), "more than that said");
  expect(!kh_narrow_only(1000, 10, 4, 1, 32, 256), "said too few: the average tells");
  expect(kh_narrow_only(3, 100, 4, 0, 32, 256), "fewer tokens than sequences");
}

int main() {
  forms();
  older();
  queries();
  walks();
  std::printf("paged_bounds_check ok\n");
  return 0;
}
