// How kh_paged_attention8 shares a step out, without a GPU: its host code with
// launches that only write down what they were given.
//   cache8_plan_check                 a grid of steps, checked
//   cache8_plan_check NAME=VALUE ...  one step: what its first launch is told
#include "../../kernel.h_amd/csrc/runtime/khrt_cache8.cpp"

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <vector>

namespace {

struct Launch {
  std::string symbol;
  khrt_dim3 grid;
  KhAttention8Params p;
};
std::vector<Launch> launches;
std::string last_error;

}  // namespace

int khrt::fail(int code, const std::string &msg) {
  last_error = msg;
  return code;
}

int khrt::launch_embedded(const char *, const char *symbol, khrt_dim3 grid, khrt_dim3, void *, void **params, size_t) {
  launches.push_back({symbol, grid, *static_cast<const KhAttention8Params *>(params[0])});
  return 0;
}

namespace {

char *const kAt = reinterpret_cast<char *>(uintptr_t(1) << 40);  // where the workspace is said to be

struct Step {
  int64_t tokens = 64, seqs = 64, hq = 32, hk = 8, d = 128, page_size = 16, width = 1024, max_len = 0, max_new = 1, shared = 0, window = 0;
  int64_t dtype = KHRT_BF16, workspace = -1;  // -1: what is reported
  double scale = 0.125, cap = 0.0;
};

kh_paged_attention8_args args_of(const Step &s) {
  kh_paged_attention8_args a{};
  const auto at = [](int n) { return reinterpret_cast<void *>(uintptr_t(n) << 30); };
  kh_paged_cache8 &c = a.cache;
  c.k = at(1), c.v = at(2), c.k_scale = static_cast<uint8_t *>(at(3)), c.v_scale = static_cast<uint8_t *>(at(4));
  c.k_page_stride = c.v_page_stride = s.page_size * s.hk * s.d, c.k_slot_stride = c.v_slot_stride = s.hk * s.d;
  c.k_head_stride = c.v_head_stride = s.d, c.scale_page_stride = s.hk * s.page_size, c.scale_head_stride = s.page_size;
  c.pages = 1000000, c.page_size = s.page_size, c.kv_heads = s.hk, c.head_dim = s.d;
  a.table.pages = static_cast<const int32_t *>(at(5)), a.table.lens = static_cast<const int32_t *>(at(6));
  a.table.row_stride = a.table.width = s.width, a.table.seqs = s.seqs, a.table.max_len = s.max_len;
  a.q = at(7), a.out = at(8), a.lse = static_cast<float *>(at(9)), a.q_starts = static_cast<const int32_t *>(at(10));
  a.q_stride = a.out_stride = s.hq * s.d, a.tokens = s.tokens, a.q_heads = s.hq, a.window = s.window;
  a.max_new = s.max_new, a.shared = s.shared;
  a.scale = static_cast<float>(s.scale), a.cap = static_cast<float>(s.cap), a.dtype = static_cast<int32_t>(s.dtype);
  return a;
}

size_t reported(const Step &s) {
  const kh_paged_attention8_args a = args_of(s);
  size_t bytes = 0;
  if (kh_paged_attention8_workspace(&a, &bytes) != 0) std::printf("FAIL: %s\n", last_error.c_str()), std::exit(1);
  return bytes;
}

// The step's first launch.
Launch run(const Step &s) {
  const kh_paged_attention8_args a = args_of(s);
  const size_t bytes = s.workspace < 0 ? reported(s) : static_cast<size_t>(s.workspace);
  launches.clear();
  if (kh_paged_attention8(&a, bytes > 0 ? kAt : nullptr, bytes, nullptr) != 0) std::printf("FAIL: %s\n", last_error.c_str()), std::exit(1);
  return launches[0];
}

void expect(bool ok, const Step &s, const char *what) {
  if (ok) return;
  std::printf("FAIL: %s: tokens=%lld seqs=%lld hq=%lld hk=%lld d=%lld page_size=%lld width=%lld max_len=%lld max_new=%lld shared=%lld workspace=%lld\n",
              what, (long long)s.tokens, (long long)s.seqs, (long long)s.hq, (long long)s.hk, (long long)s.d, (long long)s.page_size,
              (long long)s.width, (long long)s.max_len, (long long)s.max_new, (long long)s.shared, (long long)s.workspace);
  std::exit(1);
}

// Every entry is somebody's: the parts of the shared ones reach as far as the
// sequences' own begin, whatever the lengths turn out to be; and every array that
// the kernels write lies in the workspace, apart from the others.
void check(const Step &s) {
  const Launch l = run(s);
  const KhAttention8Params &p = l.p;
  const int64_t capacity = std::min(s.width * s.page_size, kCapacity), rows = s.tokens * s.hq;
  expect(p.shared >= 0 && p.shared <= std::min(s.shared, capacity), s, "no more shared than the caller said");
  expect(p.shared > 0 ? p.shared_blocks > 0 : p.shared_blocks == 0, s, "shared entries have workgroups");
  if (p.shared > 0) {
    expect(int64_t(p.shared_splits) * p.shared_each >= p.shared, s, "the parts reach the sequences' own entries");
    expect(int64_t(p.shared_splits - 1) * p.shared_each < p.shared, s, "no part is empty");
    expect(p.shared_blocks == p.shared_splits * s.hk * ceil_div(s.tokens * (s.hq / s.hk), KH_WIDE_ROWS), s, "every row has its parts");
  }
  struct Span {
    const void *at;
    int64_t bytes;
  };
  const int64_t narrow = p.whole || p.groups == 0 ? 0 : int64_t(p.groups) * 2 * KH_TILE_ROWS * p.together;
  const int64_t wide = p.wide_blocks > 0 && p.wide_splits > 1 ? p.wide_splits * rows : 0;
  const int64_t common = p.shared > 0 ? (p.shared_splits + 1) * rows : 0;
  const Span spans[] = {{p.part_o, narrow * s.d * 4}, {p.wide_o, wide * s.d * 4}, {p.shared_o, common * s.d * 4}, {p.part_ml, narrow * 8},
                        {p.wide_ml, wide * 8}, {p.shared_ml, common * 8}, {p.joins, narrow > 0 ? int64_t(p.groups) * int64_t(sizeof(KhJoin)) : 0}};
  const int64_t bytes = s.workspace < 0 ? int64_t(reported(s)) : s.workspace;
  int64_t end = 0;
  for (const Span &x : spans) {
    if (x.bytes == 0) continue;
    const int64_t at = static_cast<const char *>(x.at) - kAt;
    expect(at >= end, s, "arrays lie apart");
    end = at + x.bytes;
    expect(end <= bytes, s, "arrays lie in the workspace");
  }
}

}  // namespace

int main(int argc, char **argv) {
  if (argc > 1) {
    Step s;
    const std::map<std::string, int64_t *> fields = {
        {"tokens", &s.tokens}, {"seqs", &s.seqs}, {"hq", &s.hq}, {"hk", &s.hk}, {"d", &s.d}, {"page_size", &s.page_size}, {"width", &s.width},
        {"max_len", &s.max_len}, {"max_new", &s.max_new}, {"shared", &s.shared}, {"window", &s.window}, {"dtype", &s.dtype},
        {"workspace", &s.workspace}};
    for (int i = 1; i < argc; ++i) {
      const char *eq = std::strchr(argv[i], '=');
      if (eq == nullptr) return std::printf("FAIL: %s\n", argv[i]), 1;
      const std::string name(argv[i], static_cast<size_t>(eq - argv[i]));
      if (name == "scale") s.scale = std::atof(eq + 1);
      else if (name == "cap") s.cap = std::atof(eq + 1);
      else *fields.at(name) = std::atoll(eq + 1);
    }
    check(s);
    const KhAttention8Params p = run(s).p;
    std::printf("{\"shared\": %d, \"shared_blocks\": %d, \"shared_splits\": %d, \"shared_each\": %d, \"groups\": %d, \"wide_blocks\": %d, "
                "\"whole\": %d, \"launches\": %zu, \"cap_in\": %.9g, \"cap_out\": %.9g, \"bytes\": %zu}\n",
                p.shared, p.shared_blocks, p.shared_splits, p.shared_each, p.groups, p.wide_blocks, p.whole, launches.size(),
                static_cast<double>(p.cap_in), static_cast<double>(p.cap_out), reported(s));
    return 0;
  }
  int64_t steps = 0, sharing = 0;
  for (int64_t tokens : {2, 64, 100, 700, 8192})
    for (int64_t seqs : {1, 2, 60, 64, 120})
      for (const auto &[hq, hk, d] : std::vector<std::array<int64_t, 3>>{{32, 8, 128}, {4, 4, 64}, {8, 2, 256}, {7, 1, 80}})
        for (int64_t page_size : {16, 24})
          for (int64_t shared : {0, 1, 300, 1500, 8192, 20000, 1 << 30})
            for (int64_t max_len : {0, 1, 300, 1499, 4096, 8192, 30000})
              for (int64_t max_new : {0, 1, 400})
                for (int64_t workspace : {-1, 0, 100000, 5000000}) {
                  Step s;
                  s.tokens = tokens, s.seqs = seqs, s.hq = hq, s.hk = hk, s.d = d, s.page_size = page_size, s.shared = shared;
                  s.max_len = max_len, s.max_new = max_new, s.workspace = workspace;
                  check(s);
                  ++steps;
                  sharing += launches[0].p.shared > 0;
                }
  std::printf("%lld steps, %lld of them with shared entries apart\ncache8_plan_check ok\n", (long long)steps, (long long)sharing);
  return sharing > 1000 ? 0 : 1;
}
