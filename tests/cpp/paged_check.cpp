// Host-side check of the functions through which the paged-cache kernels reach
// memory (minicpm5.cpp_amd/csrc/mcpm_paged.h), with no GPU: whatever lens,
// starts and pages hold, every position below seq_len has an entry in the page
// table, every page that page_of gives is in the pool, every row of seq_rows is in the
// buffers, and the offsets of distinct (page, position, head) are distinct and
// inside the pool, also where they pass 32 bits.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

#include "mcpm_paged.h"

using namespace mcpm;

static int failures = 0;
#define CHECK(cond, ...)                     \
  do {                                       \
    if (!(cond)) {                           \
      ++failures;                            \
      std::printf("FAILED %s: ", #cond);     \
      std::printf(__VA_ARGS__);              \
      std::printf("\n");                     \
    }                                        \
  } while (0)

static PagedView pool(int n_pages, int shift, int heads, int hd, bool heads_first, int pad) {
  PagedView kv{};
  kv.n_pages = n_pages;
  kv.page_shift = shift;
  kv.page_mask = (1 << shift) - 1;
  kv.n_kv_heads = heads;
  kv.hd = hd;
  const int64_t row = hd + pad, page = int64_t{1} << shift;
  kv.head_stride = heads_first ? page * row : row;
  kv.pos_stride = heads_first ? row : heads * row;
  kv.page_stride = page * heads * row;
  return kv;
}

int main() {
  const int wild[] = {INT_MIN, -1000000, -1, 0, 1, 2, 7, 15, 16, 17, 31, 32, 63, 64, 65, 1000, 1 << 20, INT_MAX};
  for (int shift : {0, 4, 10, 16})
    for (int max_pages : {0, 1, 3, 70000})
      for (int max_len : {0, 1, 33, 1 << 30})
        for (int len : wild) {
          const PagedView kv = pool(5, shift, 2, 64, false, 0);
          BatchView bt{nullptr, &len, nullptr, 1, 1, 1, max_len, max_pages};
          const int n = seq_len(bt, kv, 0);
          CHECK(n >= 0 && n <= max_len && (n == 0 || ((n - 1) >> shift) < max_pages), "len %d shift %d pages %d max_len %d", len, shift,
                max_pages, max_len);
          CHECK(len < 0 || len > max_len || (int64_t{len} > (int64_t{max_pages} << shift)) || n == len, "len %d kept", len);
        }
  for (int a : wild)
    for (int b : wild)
      for (int rows : {0, 1, 16, 1000})
        for (int max_new : {0, 1, 5, 1000}) {
          const int starts[2] = {a, b};
          BatchView bt{nullptr, nullptr, starts, 1, rows, max_new, 1, 1};
          const SeqRows r = seq_rows(bt, 0);
          CHECK(r.n >= 0 && r.n <= max_new && r.r0 >= 0 && r.r0 + r.n <= rows, "starts %d %d rows %d", a, b, rows);
          CHECK(r.n <= r.given, "starts %d %d: %d rows of %d", a, b, r.n, r.given);
        }
  std::vector<int> table(wild, wild + sizeof(wild) / sizeof(wild[0]));
  for (int shift : {0, 4})
    for (int n_pages : {1, 16, 1 << 20}) {
      const PagedView kv = pool(n_pages, shift, 2, 64, false, 0);
      BatchView bt{table.data(), nullptr, nullptr, 1, 1, 1, 1 << 30, static_cast<int>(table.size())};
      for (size_t i = 0; i < table.size(); ++i) {
        const int p = page_of(bt, kv, 0, static_cast<int>(i) << shift);
        CHECK(p == (table[i] >= 0 && table[i] < n_pages ? table[i] : -1), "page %d of %d", table[i], n_pages);
      }
    }
  for (bool heads_first : {false, true})
    for (int pad : {0, 8}) {
      const PagedView kv = pool(3, 4, 3, 64, heads_first, pad);
      std::set<int64_t> at;
      std::set<float*> w;
      PagedView kw = kv;
      kw.weight = reinterpret_cast<float*>(4096);
      for (int page = 0; page < 3; ++page)
        for (int pos = 32; pos < 48; ++pos)
          for (int h = 0; h < 3; ++h) {
            const int64_t e = elem_of(kv, page, pos, h);
            CHECK(e >= 0 && e + 64 <= 3 * kv.page_stride && e % 8 == 0, "element %lld", static_cast<long long>(e));
            at.insert(e);
            w.insert(weight_of(kw, page, pos, h));
          }
      CHECK(at.size() == 3 * 16 * 3 && w.size() == 3 * 16 * 3, "%zu rows, %zu weights", at.size(), w.size());
      CHECK(*w.rbegin() - *w.begin() == 3 * 16 * 3 - 1, "weights are dense");
    }
  const PagedView big = pool(1 << 20, 6, 8, 128, true, 0);
  CHECK(elem_of(big, (1 << 20) - 1, 63, 7) == int64_t{1 << 20} * 64 * 8 * 128 - 128, "last row of a pool past 32 bits");
  if (failures) return 1;
  std::printf("paged positions ok\n");
  return 0;
}
