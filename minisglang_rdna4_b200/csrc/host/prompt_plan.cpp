// Tables of a prompt step over a 4-bit K/V pool, exported with C linkage for ctypes: what ops/cuda.py::PrefillPlan builds with
// NumPy, in a few microseconds where some twenty array operations take 80 (two requests of some 2000 rows each).
#include <algorithm>
#include <cstdint>
#include <vector>

namespace {

constexpr int64_t kLongest = 1 << 30;      // lengths are 32-bit numbers here and in the kernels

// start of the block of 128 positions that holds the first position a row at `pos` can see
int64_t first_block(int64_t pos, int64_t window) { return window > 0 ? std::max<int64_t>(0, pos - window + 1) / 128 * 128 : 0; }

}  // namespace

extern "C" {

// `out` (`room` words): per (request, block of `tile` rows) first row, rows, first position, scratch row of the first key in sight,
// blocks of 128 keys, request, position of that key, 0, the most blocks first; the request of every 128-row block of the scratch; per
// request scratch row, length, first key. `info`: rows of the scratch, items, rows, longest request, words of the tables. Returns 1; 0
// where the tables are larger than `room` (`info` is complete); -1 where a request has more rows than tokens, or fewer than none, or a row in
// front of the first.
__attribute__((visibility("default"))) int msgl_prompt_plan(const int64_t* cu_q, const int64_t* lens, int64_t b, int64_t window,
                                                            int64_t tile, int32_t* out, int64_t room, int64_t* info) {
  int64_t t_pad = 0, n_items = 0, longest = 0;
  if (b > 0 && cu_q[0] < 0) return -1;
  for (int64_t i = 0; i < b; ++i) {
    const int64_t rows = cu_q[i + 1] - cu_q[i], n = std::min(lens[i], kLongest);
    if (rows < 0 || rows > n || cu_q[i + 1] > kLongest) return -1;
    t_pad += (n - first_block(n - rows, window) + 127) / 128 * 128;
    n_items += (rows + tile - 1) / tile;
    longest = std::max(longest, n);
  }
  const int64_t words = 8 * n_items + t_pad / 128 + 3 * b;
  info[0] = t_pad;
  info[1] = n_items;
  info[2] = b > 0 ? cu_q[b] : 0;
  info[3] = longest;
  info[4] = words;
  if (words > room) return 0;
  struct Item { int32_t x[8]; };
  std::vector<Item> items;
  items.reserve(n_items);
  int32_t *blocks = out + 8 * n_items, *requests = blocks + t_pad / 128;
  int64_t at = 0;
  for (int64_t i = 0; i < b; ++i) {
    const int64_t rows = cu_q[i + 1] - cu_q[i], n = std::min(lens[i], kLongest), lo = first_block(n - rows, window);
    for (int64_t r = 0; r < rows; r += tile) {
      const int64_t some = std::min(tile, rows - r), pos = n - rows + r, key = first_block(pos, window);
      items.push_back({{(int32_t)(cu_q[i] + r), (int32_t)some, (int32_t)pos, (int32_t)(at + key - lo),
                        (int32_t)((pos + some - key + 127) / 128), (int32_t)i, (int32_t)key, 0}});
    }
    const int64_t pad = (n - lo + 127) / 128 * 128;
    std::fill(blocks, blocks + pad / 128, (int32_t)i);
    blocks += pad / 128;
    requests[3 * i] = (int32_t)at;
    requests[3 * i + 1] = (int32_t)n;
    requests[3 * i + 2] = (int32_t)lo;
    at += pad;
  }
  std::stable_sort(items.begin(), items.end(), [](const Item& x, const Item& y) { return x.x[4] > y.x[4]; });
  std::copy_n(reinterpret_cast<const int32_t*>(items.data()), 8 * n_items, out);
  return 1;
}

}  // extern "C"
