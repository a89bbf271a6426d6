// The work list of a paged attention call (host): one (sequence, query tile)
// pair per tile of `rows` query rows that holds rows, heaviest first (most
// keys to read; ties in sequence and tile order).
#pragma once

#include <stdint.h>

#include <algorithm>
#include <vector>

#include "qx_status.h"

namespace qx {

// -> the number of items (<= capacity), or QX_EINVAL
inline int64_t attention_work_list(const int* cu_q, const int* used, int64_t seqs, int rows,
                                   int causal, int* work, int64_t capacity) {
  struct Item { int64_t load; int s, qt; };
  std::vector<Item> items;
  for (int64_t s = 0; s < seqs; ++s) {
    const int q_len = cu_q[s + 1] - cu_q[s];
    const int u = used[s];
    for (int qt = 0; qt * rows < q_len; ++qt) {
      const int last = std::min(qt * rows + rows, q_len) - 1;
      const int keys = causal ? std::min(u, u - q_len + last + 1) : u;
      items.push_back({(int64_t)keys, (int)s, qt});
    }
  }
  if ((int64_t)items.size() > capacity) {
    set_error("attention_work: %zu items exceed the capacity %lld", items.size(),
              (long long)capacity);
    return QX_EINVAL;
  }
  std::stable_sort(items.begin(), items.end(),
                   [](const Item& a, const Item& b) { return a.load > b.load; });
  for (size_t i = 0; i < items.size(); ++i) {
    work[2 * i] = items[i].s;
    work[2 * i + 1] = items[i].qt;
  }
  return (int64_t)items.size();
}

}  // namespace qx
