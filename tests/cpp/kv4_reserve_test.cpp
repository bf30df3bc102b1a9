// Workspaces of the 4-bit KV cache's calls at the limits that a reserve is
// promised for, asked line by line on stdin (host headers only):
//   batch len cus -> bytes of a resize and a fork of `batch` rows in a table
//                    of ceil(len / 64) pages a row, of a compaction of a pool
//                    that `batch` such rows fill, of a step, and of the reserve
#include <algorithm>
#include <iostream>

#include "qm_kv4_check.h"

int main() {
    int64_t batch, len;
    int cus;
    while (std::cin >> batch >> len >> cus) {
        const int32_t pages = kv4_pages_of(static_cast<int32_t>(len));
        const int32_t count = static_cast<int32_t>(std::min<int64_t>(batch, QMK_KV4_MAX_COUNT));
        const int64_t pool = std::min<int64_t>(batch * pages, QMK_KV4_MAX_PAGES);
        std::cout << qm_kv4::resize_ws(count) << " " << qm_kv4::fork_ws(count, pages) << " "
                  << qm_kv4::compact_ws(static_cast<int32_t>(pool)) << " "
                  << qm_kv4::decode_ws(qm_kv4::max_splits(len, batch, cus), static_cast<int32_t>(batch)) << " "
                  << qm_kv4::reserve_ws(static_cast<int32_t>(batch), static_cast<int32_t>(len), cus) << "\n";
    }
    return 0;
}
