// The paged 4-bit KV cache's layout, checks and launch shapes, asked line by
// line on stdin (host headers only):
//   at t d                  -> K word, K nibble, V word, V nibble of a half page
//   meta t group            -> f16 index of the scale and of the minimum
//   splits len batch cus    -> bound of the decode's splits, its workspace, the reserve that covers it
//   cache pages table lens refs layers num_pages rows max_pages
//                           -> the cache that the following calls name
//   resize count rows lens flags result
//   fork count src dst result
//   compact live
//   rows layer row batch first n k v capacity
//   decode layer batch slots ptr rope_len max_len result
//                           -> status code, message
#include <iostream>
#include <string>

#include "qm_kv4_check.h"

namespace {
template <class T>
T* at(uint64_t a) { return reinterpret_cast<T*>(static_cast<uintptr_t>(a)); }
void say(const qm_kv4::Fault& f) { std::cout << f.code << " " << f.text << "\n"; }
}  // namespace

int main() {
    std::string what;
    qm_kv4_cache c{};
    while (std::cin >> what) {
        int64_t i[4];
        uint64_t p[4];
        if (what == "at" && std::cin >> i[0] >> i[1]) {
            const int t = static_cast<int>(i[0]), d = static_cast<int>(i[1]);
            std::cout << kv4_k_word(t, d) << " " << kv4_k_nibble(d) << " " << kv4_v_word(t, d) << " " << kv4_v_nibble(t) << "\n";
        } else if (what == "meta" && std::cin >> i[0] >> i[1]) {
            std::cout << kv4_s_at(static_cast<int>(i[0]), static_cast<int>(i[1])) << " "
                      << kv4_lo_at(static_cast<int>(i[0]), static_cast<int>(i[1])) << "\n";
        } else if (what == "splits" && std::cin >> i[0] >> i[1] >> i[2]) {
            const int cus = static_cast<int>(i[2]);
            const int64_t n = qm_kv4::max_splits(i[0], i[1], cus);
            std::cout << n << " " << qm_kv4::decode_ws(n, static_cast<int32_t>(i[1])) << " "
                      << qm_kv4::reserve_ws(static_cast<int32_t>(i[1]), static_cast<int32_t>(i[0]), cus) << "\n";
        } else if (what == "cache" && std::cin >> p[0] >> p[1] >> p[2] >> p[3] >> i[0] >> i[1] >> i[2] >> i[3]) {
            c = qm_kv4_cache{at<uint8_t>(p[0]), at<int32_t>(p[1]), at<int32_t>(p[2]), at<int32_t>(p[3]),
                             static_cast<int32_t>(i[0]), static_cast<int32_t>(i[1]), static_cast<int32_t>(i[2]),
                             static_cast<int32_t>(i[3])};
            std::cout << "ok\n";
        } else if (what == "resize" && std::cin >> i[0] >> p[0] >> p[1] >> i[1] >> p[2]) {
            say(qm_kv4::check_resize(&c, static_cast<int32_t>(i[0]), at<int32_t>(p[0]), at<int32_t>(p[1]),
                                     static_cast<int32_t>(i[1]), at<int32_t>(p[2])));
        } else if (what == "fork" && std::cin >> i[0] >> p[0] >> p[1] >> p[2]) {
            say(qm_kv4::check_list("qm_kv4_fork", &c, static_cast<int32_t>(i[0]), {at<void>(p[0]), at<void>(p[1])}, at<void>(p[2])));
        } else if (what == "compact" && std::cin >> p[0]) {
            say(qm_kv4::check_list("qm_kv4_compact", &c, 1, {}, at<void>(p[0])));
        } else if (what == "rows" && std::cin >> i[0] >> i[1] >> i[2] >> p[0] >> i[3] >> p[1] >> p[2] >> p[3]) {
            say(qm_kv4::check_rows("qm_kv4_store", &c, static_cast<int32_t>(i[0]), static_cast<int32_t>(i[1]),
                                   static_cast<int32_t>(i[2]), at<int32_t>(p[0]), static_cast<int32_t>(i[3]),
                                   at<uint16_t>(p[1]), at<uint16_t>(p[2]), static_cast<int64_t>(p[3])));
        } else if (what == "decode" && std::cin >> i[0] >> i[1] >> p[0] >> p[1] >> i[2] >> i[3] >> p[2]) {
            say(qm_kv4::check_decode(&c, static_cast<int32_t>(i[0]), static_cast<int32_t>(i[1]), at<int32_t>(p[0]),
                                     {at<void>(p[1])}, static_cast<int32_t>(i[2]), static_cast<int32_t>(i[3]), at<int32_t>(p[2])));
        } else {
            return 1;
        }
    }
    return 0;
}
