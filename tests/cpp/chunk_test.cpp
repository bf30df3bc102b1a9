// What the host checks, and the workspaces that it asks for, of the calls for
// chunks of new tokens and for beam search's step, asked line by line on stdin
// (host headers only; addresses are numbers that nothing reads):
//   append|chunk|select|fork key=value ...  -> the status and its message; keys that
//                                              are not given have values that pass
//   shape tokens batch max_new max_len cus  -> row blocks of many tokens and of few at
//                                              most, workgroups per kv head, workspace
//   reserve tokens batch max_len cus        -> what a reserve asks for
//   halves tokens batch                     -> half pages at most
//   slices rows vocab                       -> workspace of a selection
//   column count                            -> bytes of a row that a workgroup takes
#include <iostream>
#include <map>
#include <sstream>
#include <string>
#include <vector>

#include "qm_beam_check.h"

namespace {

struct Keys {
    std::map<std::string, int64_t> given;
    int64_t operator()(const char* key, int64_t otherwise) const {
        const auto at = given.find(key);
        return at == given.end() ? otherwise : at->second;
    }
    template <class T>
    T* pointer(const char* key, int64_t otherwise) const {
        return reinterpret_cast<T*>(static_cast<intptr_t>((*this)(key, otherwise)));
    }
};

qm_kv4_cache cache_of(const Keys& k) {
    qm_kv4_cache c{};
    c.pages_dev = k.pointer<uint8_t>("pages", 0x1000);
    c.table_dev = k.pointer<int32_t>("table", 0x2000);
    c.lens_dev = k.pointer<int32_t>("lens", 0x3000);
    c.refs_dev = k.pointer<int32_t>("refs", 0x4000);
    c.num_pages = static_cast<int32_t>(k("num_pages", 64));
    c.max_pages = static_cast<int32_t>(k("max_pages", 16));
    c.rows = static_cast<int32_t>(k("rows", 8));
    c.layers = static_cast<int32_t>(k("layers", 2));
    return c;
}

qm_kv4::Fault check(const std::string& what, const Keys& k) {
    const qm_kv4_cache cache = cache_of(k);
    const qm_kv4_cache* c = k("cache", 1) ? &cache : nullptr;
    const auto n = [&](const char* key, int64_t otherwise) { return static_cast<int32_t>(k(key, otherwise)); };
    const auto p = [&](const char* key) { return k.pointer<const void>(key, 0x10000); };
    const int32_t *slots = k.pointer<int32_t>("slots", 0), *begins = k.pointer<int32_t>("begins", 0x5000), *result = k.pointer<int32_t>("result", 0);
    if (what == "append")
        return qm_kv4::check_append(c, n("layer", 0), n("batch", 4), slots, begins, n("tokens", 100), n("dtype", QM_F32),
                                    {p("k"), p("v"), p("norm"), p("cos"), p("sin")}, n("rope_len", 1024), n("max_len", 1024), result);
    if (what == "chunk")
        return qm_kv4::check_chunk(c, n("layer", 0), n("batch", 4), slots, begins, n("tokens", 100), n("max_new", 50),
                                   {p("q"), p("norm"), p("cos"), p("sin"), p("out")}, n("rope_len", 1024), n("max_len", 1024), result);
    if (what == "select")
        return qm_beam::check_select(n("groups", 3), n("beams", 4), n("take", 4), n("vocab", 1000), k.pointer<float>("logits", 0x100),
                                     k.pointer<float>("scores", 0x200), k.pointer<int32_t>("done", 0), n("end_id", -1),
                                     k.pointer<int32_t>("parents", 0x300), k.pointer<int32_t>("tokens", 0x400),
                                     k.pointer<float>("out_scores", 0x500), k.pointer<int32_t>("out_done", 0));
    const int32_t buffers = n("buffers", 2);
    std::vector<qm_state_rows> list(buffers > 0 && buffers < 1000 ? buffers : 1);
    for (auto& b : list) b = qm_state_rows{reinterpret_cast<void*>(0x1000), 64, 128};
    list.back() = qm_state_rows{k.pointer<void>("rows_dev", 0x1000), k("row_bytes", 64), k("stride_bytes", 64)};
    return qm_beam::check_fork(buffers, k("list", 1) ? list.data() : nullptr, n("rows", 10), n("count", 4), k.pointer<int32_t>("src", 0x100),
                               k.pointer<int32_t>("dst", 0), k.pointer<int32_t>("result", 0x200));
}

}  // namespace

int main() {
    std::string line;
    while (std::getline(std::cin, line)) {
        std::istringstream in(line);
        std::string what;
        in >> what;
        if (what == "shape") {
            int32_t tokens, batch, max_new, max_len;
            int cus;
            in >> tokens >> batch >> max_new >> max_len >> cus;
            const qm_kv4::Chunk c = qm_kv4::chunk_shape(tokens, batch, max_new, max_len, cus);
            std::cout << c.columns << " " << c.many << " " << c.split << " " << c.most_many << " " << c.most_few << " " << c.groups << " "
                      << qm_kv4::chunk_ws(c) << "\n";
        } else if (what == "reserve") {
            int32_t tokens, batch, max_len;
            int cus;
            in >> tokens >> batch >> max_len >> cus;
            std::cout << qm_kv4::chunk_reserve_ws(tokens, batch, max_len, cus) << "\n";
        } else if (what == "halves") {
            int32_t tokens, batch;
            in >> tokens >> batch;
            std::cout << qm_kv4::append_halves(tokens, batch) << "\n";
        } else if (what == "slices") {
            int64_t rows;
            int32_t vocab;
            in >> rows >> vocab;
            std::cout << qm_beam::select_ws(rows, vocab) << "\n";
        } else if (what == "column") {
            int32_t count;
            in >> count;
            std::cout << qm_beam::fork_column(count) << "\n";
        } else {
            Keys keys;
            std::string word;
            while (in >> word) {
                const size_t at = word.find('=');
                keys.given[word.substr(0, at)] = std::stoll(word.substr(at + 1));
            }
            const qm_kv4::Fault f = check(what, keys);
            std::cout << f.code << " " << f.text << "\n";
        }
    }
    return 0;
}
