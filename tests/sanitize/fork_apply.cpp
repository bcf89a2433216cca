// A fork whose work outside the page lists fails leaves the pager as it was:
// no open stream, every page and slot back, the next fork as if nothing had been.
#include <cstdio>
#include <cstdlib>
#include <string>

#include "pager.h"
#include "qkv.h"

#define REQUIRE(cond)                                                   \
    do {                                                                \
        if (!(cond)) {                                                  \
            std::fprintf(stderr, "line %d: %s\n", __LINE__, #cond);     \
            std::exit(1);                                               \
        }                                                               \
    } while (0)

int main() {
    qkv::Pager p(12, 16, 2, 8, 7);
    std::string err;
    int32_t a = -1;
    REQUIRE(p.open(&a, &err) == QKV_OK && p.append(a, 70, nullptr, &err) == QKV_OK);
    const std::vector<int32_t> before = *p.pages(a);
    for (int32_t tokens : {70, 64, 33, 0}) {
        int32_t inner = -1, src = -2, dst = -2, out = -9;
        int calls = 0;
        const int64_t free_pages = p.free_pages();
        for (int k = 0; k < 20; ++k) {   // more often than there are slots and pages
            const int rc = qkv::fork_and_apply(p, a, tokens, &out, &err, [&](int32_t s, int32_t from, int32_t to) {
                ++calls;
                inner = s;
                src = from;
                dst = to;
                REQUIRE(p.is_open(s) && (tokens % 16 != 0) == (to >= 0));
                return static_cast<int>(QKV_ERR_CUDA);
            });
            REQUIRE(rc == QKV_ERR_CUDA && out == -9 && !p.is_open(inner));
            REQUIRE(p.free_pages() == free_pages && *p.pages(a) == before && p.check(&err) == QKV_OK);
        }
        REQUIRE(calls == 20);
        int32_t length = -1;
        const int rc = qkv::fork_and_apply(p, a, tokens, &out, &err, [&](int32_t s, int32_t from, int32_t to) {
            return s == inner && from == src && to == dst ? 0 : 1;
        });
        REQUIRE(rc == QKV_OK && out == inner && p.length(out, &length, &err) == QKV_OK && length == tokens);
        REQUIRE(p.close(out, &err) == QKV_OK && p.check(&err) == QKV_OK && p.free_pages() == free_pages);
    }
    // A refused fork calls nothing.
    int32_t out = -9;
    REQUIRE(qkv::fork_and_apply(p, a, 71, &out, &err, [](int32_t, int32_t, int32_t) { std::abort(); return 0; }) ==
            QKV_ERR_INVALID_ARG);
    std::puts("ok");
    return 0;
}
