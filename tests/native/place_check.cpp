// CPU check of lucid_amd/csrc/lq_place.h: places of packed tokens and cached positions, with
// starts, lengths and page numbers that are wrong in every way a caller can get them wrong.
// Built and run by tests/test_generation_host.py; prints "ok" and exits 0 on success.
#include <cstdint>
#include <cstdio>
#include <vector>

#include "lq_place.h"

using namespace lq;

static int fails = 0;
#define CHECK(c)                                                        \
    do {                                                                \
        if (!(c)) {                                                     \
            std::fprintf(stderr, "line %d: %s\n", __LINE__, #c);        \
            ++fails;                                                    \
        }                                                               \
    } while (0)

static void positions() {
    const int64_t Hkv = 3, page = 5, pages = 4, stride = 3;
    const int32_t ids[] = {2, -1, 4, 0x7fffffff, INT32_MIN, 0, 3};
    for (int32_t a : ids)
        for (int32_t b : ids) {
            const int32_t row[3] = {a, b, 1};
            for (int64_t pos = -3; pos < 20; ++pos) {
                const int64_t r = position_row(pos, row, stride, pages, Hkv, page);
                if (pos < 0 || pos >= stride * page) {
                    CHECK(r == -1);
                    continue;
                }
                const int64_t id = row[pos / page];
                if (id < 0 || id >= pages) CHECK(r == -1);
                else CHECK(r == id * Hkv * page + pos % page && r + (Hkv - 1) * page < pages * Hkv * page);
            }
        }
    const int32_t none[1] = {0};
    CHECK(position_row(0, none, 0, pages, Hkv, page) == -1);  // a table without columns is not read
    CHECK(position_row(0, none, 1, 0, Hkv, page) == -1);      // an empty pool
    // past 32 bits
    const int32_t far[1] = {70000};
    CHECK(position_row(63, far, 1, 70001, 512, 64) == 70000ll * 512 * 64 + 63);
}

static void tokens() {
    const int32_t starts[] = {0, 3, 3, 4, 10};
    const int32_t lengths[] = {3, 7, 1, 20};
    const int64_t want_seq[] = {0, 0, 0, 2, 3, 3, 3, 3, 3, 3};
    const int64_t want_pos[] = {0, 1, 2, 0, 14, 15, 16, 17, 18, 19};
    int64_t s, p;
    for (int64_t t = 0; t < 10; ++t) CHECK(token_place(t, starts, 4, lengths, s, p) && s == want_seq[t] && p == want_pos[t]);
    CHECK(!token_place(10, starts, 4, lengths, s, p));
    const int32_t late[] = {2, 4};
    CHECK(!token_place(0, late, 1, lengths, s, p));
    const int32_t one[] = {0, 5};
    CHECK(token_place(1, nullptr, 2, one, s, p) && s == 1 && p == 4);
    CHECK(token_place(0, nullptr, 2, one, s, p) && p == -1);  // a sequence of length 0 takes no token
    // any contents of starts stay in range
    const int32_t junk[] = {9, -4, 0x7fffffff, INT32_MIN, 2};
    for (int64_t t = 0; t < 12; ++t) {
        const int64_t q = sequence_of(junk, 4, t);
        CHECK(q >= 0 && q < 4);
        token_place(t, junk, 4, lengths, s, p);
        CHECK(s >= 0 && s < 4);
    }
}

static void packed() {
    const int32_t vals[] = {0, 5, -7, 100, 3, INT32_MIN, 0x7fffffff};
    for (int32_t a : vals)
        for (int32_t b : vals)
            for (int32_t c : vals)
                for (int32_t d : vals) {
                    const int32_t qs[] = {a, b}, ks[] = {c, d};
                    const Packed p = packed_sequence(qs, ks, 0, 50, 60);
                    CHECK(p.q0 >= 0 && p.nq >= 0 && p.q0 + p.nq <= 50);
                    CHECK(p.k0 >= 0 && p.nk >= 0 && p.k0 + p.nk <= 60);
                    for (int64_t i = 0; i < p.nq; ++i) {
                        const int64_t n = keys_seen(p, i, true);
                        CHECK(n >= 0 && n <= p.nk && (i + 1 < p.nq || n == p.nk));
                        CHECK(keys_seen(p, i, false) == p.nk);
                    }
                }
    const Packed few{0, 5, 0, 2};  // more queries than keys: the first ones see nothing
    CHECK(keys_seen(few, 2, true) == 0 && keys_seen(few, 3, true) == 1 && keys_seen(few, 4, true) == 2);
}

int main() {
    positions();
    tokens();
    packed();
    if (fails) return 1;
    std::puts("ok");
    return 0;
}
