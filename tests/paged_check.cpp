// CPU checks of the paged batch's host side (paged_plan.h): refusals, index rules, launch plan.
// Built and run by tests/test_paged_host.py; prints one line per failed check, exit code 1.
#include "../llmplayer_amd/csrc/paged_plan.h"

#include <cstdio>
#include <vector>

using namespace llmp;

static int failures = 0;
#define CHECK(x)                                                    \
    do {                                                            \
        if (!(x)) {                                                 \
            std::printf("line %d: %s\n", __LINE__, #x);             \
            ++failures;                                             \
        }                                                           \
    } while (0)

static int create(PagedShape s) {
    PagedMessage m;
    return paged_create_check(s, m);
}

static void refusals() {
    const PagedShape good{2, 100, 16, 1000, 8, 128, LLMP_KV_F32};
    CHECK(create(good) == LLMP_OK);
    CHECK(good.width() == 63);
    PagedShape s;
    for (int page : {0, -16, 1, 8, 15, 17, 24, 48, 96, 512}) {
        s = good, s.page_size = page;
        CHECK(create(s) == LLMP_ERR_INVALID_ARG);
    }
    for (int page : {16, 32, 64, 128, 256}) {
        s = good, s.page_size = page;
        CHECK(create(s) == LLMP_OK);
    }
    for (int d : {0, 32, 80, 100, 112, 512}) {
        s = good, s.head_dim = d;
        CHECK(create(s) == LLMP_ERR_UNSUPPORTED);
    }
    s = good, s.dtype = 3;
    CHECK(create(s) == LLMP_ERR_UNSUPPORTED);
    s = good, s.n_pages = 1 << 27;
    CHECK(create(s) == LLMP_ERR_INVALID_ARG);   // 2^31 slots
    s.n_pages = (1 << 27) - 1;
    CHECK(create(s) == LLMP_OK);
    s = good, s.max_seq = (1 << 30) + 1;
    CHECK(create(s) == LLMP_ERR_INVALID_ARG);
    for (int bad : {0, -1}) {
        s = good, s.n_layers = bad;
        CHECK(create(s) == LLMP_ERR_INVALID_ARG);
        s = good, s.n_pages = bad;
        CHECK(create(s) == LLMP_ERR_INVALID_ARG);
        s = good, s.max_seq = bad;
        CHECK(create(s) == LLMP_ERR_INVALID_ARG);
        s = good, s.n_kv_heads = bad;
        CHECK(create(s) == LLMP_ERR_INVALID_ARG);
    }

    PagedMessage m;
    const uint64_t ok[3] = {4, 8, 256}, null[3] = {4, 0, 8}, odd[3] = {4, 8, 6};
    auto tables = [&](int n, int shared, int tokens, const uint64_t* a) {
        return paged_tables_check(good, n, shared, tokens, a, 3, m);
    };
    CHECK(tables(1, 0, 1, ok) == LLMP_OK);
    CHECK(tables(kTablesMaxSeqs, 63, 1, ok) == LLMP_OK);
    CHECK(tables(0, 0, 1, ok) == LLMP_ERR_INVALID_ARG);
    CHECK(tables(kTablesMaxSeqs + 1, 0, 1, ok) == LLMP_ERR_INVALID_ARG);
    CHECK(tables(1, -1, 1, ok) == LLMP_ERR_INVALID_ARG);
    CHECK(tables(1, 64, 1, ok) == LLMP_ERR_INVALID_ARG);
    CHECK(tables(1, 0, 0, ok) == LLMP_ERR_INVALID_ARG);
    CHECK(tables(1, 0, 1, null) == LLMP_ERR_INVALID_ARG);
    CHECK(tables(1, 0, 1, odd) == LLMP_ERR_INVALID_ARG);

    const int64_t qd = 32 * 128, kvd = 8 * 128;
    auto append = [&](int tokens, uint64_t slots, int type, uint64_t q, int64_t qs, uint64_t k, int64_t ks, uint64_t v,
                      int64_t vs, uint64_t o, int64_t os) {
        return paged_append_check(good, 32, tokens, 4, slots, type, q, qs, k, ks, v, vs, o, os, m);
    };
    CHECK(append(1, 4, LLMP_IN_F32, 4, qd, 8, kvd, 12, kvd, 16, qd) == LLMP_OK);
    CHECK(append(1, 4, LLMP_IN_BF16, 2, qd, 6, kvd, 10, kvd, 16, qd) == LLMP_OK);
    CHECK(append(1, 0, LLMP_IN_F32, 4, qd, 0, 0, 0, 0, 16, qd) == LLMP_OK);
    CHECK(append(1, 4, LLMP_IN_F32, 16, qd, 8, kvd, 12, kvd, 16, qd) == LLMP_OK);            // in place
    CHECK(append(0, 4, LLMP_IN_F32, 4, qd, 8, kvd, 12, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 4, 2, 4, qd, 8, kvd, 12, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 0, LLMP_IN_F32, 4, qd, 8, kvd, 12, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 4, LLMP_IN_F32, 4, qd, 8, kvd, 0, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 4, LLMP_IN_F32, 0, qd, 8, kvd, 12, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 4, LLMP_IN_F32, 4, qd, 8, kvd, 12, kvd, 0, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 4, LLMP_IN_F32, 2, qd, 8, kvd, 12, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 4, LLMP_IN_BF16, 3, qd, 8, kvd, 12, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 6, LLMP_IN_F32, 4, qd, 8, kvd, 12, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 4, LLMP_IN_F32, 4, qd - 1, 8, kvd, 12, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 4, LLMP_IN_F32, 4, qd, 8, kvd - 1, 12, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 4, LLMP_IN_F32, 4, qd, 8, kvd, 12, 0, 16, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 4, LLMP_IN_F32, 4, qd, 8, kvd, 12, kvd, 16, 0) == LLMP_ERR_INVALID_ARG);
    CHECK(append(1, 4, LLMP_IN_BF16, 16, qd, 8, kvd, 12, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);   // in place, bf16
    CHECK(append(1, 4, LLMP_IN_F32, 16, qd + 4, 8, kvd, 12, kvd, 16, qd) == LLMP_ERR_INVALID_ARG);

    auto attn = [&](int n, int tokens, int prefix, int longest, uint64_t q, int64_t qs, uint64_t gate, uint64_t o,
                    int64_t os, uint64_t blocks = 4) {
        return paged_attn_check(good, 32, n, tokens, prefix, longest, 4, 8, blocks, q, qs, gate, o, os, m);
    };
    CHECK(attn(1, 1, 0, 0, 16, qd, 0, 32, qd) == LLMP_OK);
    CHECK(attn(1, 1, 1000, 1000, 16, qd + 4, 4, 32, qd + 8) == LLMP_OK);
    CHECK(attn(0, 1, 0, 0, 16, qd, 0, 32, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(attn(1, 0, 0, 0, 16, qd, 0, 32, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(attn(1, 1 << 26, 0, 0, 16, qd, 0, 32, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(attn(1, 1, -1, 0, 16, qd, 0, 32, qd) == LLMP_ERR_OUT_OF_RANGE);
    CHECK(attn(1, 1, 1001, 0, 16, qd, 0, 32, qd) == LLMP_ERR_OUT_OF_RANGE);
    CHECK(attn(1, 1, 0, 1001, 16, qd, 0, 32, qd) == LLMP_ERR_OUT_OF_RANGE);
    CHECK(attn(1, 1, 0, 0, 0, qd, 0, 32, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(attn(1, 1, 0, 0, 16, qd, 0, 0, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(attn(1, 1, 0, 0, 16, qd, 0, 32, qd, 0) == LLMP_ERR_INVALID_ARG);
    CHECK(attn(1, 1, 0, 0, 8, qd, 0, 32, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(attn(1, 1, 0, 0, 16, qd, 2, 32, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(attn(1, 1, 0, 0, 16, qd, 0, 40, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(attn(1, 1, 0, 0, 16, qd + 2, 0, 32, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(attn(1, 1, 0, 0, 16, qd - 4, 0, 32, qd) == LLMP_ERR_INVALID_ARG);
    CHECK(attn(1, 1, 0, 0, 16, qd, 0, 32, qd - 4) == LLMP_ERR_INVALID_ARG);
}

static void index_rules() {
    for (int page : {-2147483647 - 1, -1, 100, 2147483647}) CHECK(!paged_page_ok(page, 100));
    for (int page : {0, 99}) CHECK(paged_page_ok(page, 100));
    for (int slot : {-2147483647 - 1, -1, 1600, 2147483647}) CHECK(!paged_slot_ok(slot, 4, 100));
    for (int slot : {0, 1599}) CHECK(paged_slot_ok(slot, 4, 100));
    const std::vector<int> s{0, 0, 3, 3, 3, 7};   // sequences of 0, 3, 0, 0, 4 tokens
    for (int x = 0; x < 7; ++x) CHECK(paged_owner(s.data(), 5, x) == (x < 3 ? 1 : 4));
    const int one = 0;
    CHECK(paged_owner(&one, 1, 5) == 0);
}

// Every sequence's items lie below the next one's base, and below the grid.
static void item_bases() {
    unsigned seed = 7;
    auto rnd = [&](unsigned n) { return (seed = seed * 1664525u + 1013904223u) / 65536u % n; };
    for (int t = 0; t < 2000; ++t) {
        const int n = 1 + rnd(40), group = 1 + rnd(24), rows = 16 << rnd(3), most = 1 + rnd(t % 2 ? 4 : 300);
        int start = 0;
        std::vector<int> st{0};
        for (int b = 0; b < n; ++b) st.push_back(start += rnd(most + 1));
        const int grid = (int)((long long)start * group / rows) + n;
        for (int b = 0; b < n; ++b) {
            const int items = ((st[b + 1] - st[b]) * group + rows - 1) / rows;
            const int end = paged_item_base(st[b], group, rows, b) + items;
            CHECK(end <= (b + 1 < n ? paged_item_base(st[b + 1], group, rows, b + 1) : grid));
        }
    }
    CHECK(paged_item_base(-5, 4, 16, 3) == 3);
}

static void plans() {
    for (int n : {1, 7, 64, 4096})
        for (int tokens : {1, 5, 64, 5000})
            for (int hq : {1, 4, 32, 48})
                for (int hkv : {1, 2, 4, 8}) {
                    if (hq % hkv) continue;
                    for (int d : {64, 96, 128, 256})
                        for (int prefix : {0, 1, 31, 32, 33, 5000, 131072})
                            for (int longest : {1, 33, 5001, 140000}) {
                                const PagedPlan p = paged_plan(n, tokens, hq, hkv, d, prefix, longest, 256);
                                CHECK(p.own_splits >= 1 && p.own_splits <= 65535);
                                CHECK(p.own_wide >= 0 && p.own_wide <= paged_wide_max(d) && p.own_wide <= p.prefix_wide);
                                CHECK(p.prefix_wide <= paged_wide_max(d));
                                if (prefix == 0) {
                                    CHECK(p.prefix_splits == 0);
                                    continue;
                                }
                                const int tiles = (prefix + 31) / 32;
                                CHECK(p.prefix_splits >= 1 && p.prefix_splits <= 65535);
                                CHECK((long long)p.prefix_splits * p.prefix_tiles >= tiles);
                                CHECK((long long)(p.prefix_splits - 1) * p.prefix_tiles < tiles);
                            }
                }
}

int main() {
    refusals();
    index_rules();
    item_bases();
    plans();
    return failures ? 1 : 0;
}
