// CPU check of the paged cache's host arithmetic (paged_plan.h), built with
// g++ and its sanitizers: what the entry points refuse, and that the steps of
// a set of page copies, run as the kernel runs them (chains in any order, a
// chain's steps one after another with one held and one saved page), leave
// every page as if all sources had been read before any destination was
// written. Exit status 0 when every case holds.
#include <cmath>
#include <cstdio>
#include <functional>
#include <numeric>
#include <random>

#include "../csrc/paged_plan.h"

namespace paged = qwh::paged;

namespace {

long cases = 0, failures = 0;

void expect(bool ok, const char *what, long a = 0, long b = 0) {
    ++cases;
    if (ok) return;
    if (++failures <= 20) std::printf("FAIL %s (%ld, %ld)\n", what, a, b);
}

// A launch, as paged_copy_kernel runs it.
template <typename Steps>
void run(const Steps &s, std::vector<uint64_t> &pool, std::mt19937 &rng) {
    std::vector<uint32_t> chains(s.chains);
    std::iota(chains.begin(), chains.end(), 0u);
    std::shuffle(chains.begin(), chains.end(), rng);
    for (uint32_t c : chains) {
        uint64_t v = ~0ull, saved = ~0ull;
        uint32_t held = paged::kSaved;
        expect(s.begin(c) < s.end(c), "empty chain", c);
        for (uint32_t i = s.begin(c); i < s.end(c); ++i) {
            const uint32_t src = s.source(i), dst = s.target(i);
            if (dst == paged::kSaved) {
                saved = pool[src];
            } else if (src == paged::kSaved) {
                pool[dst] = saved;
                held = paged::kSaved;
            } else {
                if (src != held) v = pool[src];
                held = src;
                pool[dst] = v;
            }
        }
    }
}

void copies(const std::vector<uint32_t> &src, const std::vector<uint32_t> &dst, uint32_t pages, std::mt19937 &rng,
            const char *what) {
    paged::CopyPairs pairs;
    const paged::Refusal r = paged::check_copies(src.data(), dst.data(), (uint32_t)src.size(), pages, pairs);
    expect(r.status == QWH_OK, what, (long)src.size(), pages);
    if (r.status != QWH_OK) return;
    size_t moved = 0;
    for (size_t i = 0; i < src.size(); ++i) moved += src[i] != dst[i];
    for (const bool is_short : {false, true}) {
        if (is_short && pages > paged::kShortPages) continue;
        paged::CopyLaunches plan(is_short);
        paged::order_copies(pairs, plan);
        std::vector<uint64_t> pool(pages);
        std::iota(pool.begin(), pool.end(), 1000ull);
        std::vector<uint64_t> want = pool;
        for (size_t i = 0; i < src.size(); ++i) want[dst[i]] = pool[src[i]];
        size_t steps = 0;
        for (const paged::CopyLaunch &l : plan.launches) {
            expect(l.chains() >= 1 && l.chain[l.chains()] == l.steps(), "launch size", l.chains());
            expect(is_short ? l.steps() + (l.chains() == l.steps() ? 0 : (l.chains() + 2) / 2) <= paged::kShortWords
                            : l.steps() <= paged::kMaxSteps, "launch size", l.steps());
            steps += l.steps();
            if (is_short) run(paged::pack_short(l), pool, rng);
            else run(paged::pack(l), pool, rng);
        }
        expect(steps <= 2 * moved, "more than two steps a page", (long)steps, (long)moved);
        expect(pool == want, what, (long)src.size(), pages);
    }
}

void check_copies() {
    std::mt19937 rng(7);
    const auto range = [](uint32_t n, uint32_t first) {
        std::vector<uint32_t> v(n);
        std::iota(v.begin(), v.end(), first);
        return v;
    };
    copies({0}, {0}, 1, rng, "a page onto itself");
    copies({0, 1}, {1, 0}, 2, rng, "swap");
    copies({0, 0, 0, 0}, {1, 2, 3, 4}, 5, rng, "fork");
    copies({0, 0, 1, 1, 0}, {1, 2, 3, 4, 0}, 5, rng, "fork and chain");
    for (uint32_t n : {2u, 3u, 17u, 381u, 382u, 383u, 384u, 385u, 386u, 767u, 768u, 988u, 989u, 990u, 991u, 2000u}) {
        // A cycle through n pages, with readers hanging off it, and a chain.
        std::vector<uint32_t> src = range(n, 0), dst = range(n, 1);
        dst[n - 1] = 0;
        copies(src, dst, n, rng, "cycle");
        for (uint32_t k = 0; k < n; k += 3) {
            src.push_back(k);
            dst.push_back(n + k);
        }
        copies(src, dst, 2 * n, rng, "cycle with forks");
        copies(range(n, 0), range(n, 1), n + 1, rng, "chain up");
        std::vector<uint32_t> down = range(n, 1);
        std::reverse(down.begin(), down.end());
        std::vector<uint32_t> to = range(n, 0);
        std::reverse(to.begin(), to.end());
        copies(down, to, n + 1, rng, "chain down");
        copies(std::vector<uint32_t>(n, 3 % (n + 4)), range(n, 4), n + 4, rng, "one page to many");
    }
    for (int round = 0; round < 4000; ++round) {
        const uint32_t pages = 1 + rng() % (round % 50 == 0 ? 3000 : 24);
        std::vector<uint32_t> dst = range(pages, 0);
        std::shuffle(dst.begin(), dst.end(), rng);
        dst.resize(rng() % (pages + 1));
        std::vector<uint32_t> src;
        const bool permuted = rng() % 2;
        std::vector<uint32_t> order = dst;
        std::shuffle(order.begin(), order.end(), rng);
        for (size_t i = 0; i < dst.size(); ++i) src.push_back(permuted ? order[i] : rng() % pages);
        copies(src, dst, pages, rng, "random pairs");
    }
    // Few pages of a large pool, and a pool so large that no bit a page is kept.
    for (uint32_t pages : {100000u, (1u << 20) + 256 * 5 + 1}) {
        const uint32_t p = pages - 6;
        copies({p, p + 1, p + 2, 7, 7}, {p + 1, p + 2, p, p + 4, p + 5}, pages, rng, "high pages");
        copies({p, p + 1, 3}, {p + 2, p + 3, p + 4}, pages, rng, "high pages apart");
    }
    paged::CopyPairs pairs;
    const uint32_t a[] = {1, 2}, b[] = {3, 3}, c[] = {1, 9};
    expect(paged::check_copies(a, b, 2, 1u << 31, pairs).status == QWH_E_INVALID_ARGUMENT, "a destination twice in a large pool");
    expect(paged::check_copies(a, b, 2, 9, pairs).status == QWH_E_INVALID_ARGUMENT, "a destination twice");
    expect(paged::check_copies(c, a, 2, 9, pairs).status == QWH_E_INVALID_ARGUMENT, "a source past the pool");
    expect(paged::check_copies(a, c, 2, 9, pairs).status == QWH_E_INVALID_ARGUMENT, "a destination past the pool");
}

void check_refusals() {
    alignas(16) static uint8_t plane[64];
    static uint32_t words[4];
    const qwh_paged_cache good{28, 4096, 16, 8, 128, plane, plane, plane, plane};
    expect(paged::check_cache(&good).status == QWH_OK, "a pool");
    expect(paged::check_cache(nullptr).status == QWH_E_INVALID_ARGUMENT, "no pool");
    const auto cache = [&](int32_t status, const char *what, const std::function<void(qwh_paged_cache &)> &change) {
        qwh_paged_cache c = good;
        change(c);
        expect(paged::check_cache(&c).status == status, what);
    };
    qwh_paged_cache page = good;
    page.pages = 2;
    page.page_size = 1u << 23;
    expect(paged::check_page(page).status == QWH_OK, "pages of 8 GiB");
    page.page_size += 1;
    expect(paged::check_page(page).status == QWH_E_LIMIT_EXCEEDED, "pages of more");
    cache(QWH_E_SHAPE_MISMATCH, "no layers", [](auto &c) { c.layers = 0; });
    cache(QWH_E_SHAPE_MISMATCH, "no pages", [](auto &c) { c.pages = 0; });
    cache(QWH_E_SHAPE_MISMATCH, "pages of no position", [](auto &c) { c.page_size = 0; });
    cache(QWH_E_SHAPE_MISMATCH, "no heads", [](auto &c) { c.kv_heads = 0; });
    cache(QWH_E_SHAPE_MISMATCH, "head_dim 0", [](auto &c) { c.head_dim = 0; });
    cache(QWH_E_SHAPE_MISMATCH, "head_dim 96", [](auto &c) { c.head_dim = 96; });
    cache(QWH_E_UNSUPPORTED, "head_dim 320", [](auto &c) { c.head_dim = 320; });
    cache(QWH_E_LIMIT_EXCEEDED, "heads", [](auto &c) { c.kv_heads = 4097; });
    cache(QWH_E_LIMIT_EXCEEDED, "2^32 - 1 rows", [](auto &c) { c.pages = 0xffffffffu, c.page_size = 1; });
    cache(QWH_OK, "2^30 rows", [](auto &c) { c.pages = 1u << 30, c.page_size = 1, c.kv_heads = 1, c.head_dim = 64, c.pages -= 1; });
    cache(QWH_E_LIMIT_EXCEEDED, "2^33 rows", [](auto &c) { c.pages = 1u << 17, c.page_size = 1u << 16; });
    cache(QWH_E_LIMIT_EXCEEDED, "bytes", [](auto &c) { c.layers = 0xffffffffu, c.pages = 1u << 28, c.page_size = 8; });
    cache(QWH_E_LIMIT_EXCEEDED, "64 GiB", [](auto &c) { c.pages = 1u << 22, c.page_size = 16; });
    cache(QWH_OK, "below 64 GiB", [](auto &c) { c.pages = (1u << 22) - 1, c.page_size = 16; });
    cache(QWH_E_INVALID_ARGUMENT, "null scales", [](auto &c) { c.k_scales = nullptr; });
    cache(QWH_E_INVALID_ARGUMENT, "null codes", [](auto &c) { c.v_codes = nullptr; });
    cache(QWH_E_INVALID_ARGUMENT, "codes' alignment", [](auto &c) { c.k_codes += 8; });
    cache(QWH_E_INVALID_ARGUMENT, "scales' alignment", [](auto &c) { c.v_scales += 2; });
    cache(QWH_OK, "scales on 4 bytes", [](auto &c) { c.v_scales += 4; });
    expect(paged::check_layer(good, 27).status == QWH_OK, "last layer");
    expect(paged::check_layer(good, 28).status == QWH_E_INVALID_ARGUMENT, "layer past the pool");

    const qwh_paged_batch rows{4, 10, 3, words, words, words};
    expect(paged::check_batch(nullptr).status == QWH_E_INVALID_ARGUMENT, "no batch");
    const auto batch = [&](int32_t status, const char *what, const std::function<void(qwh_paged_batch &)> &change) {
        qwh_paged_batch b = rows;
        change(b);
        expect(paged::check_batch(&b).status == status, what);
    };
    batch(QWH_OK, "ragged rows", [](auto &) {});
    batch(QWH_OK, "one row each", [](auto &b) { b.row_starts = nullptr, b.rows = 4; });
    batch(QWH_OK, "no sequence", [](auto &b) { b = qwh_paged_batch{}; });
    batch(QWH_OK, "no row", [](auto &b) { b.rows = 0, b.first = nullptr; });
    batch(QWH_E_SHAPE_MISMATCH, "three rows for four", [](auto &b) { b.row_starts = nullptr, b.rows = 3; });
    batch(QWH_E_SHAPE_MISMATCH, "empty tables", [](auto &b) { b.table_pages = 0; });
    batch(QWH_E_INVALID_ARGUMENT, "null first", [](auto &b) { b.first = nullptr; });
    batch(QWH_E_INVALID_ARGUMENT, "null tables", [](auto &b) { b.tables = nullptr; });
    const auto off = [](const uint32_t *p) { return reinterpret_cast<const uint32_t *>(reinterpret_cast<uintptr_t>(p) + 2); };
    batch(QWH_E_INVALID_ARGUMENT, "starts' alignment", [&](auto &b) { b.row_starts = off(b.row_starts); });
    batch(QWH_E_INVALID_ARGUMENT, "first's alignment", [&](auto &b) { b.first = off(b.first); });
    batch(QWH_E_INVALID_ARGUMENT, "tables' alignment", [&](auto &b) { b.tables = off(b.tables); });
    batch(QWH_OK, "no row, whatever its arrays", [&](auto &b) { b.rows = 0, b.first = off(b.first); });
    const float *good_floats = reinterpret_cast<const float *>(plane), *bad_floats = reinterpret_cast<const float *>(plane + 2);
    expect(paged::check_floats(good_floats, good_floats + 1, good_floats + 2, good_floats + 3).status == QWH_OK, "norms and tables");
    for (int which = 0; which < 4; ++which)
        for (const float *p : {bad_floats, (const float *)nullptr})
            expect(paged::check_floats(which == 0 ? p : good_floats, which == 1 ? p : good_floats, which == 2 ? p : good_floats,
                                       which == 3 ? p : good_floats).status == QWH_E_INVALID_ARGUMENT, "a norm or table", which);
    batch(QWH_E_LIMIT_EXCEEDED, "sequences", [](auto &b) { b.batch = 65536; });
    batch(QWH_E_LIMIT_EXCEEDED, "rows", [](auto &b) { b.rows = (1u << 20) + 1; });

    qwh_paged_batch tall = rows;
    tall.table_pages = 0xfffefff;
    expect(paged::check_positions(good, tall).status == QWH_OK, "positions below the limit");
    ++tall.table_pages;
    expect(paged::check_positions(good, tall).status == QWH_E_LIMIT_EXCEEDED, "positions");
    expect(paged::check_row_heads(rows, 4096).status == QWH_OK, "rows times heads");
    tall.rows = 1u << 20;
    expect(paged::check_row_heads(tall, 8).status == QWH_OK, "2^23 rows times heads");
    expect(paged::check_row_heads(tall, 9).status == QWH_E_LIMIT_EXCEEDED, "past 2^23 rows times heads");
    expect(paged::check_heads(good, 16).status == QWH_OK, "16 over 8");
    expect(paged::check_heads(good, 24).status == QWH_OK, "24 over 8");
    expect(paged::check_heads(good, 0).status == QWH_E_SHAPE_MISMATCH, "no query head");
    expect(paged::check_heads(good, 12).status == QWH_E_SHAPE_MISMATCH, "12 over 8");
    expect(paged::check_heads(good, 4104).status == QWH_E_LIMIT_EXCEEDED, "4104 heads");
    // 2^15 rows of 8 heads in one sequence: 32769 tiles of 8 query rows, and
    // 259 units beside the tables'. 32769 * 65534 is 2^31 - 2.
    qwh_paged_cache wide = good;
    wide.page_size = 128;
    qwh_paged_batch units{1, 1u << 15, 65534 - 259, words, words, words};
    expect(paged::check_units(wide, units, 64).status == QWH_OK, "2^31 - 2 units");
    ++units.table_pages;
    expect(paged::check_units(wide, units, 64).status == QWH_E_LIMIT_EXCEEDED, "more units");
    // A tile more for each sequence, as many as there are rows.
    units = qwh_paged_batch{65535, 1u << 15, (uint32_t)(0x7ffffffeu / (2u << 15)) - 259, words, words, words};
    expect(paged::check_units(wide, units, 64).status == QWH_OK, "units of short sequences");
    ++units.table_pages;
    expect(paged::check_units(wide, units, 64).status == QWH_E_LIMIT_EXCEEDED, "more units of short sequences");
    const qwh_paged_cache narrow{1, 1, 1, 1, 64, plane, plane, plane, plane};
    expect(paged::check_heads(narrow, 256).status == QWH_OK, "256 over 1");
    expect(paged::check_heads(narrow, 257).status == QWH_E_LIMIT_EXCEEDED, "257 over 1");
    expect(paged::check_rows(plane, 2048, 2048, "", "").status == QWH_OK, "rows");
    expect(paged::check_rows(plane, 2050, 2048, "", "").status == QWH_E_INVALID_ARGUMENT, "an odd stride");
    expect(paged::check_rows(plane + 4, 2048, 2048, "", "").status == QWH_E_INVALID_ARGUMENT, "rows' alignment");
    expect(paged::check_rows(plane, 2044, 2048, "", "").status == QWH_E_SHAPE_MISMATCH, "a short stride");
    expect(paged::check_rows(nullptr, 2048, 2048, "", "").status == QWH_E_INVALID_ARGUMENT, "null rows");
}

// Every sequence that a call may hold takes a form that the call runs: the
// other form's records are not reserved.
void check_forms() {
    static uint32_t words[4];
    for (uint32_t ratio : {1u, 2u, 3u, 8u, 31u, 32u, 33u, 64u, 128u, 256u})
        for (uint32_t rows : {1u, 2u, 4u, 31u, 33u, 100u, 129u, 5000u, 1u << 15})
            for (uint32_t batch : {1u, 2u, 40u, 5000u})
                for (uint64_t positions : {1ull, 16ull, 130ull, 1024ull, 8192ull, 70000ull, 0xfffeffffull})
                    for (bool ragged : {false, true}) {
                        const qwh_paged_batch b{batch, ragged ? rows : batch, 1, ragged ? words : nullptr, words, words};
                        const paged::Forms forms = paged::forms_of(b, ratio, positions);
                        expect(forms.few || forms.many, "no form", ratio, rows);
                        const uint32_t border = paged::few_rows(forms);
                        // (Words that an earlier call, or nothing, left.)
                        for (uint32_t word : {0u, 1u, 2u, 0xffffffffu})
                            expect(paged::joins_many(word, border) ? forms.many : forms.few, "records that are not there", word, ratio);
                        for (uint32_t n = 1; n <= (ragged ? b.rows : 1); n += 1 + n / 5) {
                            const bool many = paged::takes_many(n * ratio, border);
                            expect(many ? forms.many : forms.few, "a form that does not run", n * ratio, ragged);
                            expect(paged::joins_many(many, border) == many, "records of the other form", n * ratio, ragged);
                            expect(!forms.few || !forms.many || many == (n * ratio > paged::kFewRows), "the border of two forms", n * ratio);
                        }
                    }
}

}  // namespace

int main() {
    check_refusals();
    check_forms();
    check_copies();
    std::printf("paged: %ld cases, %ld failures\n", cases, failures);
    return failures ? 1 : 0;
}
