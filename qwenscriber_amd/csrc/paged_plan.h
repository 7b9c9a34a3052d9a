// Host arithmetic of the paged cache's entry points (no device code): what a
// pool and a batch have to satisfy, which kernels of the attention a call
// needs, and the order in which a set of page copies runs. paged.cpp calls it; sanitize/paged_check.cpp checks it on the CPU.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <vector>

#include "../../include/qwhip.h"

namespace qwh {
namespace paged {

constexpr uint32_t kMaxBatch = 65535;
constexpr uint32_t kMaxRows = 1u << 20;
constexpr uint32_t kMaxHeads = 4096;
constexpr uint64_t kMaxRowHeads = 1u << 23;
constexpr uint32_t kMaxRatio = 256;

// A refusal: a status and why, or QWH_OK.
struct Refusal {
    int32_t status = QWH_OK;
    const char *why = "";
};

inline Refusal refuse(int32_t status, const char *why) { return Refusal{status, why}; }

inline bool aligned(const void *p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

inline Refusal check_cache(const qwh_paged_cache *c) {
    if (!c) return refuse(QWH_E_INVALID_ARGUMENT, "cache is null");
    if (!c->layers || !c->pages || !c->page_size || !c->kv_heads)
        return refuse(QWH_E_SHAPE_MISMATCH, "a pool needs layers, pages, page_size and kv_heads of at least 1");
    if (c->head_dim == 0 || c->head_dim % 64 != 0)
        return refuse(QWH_E_SHAPE_MISMATCH, "head_dim is not a multiple of 64");
    if (c->head_dim > 256) return refuse(QWH_E_UNSUPPORTED, "head_dim of more than 256 is not built");
    if (c->kv_heads > kMaxHeads) return refuse(QWH_E_LIMIT_EXCEEDED, "more than 4096 kv_heads");
    // A pool row's index fits 32 bits, with a value left for "no row"; and a
    // plane's bytes fit 63.
    if ((uint64_t)c->pages * c->page_size >= 0xffffffffull)
        return refuse(QWH_E_LIMIT_EXCEEDED, "pages * page_size of 2^32 - 1 or more");
    if ((unsigned __int128)c->pages * c->page_size * c->layers * c->kv_heads * c->head_dim >> 62)
        return refuse(QWH_E_LIMIT_EXCEEDED, "the pool's planes pass 2^62 bytes");
    if ((uint64_t)c->pages * c->page_size * c->kv_heads * (c->head_dim / 16) >> 32)
        return refuse(QWH_E_LIMIT_EXCEEDED, "a layer's code plane of 64 GiB or more");
    if (!c->k_scales || !c->k_codes || !c->v_scales || !c->v_codes)
        return refuse(QWH_E_INVALID_ARGUMENT, "a pool plane is null");
    if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16))
        return refuse(QWH_E_INVALID_ARGUMENT, "code planes must be 16-byte aligned");
    if (!aligned(c->k_scales, 4) || !aligned(c->v_scales, 4))
        return refuse(QWH_E_INVALID_ARGUMENT, "scale planes must be 4-byte aligned");
    return {};
}

// (A copy counts a page's pieces, of 16 bytes or of 2, in 32 bits.)
inline Refusal check_page(const qwh_paged_cache &c) {
    if ((uint64_t)c.page_size * c.kv_heads * c.head_dim > 8ull << 30)
        return refuse(QWH_E_LIMIT_EXCEEDED, "a page of more than 8 GiB of codes a layer");
    return {};
}

inline Refusal check_layer(const qwh_paged_cache &c, uint32_t layer) {
    if (layer >= c.layers) return refuse(QWH_E_INVALID_ARGUMENT, "layer is not one of the pool's");
    return {};
}

inline Refusal check_batch(const qwh_paged_batch *b) {
    if (!b) return refuse(QWH_E_INVALID_ARGUMENT, "batch is null");
    if (b->batch > kMaxBatch) return refuse(QWH_E_LIMIT_EXCEEDED, "more than 65535 sequences");
    if (b->rows > kMaxRows) return refuse(QWH_E_LIMIT_EXCEEDED, "more than 2^20 rows");
    if (b->batch == 0 || (b->row_starts && b->rows == 0)) return {};  // nothing to do
    if (!b->row_starts && b->rows < b->batch)
        return refuse(QWH_E_SHAPE_MISMATCH, "fewer rows than sequences of one row each");
    if (b->table_pages == 0) return refuse(QWH_E_SHAPE_MISMATCH, "page tables of no entry");
    if (!b->first || !b->tables) return refuse(QWH_E_INVALID_ARGUMENT, "first or tables is null");
    if (!aligned(b->row_starts, 4) || !aligned(b->first, 4) || !aligned(b->tables, 4))
        return refuse(QWH_E_INVALID_ARGUMENT, "row_starts, first and tables must be 4-byte aligned");
    return {};
}

// Positions are 32-bit counts, with room to step past the last one.
inline Refusal check_positions(const qwh_paged_cache &c, const qwh_paged_batch &b) {
    if ((uint64_t)b.table_pages * c.page_size >= 0xffff0000ull)
        return refuse(QWH_E_LIMIT_EXCEEDED, "page tables of 2^32 - 2^16 positions or more");
    return {};
}

inline bool nothing_to_do(const qwh_paged_batch &b) { return b.batch == 0 || (b.row_starts && b.rows == 0); }

inline Refusal check_heads(const qwh_paged_cache &c, uint32_t heads) {
    if (heads == 0 || heads % c.kv_heads != 0)
        return refuse(QWH_E_SHAPE_MISMATCH, "heads is not a multiple of kv_heads");
    if (heads > kMaxHeads) return refuse(QWH_E_LIMIT_EXCEEDED, "more than 4096 heads");
    if (heads / c.kv_heads > kMaxRatio) return refuse(QWH_E_LIMIT_EXCEEDED, "more than 256 heads per kv head");
    return {};
}

// (The grids' 32 bits.)
inline Refusal check_row_heads(const qwh_paged_batch &b, uint32_t heads) {
    if ((uint64_t)b.rows * heads > kMaxRowHeads) return refuse(QWH_E_LIMIT_EXCEEDED, "rows * heads of more than 2^23");
    return {};
}

// The attention counts units of 8 query rows (of a kv head) by 128 positions
// in 31 bits: rows in whole tiles, and one tile more a sequence; positions up
// to the tables' last, rounded up, and a token's own tile.
inline Refusal check_units(const qwh_paged_cache &c, const qwh_paged_batch &b, uint32_t heads) {
    const uint64_t tiles = (uint64_t)b.rows * (heads / c.kv_heads) / 8 + (b.batch < b.rows ? b.batch : b.rows);
    const uint64_t units = ((uint64_t)b.table_pages * c.page_size + 127) / 128 + b.rows / 128 + 3;
    if (tiles * units >= 0x7fffffffull)
        return refuse(QWH_E_LIMIT_EXCEEDED, "rows times heads per kv head times positions past 2^41");
    return {};
}

// The append's vectors and tables.
inline Refusal check_floats(const float *q_norm, const float *k_norm, const float *rope_cos, const float *rope_sin) {
    for (const float *p : {q_norm, k_norm, rope_cos, rope_sin}) {
        if (!p) return refuse(QWH_E_INVALID_ARGUMENT, "a norm or rotation table is null");
        if (!aligned(p, 4)) return refuse(QWH_E_INVALID_ARGUMENT, "norms and rotation tables must be 4-byte aligned");
    }
    return {};
}

inline Refusal check_rows(const void *p, uint32_t stride, uint64_t width, const char *what_null, const char *what) {
    if (!p) return refuse(QWH_E_INVALID_ARGUMENT, what_null);
    if (stride < width) return refuse(QWH_E_SHAPE_MISMATCH, what);
    if (!aligned(p, 16) || stride % 4 != 0)
        return refuse(QWH_E_INVALID_ARGUMENT, "rows must be 16-byte aligned, strides a multiple of 4 floats");
    return {};
}

// ---- the attention's forms ----
//
// Sequences of more query rows a key/value head take paged_many_kernel, which
// converts a code once for 128 rows instead of once for 8 (us, 8 key/value
// heads of 128, 16 sequences of 2000 positions, few / many: 16 rows 37 / 61,
// 32 rows 60 / 62, 64 rows 107 / 76). But its first answer comes 20 us after
// its start against 6, so calls of little work in all take paged_few_kernel
// alone: query rows of a key/value head times positions of the tables up to
// kLittle (one sequence of 512 rows from position 0 on: 13 / 23; 4 of 256: 18
// / 23; 8 of 256, twice the bound: 32 / 26), and up to kLittleNarrow of up to
// 128 rows, which are one tile of paged_many_kernel (128 rows at 4000: 29 /
// 41; at 16000, twice the bound: 84 / 68).
constexpr uint32_t kFewRows = 32;
constexpr uint64_t kLittle = 1 << 18, kLittleNarrow = 1 << 20;

// The kernels that a call needs (at least one): by the most query rows that a
// sequence may have (one sequence: as if it had all rows of the buffer).
struct Forms {
    bool few, many;
};

inline Forms forms_of(const qwh_paged_batch &b, uint64_t ratio, uint64_t positions) {
    const uint64_t rows = ratio * (b.row_starts ? b.rows : b.batch), work = rows * positions;
    if (rows <= kFewRows || work <= kLittle || (rows <= 128 && work <= kLittleNarrow)) return Forms{true, false};
    if (!b.row_starts) return Forms{ratio <= kFewRows, ratio > kFewRows};
    return Forms{b.batch > 1, true};
}

// Whether a sequence of `rows` query rows a key/value head takes the form for
// many rows, in a call whose forms have the border few_rows; and whether its
// records are of that form, by the word that the form left in the sequence's
// plan (1: many) or, where it left none, any word. Neither is ever a form that
// the call does not run: that has no records.
constexpr uint32_t few_rows(const Forms &f) { return !f.many ? 0xffffffffu : !f.few ? 0 : kFewRows; }
constexpr bool takes_many(uint32_t rows, uint32_t border) { return rows > border; }
constexpr bool joins_many(uint32_t word, uint32_t border) { return border == 0 || (border != 0xffffffffu && word == 1); }

// ---- page copies ----
//
// The pairs are a function from destinations to sources, all sources read
// before any destination is written. Every pair becomes a step (src, dst) of
// a chain; the steps of a chain run one after another on each piece of a page
// (one thread holds a piece from first to last), different chains touch no
// common destination and run side by side. A page is overwritten only after
// the last step that reads it: trees run from their leaves, and a cycle saves
// its last page first (kSaved as destination) and hands it on last (kSaved as
// source). Steps of one source stand together: it is read once.
constexpr uint32_t kSaved = 0xffffffffu;

// Steps of one launch, handed over in the kernel's arguments (no upload, and
// nothing that has to outlive the call). In the short form, for pools of up to
// kShortPages pages, a step is a word (its source below, its destination
// above), and the chains' starts stand behind the steps, two a word, unless
// every chain is one step.
constexpr uint32_t kMaxSteps = 384;
struct CopySteps {
    uint32_t chains;
    uint16_t chain[kMaxSteps + 1];
    uint32_t src[kMaxSteps], dst[kMaxSteps];

    constexpr uint32_t begin(uint32_t c) const { return chain[c]; }
    constexpr uint32_t end(uint32_t c) const { return chain[c + 1]; }
    constexpr uint32_t source(uint32_t i) const { return src[i]; }
    constexpr uint32_t target(uint32_t i) const { return dst[i]; }
};

constexpr uint32_t kShortPages = 0xffff, kShortWords = 990;
struct CopyStepsShort {
    uint32_t chains, steps;
    uint32_t words[kShortWords];

    constexpr uint32_t at(uint32_t c) const { return chains == steps ? c : words[steps + c / 2] >> (c % 2 * 16) & 0xffff; }
    constexpr uint32_t begin(uint32_t c) const { return at(c); }
    constexpr uint32_t end(uint32_t c) const { return at(c + 1); }
    constexpr uint32_t page(uint32_t p) const { return p == kShortPages ? kSaved : p; }
    constexpr uint32_t source(uint32_t i) const { return page(words[i] & 0xffff); }
    constexpr uint32_t target(uint32_t i) const { return page(words[i] >> 16); }
};

// The pairs, and over the pages that they name: page[] in ascending order,
// and for each of them the place in page[] of its source (kSaved: not a
// destination). `apart`: no page is both (but for pages onto themselves), so
// that any order does; the rest is then left out.
struct CopyPairs {
    const uint32_t *src, *dst;
    uint32_t count;
    bool apart;
    std::vector<uint32_t> page, source, order;  // order: the destinations' places, as given
};

inline Refusal check_copies(const uint32_t *src, const uint32_t *dst, uint32_t count, uint32_t pages, CopyPairs &out) {
    out.src = src;
    out.dst = dst;
    out.count = count;
    out.apart = false;
    out.page.clear();
    out.order.clear();
    for (uint32_t i = 0; i < count; ++i)
        if (src[i] >= pages || dst[i] >= pages) return refuse(QWH_E_INVALID_ARGUMENT, "a page is not one of the pool's");
    const char *twice = "a page is named as destination twice";
    // A bit a page, where the pool is not far larger than the call: the
    // ordering below costs the host about 0.1 us a pair.
    if (pages <= (1u << 20) + 256ull * count) {
        std::vector<uint64_t> written((pages + 63ull) / 64);
        for (uint32_t i = 0; i < count; ++i) {
            uint64_t &word = written[dst[i] / 64];
            const uint64_t bit = 1ull << dst[i] % 64;
            if (word & bit) return refuse(QWH_E_INVALID_ARGUMENT, twice);
            word |= bit;
        }
        out.apart = true;
        for (uint32_t i = 0; i < count && out.apart; ++i) out.apart = src[i] == dst[i] || !(written[src[i] / 64] >> src[i] % 64 & 1);
        if (out.apart) return {};
    }
    const bool all = pages <= 1024 + 4ull * count;  // every page has its own number as its place
    if (all) {
        out.page.resize(pages);
        for (uint32_t p = 0; p < pages; ++p) out.page[p] = p;
    } else {
        out.page.insert(out.page.end(), src, src + count);
        out.page.insert(out.page.end(), dst, dst + count);
        std::sort(out.page.begin(), out.page.end());
        out.page.erase(std::unique(out.page.begin(), out.page.end()), out.page.end());
    }
    const auto place = [&](uint32_t p) {
        return all ? p : (uint32_t)(std::lower_bound(out.page.begin(), out.page.end(), p) - out.page.begin());
    };
    out.source.assign(out.page.size(), kSaved);
    for (uint32_t i = 0; i < count; ++i) {
        const uint32_t d = place(dst[i]);
        if (out.source[d] != kSaved) return refuse(QWH_E_INVALID_ARGUMENT, twice);
        out.source[d] = place(src[i]);
        out.order.push_back(d);
    }
    return {};
}

// Steps in launches that hold as many as their form takes.
struct CopyLaunch {
    std::vector<uint32_t> chain{0}, src, dst;

    uint32_t chains() const { return (uint32_t)chain.size() - 1; }
    uint32_t steps() const { return (uint32_t)src.size(); }
};

class CopyLaunches {
  public:
    explicit CopyLaunches(bool is_short) : is_short(is_short) {}
    const bool is_short;
    std::vector<CopyLaunch> launches;

    // Starts a new chain.
    void chain() { fresh_ = true; }
    // One step of the current chain; `keep`: steps from here on that have to
    // be in one launch (this one first).
    void step(uint32_t src, uint32_t dst, uint32_t keep = 1) {
        if (launches.empty() || !fits(launches.back(), keep)) {
            launches.emplace_back();
            launches.back().src.reserve(kShortWords);
            launches.back().dst.reserve(kShortWords);
            launches.back().chain.reserve(kShortWords + 1);
            fresh_ = true;
        }
        CopyLaunch &l = launches.back();
        if (fresh_) l.chain.push_back(l.steps());
        fresh_ = false;
        l.src.push_back(src);
        l.dst.push_back(dst);
        l.chain.back() = l.steps();
    }

  private:
    bool fits(const CopyLaunch &l, uint32_t more) const {
        const uint32_t steps = l.steps() + more, chains = l.chains() + (fresh_ ? 1 : 0);
        if (!is_short) return steps <= kMaxSteps;
        return steps + (chains == steps ? 0 : (chains + 2) / 2) <= kShortWords;
    }
    bool fresh_ = true;
};

inline CopySteps pack(const CopyLaunch &l) {
    CopySteps s{};
    s.chains = l.chains();
    for (uint32_t c = 0; c <= s.chains; ++c) s.chain[c] = (uint16_t)l.chain[c];
    std::copy(l.src.begin(), l.src.end(), s.src);
    std::copy(l.dst.begin(), l.dst.end(), s.dst);
    return s;
}

inline CopyStepsShort pack_short(const CopyLaunch &l) {
    CopyStepsShort s{};
    s.chains = l.chains();
    s.steps = l.steps();
    const auto half = [](uint32_t p) { return p == kSaved ? kShortPages : p; };
    for (uint32_t i = 0; i < s.steps; ++i) s.words[i] = half(l.src[i]) | half(l.dst[i]) << 16;
    if (s.chains != s.steps)
        for (uint32_t c = 0; c <= s.chains; ++c) s.words[s.steps + c / 2] |= l.chain[c] << (c % 2 * 16);
    return s;
}

// The pairs' steps, a chain for each set of pages that copies connect.
inline void order_copies(const CopyPairs &pairs, CopyLaunches &out) {
    if (pairs.apart) {
        for (uint32_t i = 0; i < pairs.count; ++i) {
            if (pairs.src[i] == pairs.dst[i]) continue;
            if (i == 0 || pairs.src[i] != pairs.src[i - 1]) out.chain();
            out.step(pairs.src[i], pairs.dst[i]);
        }
        return;
    }
    const std::vector<uint32_t> &source = pairs.source;
    const uint32_t n_pages = (uint32_t)source.size();
    const auto is_copied = [&](uint32_t p) { return source[p] != kSaved && source[p] != p; };
    const auto emit = [&](uint32_t from, uint32_t to, uint32_t keep) {
        out.step(from == kSaved ? kSaved : pairs.page[from], to == kSaved ? kSaved : pairs.page[to], keep);
    };
    // The destinations of each source, as lists.
    std::vector<uint32_t> head(n_pages, kSaved), next(n_pages, kSaved), walked(n_pages, 0);
    for (size_t i = pairs.order.size(); i-- > 0;) {
        const uint32_t d = pairs.order[i], s = source[d];
        if (s == d) continue;  // a page onto itself
        next[d] = head[s];
        head[s] = d;
    }
    std::vector<uint8_t> done(n_pages, 0);
    std::vector<uint32_t> stack, cycle;
    for (size_t i = 0; i < pairs.order.size(); ++i) {
        uint32_t top = pairs.order[i];
        if (!is_copied(top) || done[top]) continue;
        // Up to the page that is no destination, or once around into the cycle.
        const uint32_t walk = (uint32_t)i + 1;
        while (is_copied(top) && walked[top] != walk) {
            walked[top] = walk;
            top = source[top];
        }
        const bool cyclic = is_copied(top);
        out.chain();
        stack.assign(1, top);
        cycle.clear();
        if (cyclic) {
            uint32_t p = top;  // (cycle[k + 1] is the source of cycle[k].)
            do {
                cycle.push_back(p);
                done[p] = 1;
                p = source[p];
            } while (p != top);
            stack = cycle;
        }
        // Depth order from the roots; the reverse of it has every page after
        // all pages that read it.
        for (size_t at = 0; at < stack.size(); ++at)
            for (uint32_t c = head[stack[at]]; c != kSaved; c = next[c])
                if (!done[c]) {
                    done[c] = 1;
                    stack.push_back(c);
                }
        for (size_t at = stack.size(); at-- > (cyclic ? cycle.size() : 1);) emit(source[stack[at]], stack[at], 1);
        if (!cyclic) continue;
        // The cycle, in pieces that fit a launch: content moves from
        // cycle[k + 1] to cycle[k]. A cycle (c0 <- c1 <- ... <- cn <- c0)
        // longer than a launch moves its tail first and goes on with the rest,
        // what is still on its way waiting in c0.
        const uint32_t most = kMaxSteps - 1;  // pages of one piece
        const size_t n = cycle.size();
        size_t end = n;  // cycle[1 .. end - 1] are still to be moved, through cycle[0]
        while (end > 1) {
            const size_t take = end - 1 < most - 1 ? end - 1 : most - 1;  // pages besides cycle[0]
            const size_t begin = end - take;
            const uint32_t length = (uint32_t)take + 2;
            const uint32_t c0 = cycle[0];
            if (begin == 1) {
                // c0 <- c1 <- ... <- c(end-1) <- c0
                emit(c0, kSaved, length);
                for (size_t k = 1; k < end; ++k) emit(cycle[k], cycle[k - 1], 1);
                emit(kSaved, cycle[end - 1], 1);
            } else {
                // c(begin) <- ... <- c(end-1) <- c0, and c0 <- c(begin): what
                // c(begin - 1) is to get waits in c0.
                emit(c0, kSaved, length);
                emit(cycle[begin], c0, 1);
                for (size_t k = begin + 1; k < end; ++k) emit(cycle[k], cycle[k - 1], 1);
                emit(kSaved, cycle[end - 1], 1);
            }
            end = begin;
        }
    }
}

}  // namespace paged
}  // namespace qwh
