// Host arithmetic of the paged cache's entry points (no device code): what a
// pool and a batch have to satisfy, and the order in which a set of page
// copies runs. paged.cpp calls it; sanitize/plan_check.cpp checks it on the CPU.
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

inline Refusal check_rows(const void *p, uint32_t stride, uint64_t width, const char *what_null, const char *what) {
    if (!p) return refuse(QWH_E_INVALID_ARGUMENT, what_null);
    if (stride < width) return refuse(QWH_E_SHAPE_MISMATCH, what);
    if (!aligned(p, 16) || stride % 4 != 0)
        return refuse(QWH_E_INVALID_ARGUMENT, "rows must be 16-byte aligned, strides a multiple of 4 floats");
    return {};
}

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
// nothing that has to outlive the call): at most kMaxSteps, chains starting
// at chain[0 .. chains - 1], chain[chains] their end.
constexpr uint32_t kMaxSteps = 384;
struct CopySteps {
    uint32_t chains;
    uint16_t chain[kMaxSteps + 1];
    uint32_t src[kMaxSteps], dst[kMaxSteps];
};

// The pairs over the pages that they name: page[] in ascending order, and for
// each of them the place in page[] of its source (kSaved: not a destination).
struct CopyPairs {
    std::vector<uint32_t> page, source, order;  // order: the destinations' places, as given
};

inline Refusal check_copies(const uint32_t *src, const uint32_t *dst, uint32_t count, uint32_t pages, CopyPairs &out) {
    out.page.clear();
    for (uint32_t i = 0; i < count; ++i) {
        if (src[i] >= pages || dst[i] >= pages) return refuse(QWH_E_INVALID_ARGUMENT, "a page is not one of the pool's");
        out.page.push_back(src[i]);
        out.page.push_back(dst[i]);
    }
    std::sort(out.page.begin(), out.page.end());
    out.page.erase(std::unique(out.page.begin(), out.page.end()), out.page.end());
    const auto place = [&](uint32_t p) {
        return (uint32_t)(std::lower_bound(out.page.begin(), out.page.end(), p) - out.page.begin());
    };
    out.source.assign(out.page.size(), kSaved);
    out.order.clear();
    for (uint32_t i = 0; i < count; ++i) {
        const uint32_t d = place(dst[i]);
        if (out.source[d] != kSaved) return refuse(QWH_E_INVALID_ARGUMENT, "a page is named as destination twice");
        out.source[d] = place(src[i]);
        out.order.push_back(d);
    }
    return {};
}

// Appends steps to launches of at most kMaxSteps.
class CopyLaunches {
  public:
    std::vector<CopySteps> launches;

    // Starts a new chain.
    void chain() { fresh_ = true; }
    // One step of the current chain; `keep`: steps from here on that have to
    // be in one launch (this one first).
    void step(uint32_t src, uint32_t dst, uint32_t keep = 1) {
        if (launches.empty() || used_ + keep > kMaxSteps) {
            launches.emplace_back();
            launches.back().chains = 0;
            launches.back().chain[0] = 0;
            used_ = 0;
            fresh_ = true;
        }
        CopySteps &l = launches.back();
        if (fresh_) {
            ++l.chains;
            fresh_ = false;
        }
        l.src[used_] = src;
        l.dst[used_] = dst;
        l.chain[l.chains] = (uint16_t)++used_;
    }

  private:
    uint32_t used_ = 0;
    bool fresh_ = true;
};

// The pairs' steps, a chain for each set of pages that copies connect.
inline void order_copies(const CopyPairs &pairs, CopyLaunches &out) {
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
