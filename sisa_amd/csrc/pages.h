// Pages of a generation cache (include/sisa_hip_cache.h): where a position lives, and the host's checks of a pool.
#pragma once
#include "common.h"
#include "host.h"
#include "sisa_hip_cache.h"

// The page of position pos of a sequence, or -1 where the table has none of the pool's there. W, pages > 0.
SISA_DEV int page_of(const int32_t* row, int W, int shift, int pages, int64_t pos) {
    const int64_t w = pos >> shift;
    if (pos < 0 || w >= W) return -1;
    const int p = row[w];
    return p >= 0 && p < pages ? p : -1;
}

namespace sisa {

inline int log2_of(int32_t page_size) { return 31 - __builtin_clz((unsigned)page_size); }

// Null where the pool can be used, else what is wrong with it.
inline const char* pool_fault(const sisa_page_pool& p) {
    if (p.pages < 1 || p.heads < 1) return "a pool needs pages and heads";
    if (p.page_size < SISA_MIN_PAGE_SIZE || (p.page_size & (p.page_size - 1)))
        return "the page size must be a power of two of at least 16";
    if (p.dtype != SISA_BF16 && p.dtype != SISA_F16 && p.dtype != SISA_F32) return "the pool's dtype";
    if (!view_ok(p.k, p.dtype) || !view_ok(p.v, p.dtype) || !view_ok(p.b, p.dtype))
        return "the pool's k, v and b rows must be 16-byte aligned";
    if (!p.g.ptr) return "the pool has no g";
    return nullptr;
}

}  // namespace sisa

#define SISA_REQUIRE_POOL(name, pool)                                       \
    do {                                                                    \
        const char* fault_ = ::sisa::pool_fault(pool);                      \
        SISA_REQUIRE(fault_ == nullptr, "%s: %s", name, fault_);            \
    } while (0)
