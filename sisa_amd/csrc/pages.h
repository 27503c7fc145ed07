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

// 256 MB, the last-level cache: what is larger cannot be found there again and is loaded with the non-temporal hint.
constexpr int64_t STREAM_BYTES = (int64_t)256 << 20;
template <class V, bool HINT> SISA_DEV V load_hint(const void* p) {
    if constexpr (HINT) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
    else return *reinterpret_cast<const V*>(p);
}
template <class V, bool HINT> SISA_DEV void store_hint(void* p, V x) {
    if constexpr (HINT) __builtin_nontemporal_store(x, reinterpret_cast<V*>(p));
    else *reinterpret_cast<V*>(p) = x;
}

struct RowViews {
    sisa_view k, v, b, g, f;
};

SISA_DEV int64_t lane_value(int64_t x, int lane) {
    const int lo = __shfl((int)x, lane), hi = __shfl((int)(x >> 32), lane);
    return (int64_t)hi << 32 | (unsigned)lo;
}

// Up to ROWS rows of a cache moved by a wave: lane r's row, if `ok`, from (s0, h, s2) of the source views to (d0, h, d2) of the
// destination's; no lane from ROWS on has one. 64, or 8 where there are too few rows to fill the chip with waves of 64.
//
// Every load and store instruction covers whole rows (k and v of 16 bits: 8 rows of 128 bytes, 8 lanes a row), and all of a
// pass's loads are under way before its first store: 32 rows a pass in 16 bits, 16 in fp32 (40 registers either way). A row
// per half wave instead, with three dependent loads in front of each, left the chip waiting: an eviction of 8 x 12 heads from
// 16,384 to 4,096 positions took 147 us for its copies.
//
// Many rows (ROWS = 64) are stored with the non-temporal hint: nothing reads them before the launch ends. Out of a cache larger
// than the last-level cache those of k and v are loaded with it, too (STREAM; b rows share their lines: with the hint 59.7 us
// in place of 54.1). Copies of evictions, plain / stores / both: 92 MB out of caches of 130 MB 21.4 / 17.7 / 21.4 us, 258 MB out
// of 516 MB 64.1 / 62.1 / 54.1 (4.8 TB/s).
template <class T, int ROWS, bool STREAM>
SISA_DEV void move_rows(const RowViews& src, const RowViews& dst, bool ok, int64_t s0, int64_t d0, int64_t h, int64_t s2,
                        int64_t d2, int lane) {
    constexpr int E = 16 / (int)sizeof(T);             // elements of a piece
    constexpr int KP = 64 / E, BP = 32 / E;            // pieces of a k or v row, of a b row
    constexpr int MOST = sizeof(T) == 2 ? 32 : 16, PASS = ROWS < MOST ? ROWS : MOST;      // rows of a pass
    constexpr int NK = PASS * KP / 64, NB = (PASS * BP + 63) / 64;
    static_assert(PASS * KP % 64 == 0, "whole instructions");
    const uint64_t rows = __ballot(ok);
    auto at = [&](const sisa_view& x, int64_t i0, int64_t i2) { return i0 * x.sb + h * x.sh + i2 * x.sl; };
    const int64_t sk = at(src.k, s0, s2), sv = at(src.v, s0, s2), sb = at(src.b, s0, s2);
    const int64_t dk = at(dst.k, d0, d2), dv = at(dst.v, d0, d2), db = at(dst.b, d0, d2);
    float g = 0.f, f = 0.f;
    if (ok) {
        g = ((const float*)src.g.ptr)[at(src.g, s0, s2)];
        if (src.f.ptr) f = ((const float*)src.f.ptr)[at(src.f, s0, s2)];
    }
#pragma unroll 1
    for (int r0 = 0; r0 < ROWS; r0 += PASS) {
        u32x4 xk[NK], xv[NK], xb[NB];
        const int pk = lane % KP, rk = r0 + lane / KP, pb = lane % BP, rb = r0 + lane / BP;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int r = rk + i * (64 / KP);
            const int64_t ok_ = lane_value(sk, r), ov = lane_value(sv, r);
            if (rows >> r & 1) {
                xk[i] = load_hint<u32x4, STREAM>((const T*)src.k.ptr + ok_ + E * pk);
                xv[i] = load_hint<u32x4, STREAM>((const T*)src.v.ptr + ov + E * pk);
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int r = rb + i * (64 / BP);
            const int64_t o = lane_value(sb, r);
            if (rows >> r & 1) xb[i] = load_hint<u32x4, false>((const T*)src.b.ptr + o + E * pb);
        }
        __builtin_amdgcn_sched_barrier(0);             // the destinations are worked out while the loads are under way
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int r = rk + i * (64 / KP);
            const int64_t ok_ = lane_value(dk, r), ov = lane_value(dv, r);
            if (rows >> r & 1) {
                store_hint<u32x4, ROWS == 64>((T*)dst.k.ptr + ok_ + E * pk, xk[i]);
                store_hint<u32x4, ROWS == 64>((T*)dst.v.ptr + ov + E * pk, xv[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int r = rb + i * (64 / BP);
            const int64_t o = lane_value(db, r);
            if (rows >> r & 1) store_hint<u32x4, ROWS == 64>((T*)dst.b.ptr + o + E * pb, xb[i]);
        }
    }
    if (ok) {
        ((float*)dst.g.ptr)[at(dst.g, d0, d2)] = g;
        if (dst.f.ptr) ((float*)dst.f.ptr)[at(dst.f, d0, d2)] = f;
    }
}

SISA_DEV RowViews rows_of_pool(const sisa_page_pool& p) { return RowViews{p.k, p.v, p.b, p.g, p.f}; }

namespace sisa {

// Bytes of a row of k, v, b, g and F.
inline int64_t row_bytes(int dtype) { return 160 * (int64_t)elem_size(dtype) + 8; }

// Bytes that a call reads at most of a pool's caches: the host does not know the lengths, but max_len positions of each
// sequence and the whole pool bound them.
inline int64_t cache_bytes(const sisa_page_pool& p, int64_t sequences, int64_t max_len) {
    const int64_t most = sequences * p.heads * max_len, held = (int64_t)p.pages * p.heads * p.page_size;
    return (most < held ? most : held) * row_bytes(p.dtype);
}

// Rows a wave moves: 64 from two waves of that on every SIMD on.
inline int rows_per_wave(int64_t rows) { return rows >= 64 * 2048 ? 64 : 8; }

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

// What attention over common positions asks of a pool beside: rows of a page behind each other, within 32-bit offsets.
inline bool near_rows(const sisa_page_pool& p) {
    auto ok = [&](const sisa_view& x, int width, int size) {
        return x.sl >= width && x.sl <= 0x7fffff00 / ((int64_t)p.page_size * size);
    };
    const int es = elem_size(p.dtype);
    return ok(p.k, 64, es) && ok(p.v, 64, es) && ok(p.b, 32, es) && ok(p.g, 1, 4) && (!p.f.ptr || ok(p.f, 1, 4));
}

}  // namespace sisa

#define SISA_REQUIRE_POOL(name, pool)                                       \
    do {                                                                    \
        const char* fault_ = ::sisa::pool_fault(pool);                      \
        SISA_REQUIRE(fault_ == nullptr, "%s: %s", name, fault_);            \
    } while (0)
#define SISA_REQUIRE_NEAR_ROWS(name, pool)                                  \
    SISA_REQUIRE(::sisa::near_rows(pool), "%s: the positions of a page must be at least a row apart, and all of a head's within 2 GiB", name)
