// Eviction from a paged generation cache by accumulated attention weight for gfx950 (include/sisa_hip_cache.h): which
// positions of each head stay, and their rows copied in order to other pages.
//
// The selection is a radix select on the weights' bit patterns, mapped so that they order as unsigned integers: one
// workgroup per (sequence, head) counts the digits of eight bits from the top in LDS (integer counts: their order does not
// matter), narrows to the digit that holds the last position to keep, and after four digits, or once all that have the digit
// stay, knows the smallest weight that stays and how many of its equals do. Waves own contiguous ranges of positions, so
// positions come out in order. The keys stay in registers (up to 24 a thread: 24,576 positions; longer caches are read again
// for every digit), loaded beside the length. Accumulated weights share their leading bits, so that the lanes of a wave count
// the same few digits: eight copies of the counters, one per lane modulo 8, keep a count from waiting for 63 others.
//
// Bound by latency: 96 workgroups of 16,384 positions take 11.8 us, of it 3.5 before the first count (the weights, from HBM),
// 1.7 for the first digit, whose counts meet most often, 1.2 for each other one (two barriers, wave 0's scan between them) and
// 1.5 for the positions; 256 of up to 5,003 positions 7.5 us (room for 16 keys a thread in place of 8: 9.8).
#include "pages.h"

namespace {

constexpr int SW = 16;                // waves of the selection

// Orders as the weight does: NaN above all, both zeros alike.
SISA_DEV unsigned order_of(float x) {
    if (x != x) return 0xffffffffu;
    const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

SISA_DEV int count_of(uint64_t lanes) { return __builtin_popcountll(lanes); }
SISA_DEV int below(uint64_t lanes) {                   // of them before this lane
    return __builtin_amdgcn_mbcnt_hi((unsigned)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)lanes, 0u));
}

// x summed over the wave's lanes up to this one.
template <int CTRL, int ROWS> SISA_DEV unsigned from_lane(unsigned x) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
SISA_DEV unsigned wave_scan(unsigned x) {
    x += from_lane<0x111, 0xf>(x);                     // 1, 2, 4, 8 lanes below within the rows of 16
    x += from_lane<0x112, 0xf>(x);
    x += from_lane<0x114, 0xf>(x);
    x += from_lane<0x118, 0xf>(x);
    x += from_lane<0x142, 0xa>(x);                     // the last lane of rows 0 and 2 to rows 1 and 3
    return x + from_lane<0x143, 0xc>(x);               // lane 31 to rows 2 and 3
}

constexpr int COPIES = 8, COPY = 260;  // counters' copies, and from one to the next (a digit's copies on banks of their own)

// NK keys a thread in registers, or 0: read from memory each time they are needed.
template <int NK>
__global__ __launch_bounds__(64 * SW) void evict_select_kernel(sisa_cache_evict_args a, int shift, int new_shift) {
    __shared__ __attribute__((aligned(16))) unsigned hists[4][COPIES * COPY];       // of the four digits
    __shared__ unsigned found, left;                   // the digit with the last one to keep, and how many to keep in it
    __shared__ bool whole;                             // which are all that have it
    __shared__ int gt[SW], eq[SW];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int H = a.from.heads, nh = blockIdx.x, h = nh % H, n = nh / H;
    // The wave's range of positions, 64 at a time. Its weights are under way beside the length, not after it.
    const int steps = ((a.max_len + SW - 1) / SW + 63) / 64, i0 = w * steps * 64;
    const int64_t step = 64 * a.weights.sl;
    const float* W = (const float*)a.weights.ptr + (n * a.weights.sb + h * a.weights.sh) + (int64_t)(i0 + lane) * a.weights.sl;
    float x[NK ? NK : 1];
    if constexpr (NK > 0) {
#pragma unroll
        for (int s = 0; s < NK; ++s) {
            x[s] = s < steps && i0 + 64 * s + lane < a.max_len ? W[s * step] : 0.f;
        }
    }
    const int len = a.lengths[n], keep = a.keep, recent = a.recent;
    int32_t* pos = a.positions + (int64_t)nh * keep;
    const int out = len < keep ? len : keep;
    const bool bad = len < 0 || len > a.max_len || len > ((int64_t)a.W << shift) || out > ((int64_t)a.W_new << new_shift);
    if (h == 0 && tid == 0) a.new_lengths[n] = bad ? -1 : out;
    for (int i = (bad ? 0 : out) + tid; i < keep; i += 64 * SW) pos[i] = -1;
    if (bad) return;
    if (len <= keep) {
        for (int i = tid; i < len; i += 64 * SW) pos[i] = i;
        return;
    }
    const int old = len - recent, pick = keep - recent;        // pick of the first `old`, then the recent ones
    unsigned key[NK ? NK : 1];                         // 0, below every weight's, where there is no position
    if constexpr (NK > 0) {
#pragma unroll
        for (int s = 0; s < NK; ++s) key[s] = i0 + 64 * s + lane < old ? order_of(x[s]) : 0u;
    }
    for (int i = tid; i < recent; i += 64 * SW) pos[pick + i] = old + i;
    if (pick == 0) return;
    // f(position, key) for each of the wave's positions in order, all lanes together; key 0 where there is none
    const int mine = i0 >= old ? 0 : (old - i0 + 63) / 64 < steps ? (old - i0 + 63) / 64 : steps;
    auto each = [&](auto&& f) {
        if constexpr (NK > 0) {
#pragma unroll
            for (int s = 0; s < NK; ++s)
                if (s < mine) f(i0 + 64 * s + lane, key[s]);
        } else {
            for (int s0 = 0; s0 < mine; s0 += 8) {             // eight loads under way
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int i = i0 + 64 * (s0 + e) + lane;
                    y[e] = s0 + e < mine && i < old ? W[(s0 + e) * step] : 0.f;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (s0 + e < mine) {
                        const int i = i0 + 64 * (s0 + e) + lane;
                        f(i, i < old ? order_of(y[e]) : 0u);
                    }
            }
        }
    };

    // The smallest key that stays, digit by digit; `want` of the keys with the digits so far are still to be picked.
    unsigned prefix = 0, want = pick;
    for (int i = tid; i < 4 * COPIES * COPY; i += 64 * SW) (&hists[0][0])[i] = 0;
    __syncthreads();
    for (int d = 24; d >= 0; d -= 8) {
        unsigned* hist = hists[d >> 3];
        const unsigned high = d == 24 ? 0u : prefix >> (d + 8);
        each([&](int, unsigned k) {
            if (k && (d == 24 || k >> (d + 8) == high)) atomicAdd(&hist[(lane & (COPIES - 1)) * COPY + (k >> d & 255)], 1u);
        });
        __syncthreads();
        if (w == 0) {
            // lane l: digits 255 - 4 l down to 252 - 4 l; above: how many keys have a larger digit
            u32x4 c = {0, 0, 0, 0};                        // of digits 252 - 4 l up
#pragma unroll
            for (int k = 0; k < COPIES; ++k) c += *reinterpret_cast<const u32x4*>(hist + k * COPY + 252 - 4 * lane);
            const unsigned four = (c[0] + c[1]) + (c[2] + c[3]);
            unsigned above = wave_scan(four) - four;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (above < want && want <= above + c[3 - e])
                    found = 255 - 4 * lane - e, left = want - above, whole = want == above + c[3 - e];
                above += c[3 - e];
            }
        }
        __syncthreads();
        prefix |= found << d;
        want = left;
        if (whole && prefix) {                         // all with this digit stay: nothing is left to tell apart
            --prefix, want = 0;
            break;
        }
    }

    // Those above the smallest key, and its equals from the lowest position on.
    unsigned ng = 0, ne = 0;
    each([&](int, unsigned k) {
        ng += k > prefix;
        ne += k == prefix;
    });
    ng = wave_scan(ng);
    ne = wave_scan(ne);
    if (lane == 63) gt[w] = ng, eq[w] = ne;
    __syncthreads();
    int at = 0, equals = 0;
    for (int k = 0; k < w; ++k) {
        const int take = (int)want - equals;           // equals that are still to be picked from wave k on
        at += gt[k] + (take < 0 ? 0 : take < eq[k] ? take : eq[k]);
        equals += eq[k];
    }
    if (equals >= (int)want) {                         // no equals of this wave
        each([&](int i, unsigned k) {
            const uint64_t stays = __ballot(k > prefix);
            if (k > prefix) pos[at + below(stays)] = i;
            at += count_of(stays);
        });
        return;
    }
    each([&](int i, unsigned k) {
        const uint64_t same = __ballot(k == prefix);
        const bool stay = k > prefix || (k == prefix && equals + below(same) < (int)want);
        const uint64_t stays = __ballot(stay);
        if (stay) pos[at + below(stays)] = i;
        at += count_of(stays);
        equals += count_of(same);
    });
}

// A wave moves ROWS kept rows and their weights. A row without a page marks its sequence.
template <class T, int ROWS, bool STREAM>
__global__ __launch_bounds__(256) void evict_copy_kernel(sisa_cache_evict_args a, int shift, int new_shift) {
    const int lane = threadIdx.x & 63;
    const unsigned id = (blockIdx.x * 4 + (threadIdx.x >> 6)) * ROWS + lane, keep = a.keep, H = a.from.heads;
    const unsigned nh = id / keep, h = nh % H;
    const int i = id % keep;
    const int64_t n = nh / H;
    const bool mine = lane < ROWS && n < a.B;
    const int j = mine ? a.positions[id] : -1;
    int src = -1, dst = -1;
    float weight = 0.f;
    if (j >= 0) {
        weight = ((const float*)a.weights.ptr)[n * a.weights.sb + h * a.weights.sh + j * a.weights.sl];
        src = page_of(a.table + n * a.s_table, a.W, shift, a.from.pages, j);
        dst = page_of(a.new_table + n * a.s_new, a.W_new, new_shift, a.to.pages, i);
        if (src < 0 || dst < 0) a.new_lengths[n] = -1;
    }
    if (mine) a.new_weights[id] = weight;
    move_rows<T, ROWS, STREAM>(rows_of_pool(a.from), rows_of_pool(a.to), src >= 0 && dst >= 0, src, dst, h,
                               j & (a.from.page_size - 1), i & (a.to.page_size - 1), lane);
}

template <class T>
void launch_copy(const sisa_cache_evict_args* a, int64_t rows, hipStream_t st) {
    const int shift = sisa::log2_of(a->from.page_size), new_shift = sisa::log2_of(a->to.page_size);
    const int per = 4 * sisa::rows_per_wave(rows);
    const unsigned grid = (unsigned)sisa::cdiv(rows, per);
    if (per != 256) evict_copy_kernel<T, 8, false><<<grid, 256, 0, st>>>(*a, shift, new_shift);
    else if (sisa::cache_bytes(a->from, a->B, a->max_len) < STREAM_BYTES)
        evict_copy_kernel<T, 64, false><<<grid, 256, 0, st>>>(*a, shift, new_shift);
    else evict_copy_kernel<T, 64, true><<<grid, 256, 0, st>>>(*a, shift, new_shift);
}

}  // namespace

extern "C" int sisa_cache_evict(const sisa_cache_evict_args* a, void* stream) {
    SISA_REQUIRE(a != nullptr, "sisa_cache_evict: null args");
    SISA_REQUIRE_POOL("sisa_cache_evict", a->from);
    SISA_REQUIRE_POOL("sisa_cache_evict", a->to);
    SISA_REQUIRE(a->from.heads == a->to.heads && a->from.dtype == a->to.dtype &&
                     (a->from.f.ptr == nullptr) == (a->to.f.ptr == nullptr),
                 "sisa_cache_evict: the pools must agree in heads, dtype and the forget term");
    SISA_REQUIRE(a->B >= 0 && a->W >= 1 && a->W_new >= 1 && a->max_len >= 1 &&
                     a->max_len <= (int64_t)a->W * a->from.page_size && a->max_len <= (1 << 30),
                 "sisa_cache_evict: bad shape B=%d W=%d W_new=%d max_len=%d (at most W pages of %d, and 2^30)", a->B, a->W,
                 a->W_new, a->max_len, a->from.page_size);
    SISA_REQUIRE(a->recent >= 1 && a->recent <= a->keep, "sisa_cache_evict: recent=%d must be in 1 .. keep=%d", a->recent,
                 a->keep);
    if (a->B == 0) return SISA_OK;
    SISA_REQUIRE(a->table && a->new_table && a->lengths && a->weights.ptr && a->new_lengths && a->new_weights && a->positions,
                 "sisa_cache_evict: null pointer");
    const int64_t heads = (int64_t)a->B * a->from.heads, rows = heads * a->keep;
    SISA_REQUIRE(rows < ((int64_t)1 << 31) && heads <= sisa::MAX_THREADS / (64 * SW),
                 "sisa_cache_evict: B*H*keep must be below 2^31, B*H below 2^22");
    const int shift = sisa::log2_of(a->from.page_size), new_shift = sisa::log2_of(a->to.page_size);
    hipStream_t st = (hipStream_t)stream;
    const int64_t per = sisa::cdiv(a->max_len, 64 * SW);       // keys a thread
    if (per <= 4) evict_select_kernel<4><<<(unsigned)heads, 64 * SW, 0, st>>>(*a, shift, new_shift);
    else if (per <= 8) evict_select_kernel<8><<<(unsigned)heads, 64 * SW, 0, st>>>(*a, shift, new_shift);
    else if (per <= 16) evict_select_kernel<16><<<(unsigned)heads, 64 * SW, 0, st>>>(*a, shift, new_shift);
    else if (per <= 24) evict_select_kernel<24><<<(unsigned)heads, 64 * SW, 0, st>>>(*a, shift, new_shift);
    else evict_select_kernel<0><<<(unsigned)heads, 64 * SW, 0, st>>>(*a, shift, new_shift);
    const int rc = sisa::launch_status("sisa_cache_evict (selection)");
    if (rc) return rc;
    switch (a->from.dtype) {
        case SISA_BF16: launch_copy<__bf16>(a, rows, st); break;
        case SISA_F16: launch_copy<_Float16>(a, rows, st); break;
        default: launch_copy<float>(a, rows, st);
    }
    return sisa::launch_status("sisa_cache_evict (copy)");
}
