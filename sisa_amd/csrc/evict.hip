// Eviction from a paged generation cache by accumulated attention weight for gfx950 (include/sisa_hip_cache.h): which
// positions of each head stay, and their rows copied in order to other pages.
//
// The selection is a radix select on the weights' bit patterns, mapped so that they order as unsigned integers: one
// workgroup per (sequence, head) counts the digits of eight bits from the top in LDS (integer counts: their order does not
// matter), narrows to the digit that holds the last position to keep, and after four digits knows the smallest weight that
// stays and how many of its equals do. Waves own contiguous ranges of positions, so positions come out in order.
#include "pages.h"

namespace {

constexpr int DH = 64, DS = 32;
constexpr int SW = 16;                // waves of the selection

// Orders as the weight does: NaN above all, both zeros alike.
SISA_DEV unsigned order_of(float x) {
    if (x != x) return 0xffffffffu;
    const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

SISA_DEV int count_of(uint64_t lanes) { return __builtin_popcountll(lanes); }
SISA_DEV int below(uint64_t lanes, int lane) { return __builtin_popcountll(lanes & ((1ull << lane) - 1)); }

__global__ __launch_bounds__(64 * SW) void evict_select_kernel(sisa_cache_evict_args a, int shift, int new_shift) {
    __shared__ unsigned hist[256];
    __shared__ unsigned found, left;                   // the digit with the last one to keep, and how many to keep in it
    __shared__ int gt[SW], eq[SW];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int H = a.from.heads, nh = blockIdx.x, h = nh % H, n = nh / H;
    const int len = a.lengths[n], keep = a.keep, recent = a.recent;
    int32_t* pos = a.positions + (int64_t)nh * keep;
    float* neww = a.new_weights + (int64_t)nh * keep;
    const float* W = (const float*)a.weights.ptr + n * a.weights.sb + h * a.weights.sh;
    const int64_t sl = a.weights.sl;
    const int out = len < keep ? len : keep;
    const bool bad = len < 0 || len > a.max_len || len > ((int64_t)a.W << shift) || out > ((int64_t)a.W_new << new_shift);
    if (h == 0 && tid == 0) a.new_lengths[n] = bad ? -1 : out;
    for (int i = (bad ? 0 : out) + tid; i < keep; i += 64 * SW) pos[i] = -1, neww[i] = 0.f;
    if (bad) return;
    if (len <= keep) {
        for (int i = tid; i < len; i += 64 * SW) pos[i] = i, neww[i] = W[i * sl];
        return;
    }
    const int old = len - recent, pick = keep - recent;        // pick of the first `old`, then the recent ones
    for (int i = tid; i < recent; i += 64 * SW) pos[pick + i] = old + i, neww[pick + i] = W[(old + i) * sl];
    if (pick == 0) return;

    // The smallest key that stays, digit by digit; `want` of the keys with the digits so far are still to be picked.
    unsigned prefix = 0, want = pick;
    for (int d = 24; d >= 0; d -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < old; i += 64 * SW) {
            const unsigned k = order_of(W[i * sl]);
            if (d == 24 || (k >> (d + 8)) == (prefix >> (d + 8))) atomicAdd(&hist[(k >> d) & 255], 1u);
        }
        __syncthreads();
        if (w == 0) {
            // lane l: digits 255 - 4 l down to 252 - 4 l; above: how many keys have a larger digit
            unsigned c[4], mine = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = hist[255 - 4 * lane - e], mine += c[e];
            unsigned incl = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const unsigned t = __shfl_up(incl, o);
                if (lane >= o) incl += t;
            }
            unsigned above = incl - mine;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (above < want && want <= above + c[e]) found = 255 - 4 * lane - e, left = want - above;
                above += c[e];
            }
        }
        __syncthreads();
        prefix |= found << d;
        want = left;
        __syncthreads();
    }

    // A wave's range of positions: those above the smallest key, and its equals from the lowest position on.
    const int per = ((old + SW - 1) / SW + 63) / 64 * 64, i0 = w * per, i1 = i0 + per < old ? i0 + per : old;
    int ng = 0, ne = 0;
    for (int i = i0; i < i1; i += 64) {
        const bool in = i + lane < i1;
        const unsigned k = in ? order_of(W[(i + lane) * sl]) : 0;
        ng += count_of(__ballot(in && k > prefix));
        ne += count_of(__ballot(in && k == prefix));
    }
    if (lane == 0) gt[w] = ng, eq[w] = ne;
    __syncthreads();
    int at = 0, equals = 0;
    for (int k = 0; k < w; ++k) {
        const int take = (int)want - equals;           // equals that are still to be picked from wave k on
        at += gt[k] + (take < 0 ? 0 : take < eq[k] ? take : eq[k]);
        equals += eq[k];
    }
    for (int i = i0; i < i1; i += 64) {
        const bool in = i + lane < i1;
        const float x = in ? W[(i + lane) * sl] : 0.f;
        const unsigned k = order_of(x);
        const uint64_t same = __ballot(in && k == prefix);
        const bool stay = in && (k > prefix || (k == prefix && equals + below(same, lane) < (int)want));
        const uint64_t stays = __ballot(stay);
        if (stay) {
            const int to = at + below(stays, lane);
            pos[to] = i + lane;
            neww[to] = x;
        }
        at += count_of(stays);
        equals += count_of(same);
    }
}

// 32 threads per (sequence, head, kept row), as the write of new positions. A row without a page marks its sequence.
template <class T>
__global__ __launch_bounds__(256) void evict_copy_kernel(sisa_cache_evict_args a, int shift, int new_shift) {
    const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int t = threadIdx.x & 31, H = a.from.heads;
    if (id >= (int64_t)a.B * H * a.keep) return;
    const int i = (int)(id % a.keep);
    const int64_t nh = id / a.keep;
    const int h = (int)(nh % H), n = (int)(nh / H);
    const int j = a.positions[id];
    if (j < 0) return;
    const int src = page_of(a.table + n * a.s_table, a.W, shift, a.from.pages, j);
    const int dst = page_of(a.new_table + n * a.s_new, a.W_new, new_shift, a.to.pages, i);
    if (src < 0 || dst < 0) {
        if (t == 0) a.new_lengths[n] = -1;
        return;
    }
    const int64_t sslot = j & (a.from.page_size - 1), dslot = i & (a.to.page_size - 1);
    if (t < 20) {
        const sisa_view& s = t < 8 ? a.from.k : t < 16 ? a.from.v : a.from.b;
        const sisa_view& d = t < 8 ? a.to.k : t < 16 ? a.to.v : a.to.b;
        const int e = 8 * (t < 16 ? t & 7 : t - 16);
        *reinterpret_cast<frag8<T>*>((T*)d.ptr + dst * d.sb + h * d.sh + dslot * d.sl + e) =
            load8<T>((const T*)s.ptr + src * s.sb + h * s.sh + sslot * s.sl + e);
    } else if (t < 22) {
        const sisa_view& s = t == 20 ? a.from.g : a.from.f;
        const sisa_view& d = t == 20 ? a.to.g : a.to.f;
        if (s.ptr)
            ((float*)d.ptr)[dst * d.sb + h * d.sh + dslot * d.sl] =
                ((const float*)s.ptr)[src * s.sb + h * s.sh + sslot * s.sl];
    }
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
    const int64_t heads = (int64_t)a->B * a->from.heads, groups = sisa::cdiv(heads * a->keep, 8);
    SISA_REQUIRE(groups < ((int64_t)1 << 31), "sisa_cache_evict: B*H*keep too large for one launch");
    const int shift = sisa::log2_of(a->from.page_size), new_shift = sisa::log2_of(a->to.page_size);
    hipStream_t st = (hipStream_t)stream;
    evict_select_kernel<<<(unsigned)heads, 64 * SW, 0, st>>>(*a, shift, new_shift);
    const int rc = sisa::launch_status("sisa_cache_evict (selection)");
    if (rc) return rc;
    switch (a->from.dtype) {
        case SISA_BF16: evict_copy_kernel<__bf16><<<(unsigned)groups, 256, 0, st>>>(*a, shift, new_shift); break;
        case SISA_F16: evict_copy_kernel<_Float16><<<(unsigned)groups, 256, 0, st>>>(*a, shift, new_shift); break;
        default: evict_copy_kernel<float><<<(unsigned)groups, 256, 0, st>>>(*a, shift, new_shift);
    }
    return sisa::launch_status("sisa_cache_evict (copy)");
}
