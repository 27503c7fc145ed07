// Attention of the new positions of sequences that share their first positions, for gfx950 (include/sisa_hip_branch.h).
//
//   s_mj = q_m.k_j / 8 + lam exp(g_m - g_j) (c_m.b_j) + (F_m - F_j);   out_m = softmax_j(s_mj) v_j
//
// The softmax over a sequence's positions is joined from its parts: the common positions, which the query rows of a group see
// alike, and its own. Both are the same work for a wave: up to 16 query rows against a range of positions in the pages of one
// table row, 32 positions (a tile) at a time on the matrix cores. Of a group of more than 16 rows, two or four waves of a
// workgroup have rows of their own and go through the same positions side by side, so that the cached rows come from memory
// once and from the nearest cache for the others; the remaining ones split the positions.
//
// Scores are computed transposed (S^T = K Q^T), so that a lane has one query row's softmax and the weights are the operand of
// O^T += V^T P^T as they are. K and b~ go from memory to the operand registers; v passes through LDS, which transposes it. The
// weights enter their product as a sum of two (fp16) or three (bf16) operands, so that the result is an fp32 one: rounded once
// to bf16 they would be off by 2^-9.
//
// Both launches, from a kernel trace, bf16: 64 rows against 16,384 common positions of 12 heads 41 us (114 MB at 2.8 TB/s; reading
// alone reaches 7.1), 24 x 8 drafts against up to 6,000 46 us (169 MB, 3.7 TB/s), 256 rows against 1,500 and up to 1,000 of
// their own 60 us. What bounds the first launch of the 64 rows is the L1, which serves four waves that each load the same rows
// (52,000 accesses a CU in 67,000 cycles; VALU 46 %, matrix cores 12 %); that of the drafts, waves that wait for their one tile
// (45 % of their cycles). What a wave holds is kept few enough for four waves a SIMD, strides and bases in scalar registers. The first
// launch for the 64 rows: 64 rows to a wave, 256 registers 91 us; 16 rows to a wave, 168 registers 41; this form 34. A head's
// positions are read beside the other heads', whose rows follow in memory: with each head by itself an earlier form of the
// loads took 47 us there, against 36.
#include "pages.h"
#include "sisa_hip_branch.h"

namespace {

constexpr int DH = 64, DS = 32;
constexpr int KT = 32;                // positions of a tile
constexpr int NW = 4;                 // waves of a workgroup
constexpr int MOST = 64;              // most parts of a range: the join has a lane for each

// How a call is cut: the query rows of all groups into tiles of 16 << log_rw, 16 to a wave; a group's common positions into
// `parts` workgroups of 4 >> log_rw waves a row, a sequence's own ones into `own_parts` waves.
struct Plan {
    int log_rw;
    unsigned tiles, own_tiles, parts, own_parts, own_rows;
    unsigned items, own_items;        // workgroups and waves of a head
    unsigned blocks;                  // workgroups of the common parts, of all heads
};

// Tiles of all groups' query rows: group r's begin at r + floor(first[r] M / rows of a tile), which leaves room for each.
SISA_DEV int64_t tile_base(const sisa_prefix_decode_args& a, int r, int log_per) {
    const int64_t n = a.first[r];
    return r + ((n < 0 ? 0 : n > a.B ? a.B : n) * a.M >> log_per);
}

// The tiles of KT positions that part p of a range of n tiles has: [from, to).
struct Range { int from, to; };
SISA_DEV Range part_of(int n, unsigned parts, unsigned p) {
    const int each = ((unsigned)n + parts - 1) / parts, from = each * p;
    return Range{from, from + each < n ? from + each : n};
}

// What a row sees at most of its sequence; -1 for a length that the call does not take.
SISA_DEV int visible(const sisa_prefix_decode_args& a, int64_t held, int n, int m) {
    const int len = a.lengths[n];
    if (len < 0 || len > a.max_len || len > held) return -1;
    const int last = len - a.M + m + 1;
    return last > 0 ? last : 0;
}
SISA_DEV int common(const sisa_prefix_decode_args& a, int64_t held, int r) {
    const int s = a.shared[r];
    return s < 0 || s > a.max_shared || s > held ? -1 : s;
}

template <class T> struct Split;      // operands that a weight is the sum of: what is left of 24 bits is not seen in an fp32 sum
template <> struct Split<__bf16> { static constexpr int terms = 3; };
template <> struct Split<_Float16> { static constexpr int terms = 2; };
template <> struct Split<float> { static constexpr int terms = 1; };

// Weights are exponentials over a row's reference, which is moved to its largest score when a lane's eight weights of a tile
// sum up to more than 2^8 (a column of the operand is summed by four lanes, each of which can move it). fp16 weights are
// larger by 2^7: at most 2^15, and the low parts of small ones stay above the subnormals.
template <class T> constexpr float UP = __is_same(T, _Float16) ? 7.f : 0.f;
constexpr float RAISE = 8.f;
constexpr float LEAST = -3.402823466e38f;      // a row's first reference: finite, so that no weight is inf - inf
constexpr float FACTORED = 60.f;               // largest exponent (log2) of a factor of a decay

template <class T>
struct __attribute__((aligned(16))) WaveLds {
    T v[KT * DH];
    float g[KT], f[KT];
};

// Up to 16 query rows, counted from sequence n0's first, against positions lo <= j < hi of a table row.
struct Work {
    int h, n0, r0, rows, lo, hi;
};

// What a wave loads of a tile: K and b~ as operands, v in 16-byte pieces, g and F of the position lane % 16 of either half.
template <class T>
struct Tile {
    static constexpr int E = 16 / (int)sizeof(T), CPR = DH / E, PASS = KT * CPR / 64;     // elements and pieces of a row
    frag8<T> k[2][2], b[2];
    u32x4 v[PASS];
    float g[2], f[2];
};

// A scalar in registers of its own: as part of the wide load of the kernel's arguments it would keep all of that alive.
template <class X> SISA_DEV X apart(X x) {
    asm("" : "+s"(x));
    return x;
}

// The exponents of a 32-bit word of T, 1 in their lowest places, and the signs.
template <class T> constexpr unsigned EXPONENT = sizeof(T) == 4 ? 0x7f800000 : __is_same(T, __bf16) ? 0x7f807f80 : 0x7c007c00;
template <class T> constexpr unsigned EXPONENT_ONE = sizeof(T) == 4 ? 0x00800000 : __is_same(T, __bf16) ? 0x00800080 : 0x04000400;
template <class T> constexpr unsigned SIGN = sizeof(T) == 4 ? 0x80000000 : 0x80008000;

// Loads at a lane's offset from a scalar base and a scalar one, 0 from `bytes` on.
template <class V> SISA_DEV V load_at(const char* base, int bytes, int voff, int soff) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(base, bytes);
    if constexpr (sizeof(V) == 4) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b32(r, voff, soff, 0));
    else return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 0));
}
template <class T> SISA_DEV frag8<T> load_frag(const char* base, int bytes, int voff, int soff) {
    if constexpr (sizeof(T) == 2) return load_at<frag8<T>>(base, bytes, voff, soff);
    else return join<T>(load_at<f32x4>(base, bytes, voff, soff), load_at<f32x4>(base, bytes, voff, soff + 16));
}

// One tensor of the pool as a head's waves see it: where the head begins, bytes from page to page and from row to row, and
// what a lane adds to the first of 16 rows.
struct Stream {
    const char* base;
    int64_t page;
    int row, lane;
    SISA_DEV void init(const sisa_view& x, int h, int size, int lane_row, int lane_col) {
        base = apart((const char*)x.ptr + h * x.sh * size);
        page = apart(x.sb * size);
        row = apart((int)x.sl * size);
        lane = lane_row * row + lane_col;
    }
    SISA_DEV const char* at(int p) const { return base + p * page; }
};

struct Space {
    f32x2 *stat, *own_stat;
    float *part, *own;
    int64_t bytes;
};
struct PartArgs {
    sisa_prefix_decode_args a;
    Plan plan;
    int shift;
    Space ws;
};
// A kernel's argument read again where it is needed: kept from the beginning they do not fit the scalar registers.
template <class X> SISA_DEV X again(size_t offset) {
    typedef const __attribute__((address_space(4))) char* Const;
    Const p = (Const)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const __attribute__((address_space(4))) X*)(p + offset);
}
#define AGAIN(field) again<decltype(PartArgs::field)>(offsetof(PartArgs, field))

// The workgroups of the common parts, then those of the own ones, whose waves are on their own. Unnormalised outputs go to
// `part`, a tile of rows an item, and `own_part`; each row's reference (log2) and sum to `stat` and `own_stat`.
template <class T>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 2 ? 4 : 3))) void prefix_part_kernel(
    PartArgs args) {
    constexpr int LD = DH + 4;         // rows apart by 4 banks
    __shared__ WaveLds<T> lds[NW];
    __shared__ __attribute__((aligned(16))) float ms[NW][16], ls[NW][16], os[NW][16][LD];
    const sisa_prefix_decode_args& a = args.a;
    const Plan& plan = args.plan;
    const int tid = threadIdx.x, lane = tid & 63, grp = lane >> 4, lc = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // The heads of an item, whose rows are neighbours in memory, follow each other.
    const unsigned H = a.pool.heads;
    const bool own = blockIdx.x >= plan.blocks;
    const unsigned nth = own ? (blockIdx.x - plan.blocks) * NW + w : blockIdx.x, item = nth / H;
    const int64_t held = (int64_t)a.W << args.shift;
    const int log_rw = plan.log_rw, rw = 1 << log_rw, log_per = 4 + log_rw;
    Work k;
    k.h = nth - item * H;
    Range t;                                             // the wave's tiles
    if (own) {
        if (item >= plan.own_items) return;
        const unsigned pn = plan.own_tiles == 1 ? item : item / plan.own_tiles, p = pn / (unsigned)a.B, n = pn - p * a.B;
        k.n0 = n;
        k.r0 = 16 * (item - pn * plan.own_tiles);
        k.rows = a.M - k.r0 < 16 ? a.M - k.r0 : 16;
        const int r = a.group[n];
        k.hi = visible(a, held, n, k.r0 + k.rows - 1);
        if (r < 0 || r >= a.G) return;
        k.lo = common(a, held, r);
        if (k.lo < 0 || k.hi <= k.lo) return;
        const int first = k.lo / KT;
        t = part_of((k.hi + KT - 1) / KT - first, plan.own_parts, p);
        if (t.from >= t.to) return;
        t.from += first;
        t.to += first;
    } else {
        // tile by tile: those that no group needs come last
        const unsigned tile = item / plan.parts, p = item - tile * plan.parts;
        int r = 0;                                       // the last group whose tiles begin at or before this one
        if (a.G > 1) {
            r = -1;
            for (int i = 0; i < a.G; i += 64) r += __popcll(__ballot(i + lane < a.G && tile_base(a, i + lane, log_per) <= tile));
            if (r < 0) return;
        }
        const int f0 = a.first[r], f1 = a.first[r + 1];
        k.hi = common(a, held, r);
        if (f0 < 0 || f1 > a.B || f1 <= f0 || k.hi <= 0) return;
        const int64_t all = (int64_t)(f1 - f0) * a.M, past = (int64_t)tile - tile_base(a, r, log_per);
        const int64_t at = (past << log_per) + 16 * (w & (rw - 1));
        if (past < 0 || past << log_per >= all) return;
        k.n0 = f0;
        k.r0 = at;
        k.rows = at >= all ? 0 : all - at < 16 ? all - at : 16;
        k.lo = 0;
        const int n = (k.hi + KT - 1) / KT, kw = NW >> log_rw;
        if (part_of(n, plan.parts * kw, p * kw).from >= n) return;
        t = part_of(n, plan.parts * kw, p * kw + (w >> log_rw));
        if (!k.rows) t.to = t.from;
    }
    const auto table = apart((const __attribute__((address_space(1))) int32_t*)a.table + k.n0 * a.s_table);

    // Column lc of the operand is query row lc, in all four groups of lanes; behind the last row the last again.
    frag8<T> q[2], c;
    float gq, fq = 0.f, m2 = LEAST, l = 0.f;             // l: the lane's part
    int len, back, lim = 0, least = 0;                   // positions that the row sees, and that every row does
    f32x4 o[4] = {zero4(), zero4(), zero4(), zero4()};   // output features 16 db + 4 grp + i
    {
        const int r = k.r0 + (lc < k.rows ? lc : k.rows - 1);
        int n = k.n0, m = r;
        if (!own) {
            const unsigned d = a.M == 1 ? r : (unsigned)r / (unsigned)a.M;
            n += d;
            m -= d * a.M;
        }
        if (!k.rows) n = m = 0;
        len = a.lengths[n];
        back = a.M - 1 - m;
        gq = ((const float*)a.gq.ptr)[n * a.gq.sb + k.h * a.gq.sh + m * a.gq.sl];
        if (a.fq.ptr) fq = ((const float*)a.fq.ptr)[n * a.fq.sb + k.h * a.fq.sh + m * a.fq.sl];
        const T *rq = (const T*)a.q.ptr + (n * a.q.sb + k.h * a.q.sh + m * a.q.sl) + 8 * grp;
        q[0] = load8<T>(rq);
        q[1] = load8<T>(rq + 32);
        c = load8<T>((const T*)a.c.ptr + (n * a.c.sb + k.h * a.c.sh + m * a.c.sl) + 8 * grp);
    }
    const float lam = a.lam[k.h * a.s_lam] * LOG2E;
    const int mask = apart(a.pool.page_size - 1), pages = apart(a.pool.pages), W = apart(a.W), shift = apart(args.shift);
    const int max_len = apart(a.max_len);
    const bool has_f = a.pool.f.ptr != nullptr;
    using X = Tile<T>;
    Stream sk, sv, sb, sg, sf;
    {
        const int row = lane / X::CPR, col = 16 * (lane % X::CPR), part = 8 * grp * (int)sizeof(T);
        sk.init(a.pool.k, k.h, sizeof(T), lc, part);
        sv.init(a.pool.v, k.h, sizeof(T), row, col);
        sb.init(a.pool.b, k.h, sizeof(T), lc, part);
        sg.init(a.pool.g, k.h, 4, lc, 0);
        sf.init(has_f ? a.pool.f : a.pool.g, k.h, 4, lc, 0);
    }

    auto page_at = [&](int j) {                          // -1: none of the pool's
        const int i = j >> shift, p = i < W ? table[i] : -1;
        return p < pages ? p : -1;
    };
    WaveLds<T>& sm = lds[w];
    bool odd = false;
    int near_pages = -1, base = t.from - 32;             // lane i: the page of the 16 positions from 16 (2 base + i) on
#pragma unroll 1
    for (int tile = t.from; tile < t.to; ++tile) {
        const int jt = tile * KT;
        if (tile - base >= 32) {
            base = tile;
            const int j = 16 * (2 * base + lane);
            near_pages = j < k.hi ? page_at(j) : -1;
        }
        // Rows from hi on are 0, and so are those of pages that are not there, whose F is NaN. The second half lies in the
        // first one's page but for pages of 16.
        X x;
        {
            const int i = 2 * (tile - base), p0 = __builtin_amdgcn_readlane(near_pages, i), p1 = __builtin_amdgcn_readlane(near_pages, i + 1);
            const int left = k.hi - jt < KT ? k.hi - jt : KT, at0 = p0 < 0 ? 0 : p0, at1 = p1 < 0 ? 0 : p1;
            int slot = jt & mask, end = slot + left;     // a row of the page, so that end times a row's bytes fits 32 bits
            end = p0 < 0 ? 0 : end <= mask ? end : mask + 1;
            const char *bk = sk.at(at0), *bv = sv.at(at0), *bb = sb.at(at0), *bg = sg.at(at0), *bf = sf.at(at0);
            constexpr int ROWS = 64 / X::CPR, HALF = X::PASS / 2;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                if (kb) {
                    if (mask < 16) {
                        bk = sk.at(at1), bv = sv.at(at1), bb = sb.at(at1), bg = sg.at(at1), bf = sf.at(at1);
                        slot = -16;
                        end = p1 < 0 || left < 16 ? 0 : left - 16;
                    }
                    slot += 16;
                }
                x.k[kb][0] = load_frag<T>(bk, end * sk.row, sk.lane, slot * sk.row);
                x.k[kb][1] = load_frag<T>(bk, end * sk.row, sk.lane, slot * sk.row + 32 * (int)sizeof(T));
                x.b[kb] = load_frag<T>(bb, end * sb.row, sb.lane, slot * sb.row);
                x.g[kb] = load_at<float>(bg, end * sg.row, sg.lane, slot * sg.row);
                x.f[kb] = load_at<float>(bf, has_f ? end * sf.row : 0, sf.lane, slot * sf.row);
#pragma unroll
                for (int r = 0; r < HALF; ++r) x.v[HALF * kb + r] = load_at<u32x4>(bv, end * sv.row, sv.lane, (slot + ROWS * r) * sv.row);
            }
            if (p0 < 0) x.f[0] = __builtin_nanf("");
            if (p1 < 0) x.f[1] = __builtin_nanf("");
        }
        if (tile == t.from) {                            // the first loads are under way: what has come of the query rows
            lim = len < 0 || len > max_len || len > held ? -1 : len > back ? len - back : 0;
            lim = lim < k.hi ? lim : k.hi;
            least = lim < 0 ? k.hi : lim;                // the join answers for rows that see nothing defined
            if (lc >= k.rows) lim = 0, least = k.hi, gq = -__builtin_inff();
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) {
                const int y = __shfl_xor(least, d);
                least = y < least ? y : least;
            }
            least = __builtin_amdgcn_readfirstlane(least);
        }
        const bool mixed = jt + KT > least || jt < k.lo;               // some row does not see all of the tile
        if (mixed) {
            // Values that are not finite, at positions that some row does not see: 0 in the product (0 times them would be
            // NaN there), and added to the rows that see them at the end. An exponent of ones carries into the sign's place.
            unsigned ones = 0;
#pragma unroll
            for (int i = 0; i < X::PASS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) ones |= (x.v[i][e] & EXPONENT<T>) + EXPONENT_ONE<T>;
            if (__ballot((ones & SIGN<T>) != 0)) {
                odd = true;
#pragma unroll
                for (int i = 0; i < X::PASS; ++i) {
                    T e[X::E];
                    __builtin_memcpy(e, &x.v[i], 16);
#pragma unroll
                    for (int j = 0; j < X::E; ++j) {
                        const float y = (float)e[j];
                        if (!(y - y == 0.f)) e[j] = (T)0.f;
                    }
                    __builtin_memcpy(&x.v[i], e, 16);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < X::PASS; ++i)
            *reinterpret_cast<u32x4*>(sm.v + toff<T, DH>((64 * i + lane) / X::CPR, lane % X::CPR)) = x.v[i];
        // Where every row sees the tile: exp(g_m - g_j) as exp(g_m - g_e) exp(g_e - g_j) and F_m - F_j as (F_m - F_e) +
        // (F_e - F_j), e the tile's last position, one factor a row and one a position. Both are at most 1 where g falls;
        // where it rises too far for them, or F_e is not finite, the tile is taken pair by pair.
        const float ge = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x.g[1]), 15));
        const float fe = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x.f[1]), 15));
        const float d0 = (ge - x.g[0]) * LOG2E, d1 = (ge - x.g[1]) * LOG2E, dq = (gq - ge) * LOG2E;
        const bool near = fabsf(d0) <= FACTORED && fabsf(d1) <= FACTORED && dq <= FACTORED && fe - fe == 0.f;
        const bool fast = !mixed && __ballot(!near) == 0;
        if (grp == 0) {
            sm.g[lc] = fast ? fast_exp2(d0) : x.g[0];
            sm.g[16 + lc] = fast ? fast_exp2(d1) : x.g[1];
            sm.f[lc] = fast ? (fe - x.f[0]) * LOG2E : x.f[0];
            sm.f[16 + lc] = fast ? (fe - x.f[1]) * LOG2E : x.f[1];
        }
        f32x4 s[2], cb[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            s[kb] = mma(x.k[kb][1], q[1], mma(x.k[kb][0], q[0], zero4()));
            cb[kb] = mma(x.b[kb], c, zero4());
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float more = 0.f;                                // to be added to the scores
        if (fast) {
            more = (fq - fe) * LOG2E;
            const float rowf = lam * fast_exp2(dq);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const f32x4 gk = lds4f(sm.g + 16 * kb + 4 * grp), fk = lds4f(sm.f + 16 * kb + 4 * grp);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[kb][e] = fmaf(cb[kb][e] * gk[e], rowf, fmaf(s[kb][e], 0.125f * LOG2E, fk[e]));
            }
        } else {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const f32x4 gk = lds4f(sm.g + 16 * kb + 4 * grp), fk = lds4f(sm.f + 16 * kb + 4 * grp);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = jt + 16 * kb + 4 * grp + e;
                    const float dec = lam * fast_exp2((gq - gk[e]) * LOG2E);
                    s[kb][e] = fmaf(fq - fk[e], LOG2E, fmaf(s[kb][e], 0.125f * LOG2E, dec * cb[kb][e]));
                    s[kb][e] = j >= k.lo && j < lim ? s[kb][e] : -__builtin_inff();
                }
            }
        }
        f32x4 p[2];
        float sum;
        auto weights = [&]() {
            const float off = more - m2 + UP<T>;
            sum = 0.f;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[kb][e] = fast_exp2(s[kb][e] + off);
                    sum += p[kb][e];
                }
        };
        weights();
        const bool over = sum > __builtin_exp2f(RAISE + UP<T>);
        if (__ballot(over)) {
            float mx = -__builtin_inff();
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[kb][e]);
            mx = group_max(mx) + more;
            const float to = group_max(over ? 1.f : 0.f) > 0.f ? fmaxf(m2, mx) : m2, corr = fast_exp2(m2 - to);
            m2 = to;
            l *= corr;
#pragma unroll
            for (int db = 0; db < 4; ++db) o[db] *= corr;
            weights();
        }
        l += sum;
#pragma unroll
        for (int i = 0; i < Split<T>::terms; ++i) {
            const frag8<T> pf = pack8<T>(p[0], p[1]);
#pragma unroll
            for (int db = 0; db < 4; ++db) o[db] = mma(frag_tr<T, DH>(sm.v, 16 * db, 0, lane), pf, o[db]);
            if (i + 1 < Split<T>::terms) {
                const f32x8 back = __builtin_convertvector(pf, f32x8);
#pragma unroll
                for (int e = 0; e < 4; ++e) p[0][e] -= back[e], p[1][e] -= back[4 + e];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();                 // the tile has been read
    }
    if (odd) {
        const int from = t.from * KT > k.lo ? t.from * KT : k.lo, to = t.to * KT < k.hi ? t.to * KT : k.hi;
        for (int j = from; j < to; ++j) {
            if ((j / KT + 1) * KT <= least && j / KT * KT >= k.lo) continue;       // its tile was taken whole
            const int page = page_at(j);
            if (page < 0) continue;
            const T* v = (const T*)(sv.at(page) + (j & mask) * sv.row) + 4 * grp;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = (float)v[16 * db + e];
                    if (!(y - y == 0.f) && j < lim) o[db][e] += y;
                }
        }
    }
    l = group_sum(l);
    f32x2 *const stat = AGAIN(ws.stat), *const own_stat = AGAIN(ws.own_stat);
    float *const part = AGAIN(ws.part), *const own_part = AGAIN(ws.own);
    const unsigned own_rows = AGAIN(plan.own_rows), own_items = AGAIN(plan.own_items), items = AGAIN(plan.items);
    // a row's output and sum, where no other wave of the workgroup has it
    auto alone = [&](f32x2* to_stat, float* to_part, int64_t r) {
        if (lc >= k.rows) return;
        if (grp == 0) to_stat[r] = f32x2{m2 - UP<T>, l};
#pragma unroll
        for (int db = 0; db < 4; ++db) *reinterpret_cast<f32x4*>(to_part + r * DH + 16 * db + 4 * grp) = o[db];
    };
    if (own) {
        alone(own_stat, own_part, ((int64_t)k.h * own_items + item) * own_rows + lc);
        return;
    }
    const int64_t to = ((int64_t)k.h * items + item) << log_per;
    if (log_rw == 2) {
        alone(stat, part, to + 16 * w + lc);
        return;
    }
    // the parts of the waves that have the same rows (every rw-th) joined, in order
    if (grp == 0) ms[w][lc] = m2 - UP<T>, ls[w][lc] = l;
    __syncthreads();
    const int g0 = w & (rw - 1);
    float cm = ms[g0][lc];
    for (int i = g0 + rw; i < NW; i += rw) cm = fmaxf(cm, ms[i][lc]);
    const float mine = fast_exp2(m2 - UP<T> - cm);
#pragma unroll
    for (int db = 0; db < 4; ++db) *reinterpret_cast<f32x4*>(&os[w][lc][16 * db + 4 * grp]) = o[db] * mine;
    if (w < rw && grp == 0 && lc < k.rows) {
        float cl = 0.f;
        for (int i = g0; i < NW; i += rw) cl = fmaf(ls[i][lc], fast_exp2(ms[i][lc] - cm), cl);
        stat[to + 16 * w + lc] = f32x2{cm, cl};
    }
    __syncthreads();
    static_assert(64 * NW == 16 * (DH / 4), "a thread per row of 16 and 4 features");
    const int rr = tid / (DH / 4), d = 4 * (tid % (DH / 4));
    for (int g = 0; g < rw; ++g) {
        f32x4 y = lds4f(&os[g][rr][d]);
        for (int i = g + rw; i < NW; i += rw) y += lds4f(&os[i][rr][d]);
        *reinterpret_cast<f32x4*>(part + (to + 16 * g + rr) * DH + d) = y;
    }
}

// The join of a row's parts by WPR waves: lane i has part i's reference and sum, the common parts' and the own ones'; the
// outputs follow eight at a time, in order.
template <class TO, int WPR>
__global__ __launch_bounds__(64 * NW) void prefix_join_kernel(sisa_prefix_decode_args a, Plan plan, int shift, int log_per,
                                                              const f32x2* stat, const float* part, const f32x2* own_stat,
                                                              const float* own) {
    __shared__ float os[NW][DH];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned H = a.pool.heads, M = a.M, per = 1u << log_per;
    const unsigned row = blockIdx.x * (NW / WPR) + w / WPR;
    if (WPR == 1 && row >= (unsigned)a.B * H * M) return;
    const unsigned nh = M == 1 ? row : row / M, m = row - nh * M, n = nh / H, h = nh - n * H;
    const int64_t held = (int64_t)a.W << shift;
    TO* out = (TO*)a.out.ptr + n * a.out.sb + h * a.out.sh + m * a.out.sl + lane;
    const int r = a.group[n], vis = visible(a, held, n, m), last = (m | 15) < M ? m | 15 : M - 1;
    const int end = visible(a, held, n, last);
    int lo = -1, f0 = 0, f1 = 0;
    int64_t tile = -1;
    if (r >= 0 && r < a.G) {
        lo = common(a, held, r), f0 = a.first[r], f1 = a.first[r + 1];
        tile = tile_base(a, r, log_per);
    }
    const int64_t mine = (int64_t)((int)n - f0) * M + m;
    tile += mine >> log_per;
    if (vis < 0 || lo < 0 || f0 < 0 || f1 > a.B || (int)n < f0 || (int)n >= f1 || (lo > 0 && (tile < 0 || tile >= plan.tiles))) {
        if (w % WPR == 0) *out = cvt<TO>(__builtin_nanf(""));
        return;
    }
    // parts of `each` of n tiles from `first` on that hold something that the row sees
    auto active = [&](int n, int each, int first) {
        const int seen = (vis + KT - 1) / KT - first, upto = seen < n ? seen : n;
        return upto <= 0 ? 0 : (int)((unsigned)(upto + each - 1) / (unsigned)each);
    };
    auto each_of = [](int n, unsigned parts) { return (int)(((unsigned)n + parts - 1) / parts); };
    const int first = lo / KT, tiles = (lo + KT - 1) / KT, own_tiles = (end + KT - 1) / KT - first;
    const int kw = NW << 4 >> log_per, nc = active(tiles, kw * each_of(tiles, plan.parts * kw), 0);
    const int no = vis > lo ? active(own_tiles, each_of(own_tiles, plan.own_parts), first) : 0;
    const int64_t at = (((int64_t)h * plan.items + tile * plan.parts) << log_per) + (mine & (per - 1)), step = per;
    const int64_t own_at = ((int64_t)h * plan.own_items + (int64_t)n * plan.own_tiles + (m >> 4)) * plan.own_rows + (m & 15),
                  own_step = (int64_t)a.B * plan.own_tiles * plan.own_rows;
    const f32x2 s0 = lane < nc ? stat[at + lane * step] : f32x2{LEAST, 0.f};
    const f32x2 s1 = lane < no ? own_stat[own_at + lane * own_step] : f32x2{LEAST, 0.f};
    float mx = fmaxf(s0[0], s1[0]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    auto factor = [&](float y) { return fast_exp2(y - mx); };
    const float x0 = factor(s0[0]), x1 = factor(s1[0]);
    float l = fmaf(s0[1], x0, s1[1] * x1);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
    float o = 0.f;
    auto add = [&](int count, float factors, const float* from, int64_t step) {
        constexpr int AHEAD = 8;
        for (int c0 = w % WPR; c0 < count; c0 += WPR * AHEAD) {
            float y[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int c = c0 + WPR * i < count ? c0 + WPR * i : count - 1;
                y[i] = from[c * step * DH + lane];
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int c = c0 + WPR * i;
                if (c < count) o = fmaf(y[i], __int_as_float(__builtin_amdgcn_readlane(__float_as_int(factors), c)), o);
            }
        }
    };
    add(nc, x0, part + at * DH, step);
    add(no, x1, own + own_at * DH, own_step);
    if constexpr (WPR > 1) {
        os[w][lane] = o;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int i = 1; i < WPR; ++i) o += os[i][lane];
    }
    *out = cvt<TO>(vis == 0 ? 0.f : o / l);
}

Plan plan_of(int64_t B, int64_t H, int64_t M, int64_t G, int64_t max_len, int64_t max_shared) {
    Plan p{};
    const int64_t rows = sisa::cdiv(B, G) * M;           // of a group, on average
    p.log_rw = rows <= 16 ? 0 : rows <= 32 ? 1 : 2;
    const int64_t per = (int64_t)16 << p.log_rw;
    p.tiles = (unsigned)(max_shared > 0 ? G - 1 + sisa::cdiv(B * M, per) : 0);
    p.own_tiles = (unsigned)sisa::cdiv(M, 16);
    p.own_rows = (unsigned)(M < 16 ? M : 16);
    // As many parts as fill the chip while a wave keeps a tile, or, for longer ranges, more of them of twelve tiles to a wave,
    // which even out: `few` and `many` workgroups, or waves, in all. us of the first launch with `few` alone / `many` alone /
    // the larger of both: 16 rows of 2,000 common positions of 12 heads 9.9 / 17.5 / 10.7, 64 of 16,384 33 / 34 / 34, 24 x 8
    // drafts of up to 6,000 53 / 40 / 40, 256 rows of 1,500 and up to 1,000 of their own 69 / 49 / 52.
    auto parts = [](int64_t items, int64_t positions, int64_t tile, int64_t few, int64_t many) {
        auto of = [&](int64_t total, int64_t each) {
            const int64_t most = sisa::cdiv(positions, each), want = items > 0 ? sisa::cdiv(total, items) : 1;
            return want < most ? want : most;
        };
        const int64_t a = of(few, tile), b = of(many, 12 * tile), n = a > b ? a : b;
        return (unsigned)(n < 1 ? 1 : n > MOST ? MOST : n);
    };
    p.parts = parts(p.tiles * H, max_shared, KT * NW >> p.log_rw, 512, 2048);
    p.own_parts = parts(B * p.own_tiles * H, max_len, KT, 2048, 16384);
    p.items = p.parts * p.tiles;
    p.own_items = (unsigned)(p.own_parts * B * p.own_tiles);
    p.blocks = (unsigned)(H * p.items);
    return p;
}

Space space_of(char* base, const Plan& p, int64_t H) {
    const int64_t rows = H * p.items * 16 << p.log_rw, own = H * p.own_items * p.own_rows;
    Space s{};
    char* at = base;
    auto take = [&](int64_t bytes) {
        char* x = at;
        at += (bytes + 255) / 256 * 256;
        return x;
    };
    s.stat = (f32x2*)take(rows * 8);
    s.own_stat = (f32x2*)take(own * 8);
    s.part = (float*)take(rows * DH * 4);
    s.own = (float*)take(own * DH * 4);
    s.bytes = at - base;
    return s;
}

int64_t workgroups(const Plan& p, int64_t H) { return H * p.items + sisa::cdiv(H * p.own_items, NW); }

template <class T, class TO>
int launch_join(const sisa_prefix_decode_args* a, const Plan& p, int shift, const Space& ws, hipStream_t st) {
    const int64_t rows = (int64_t)a->B * a->pool.heads * a->M;
    const int log_per = 4 + p.log_rw;
    if (rows < 2048)
        prefix_join_kernel<TO, NW><<<(unsigned)rows, 64 * NW, 0, st>>>(*a, p, shift, log_per, ws.stat, ws.part, ws.own_stat, ws.own);
    else prefix_join_kernel<TO, 1><<<(unsigned)sisa::cdiv(rows, NW), 64 * NW, 0, st>>>(*a, p, shift, log_per, ws.stat, ws.part, ws.own_stat, ws.own);
    return sisa::launch_status("sisa_prefix_decode (join)");
}

template <class T>
int launch(const sisa_prefix_decode_args* a, const Plan& p, hipStream_t st) {
    const int shift = sisa::log2_of(a->pool.page_size);
    const Space ws = space_of((char*)a->workspace, p, a->pool.heads);
    const unsigned grid = (unsigned)workgroups(p, a->pool.heads);
    prefix_part_kernel<T><<<grid, 64 * NW, 0, st>>>(PartArgs{*a, p, shift, ws});
    const int rc = sisa::launch_status("sisa_prefix_decode");
    if (rc) return rc;
    return a->out_dtype == SISA_F32 ? launch_join<T, float>(a, p, shift, ws, st) : launch_join<T, T>(a, p, shift, ws, st);
}

bool sizes_ok(int64_t B, int64_t H, int64_t M, int64_t G, int64_t max_len, int64_t max_shared) {
    return B >= 1 && H >= 1 && M >= 1 && G >= 1 && G <= B && max_len >= 1 && max_len <= (1 << 30) && max_shared >= 0 &&
           max_shared <= (1 << 30) && B * M <= (1 << 28) / H;
}

}  // namespace

extern "C" int64_t sisa_prefix_decode_workspace_bytes(int32_t B, int32_t H, int32_t M, int32_t G, int32_t max_len,
                                                      int32_t max_shared) {
    if (!sizes_ok(B, H, M, G, max_len, max_shared)) return 0;
    return space_of(nullptr, plan_of(B, H, M, G, max_len, max_shared), H).bytes;
}

extern "C" int sisa_prefix_decode(const sisa_prefix_decode_args* a, void* stream) {
    SISA_REQUIRE(a != nullptr, "sisa_prefix_decode: null args");
    SISA_REQUIRE_POOL("sisa_prefix_decode", a->pool);
    if (a->B == 0) return SISA_OK;
    const int64_t held = (int64_t)a->W * a->pool.page_size;
    SISA_REQUIRE(a->W >= 1 && sizes_ok(a->B, a->pool.heads, a->M, a->G, a->max_len, a->max_shared) && a->max_len <= held &&
                     a->max_shared <= held,
                 "sisa_prefix_decode: bad shape B=%d M=%d W=%d G=%d max_len=%d max_shared=%d (1 to B groups; at most W pages of "
                 "%d, and 2^30 positions; B*M*H at most 2^28)",
                 a->B, a->M, a->W, a->G, a->max_len, a->max_shared, a->pool.page_size);
    SISA_REQUIRE(a->table && a->lengths && a->first && a->group && a->shared && a->lam && a->out.ptr,
                 "sisa_prefix_decode: null pointer");
    SISA_REQUIRE(a->workspace && sisa::aligned16(a->workspace), "sisa_prefix_decode: null workspace, or not 16-byte aligned");
    SISA_REQUIRE(a->out_dtype == SISA_F32 || a->out_dtype == a->pool.dtype, "sisa_prefix_decode: out_dtype");
    SISA_REQUIRE_NEAR_ROWS("sisa_prefix_decode", a->pool);
    SISA_REQUIRE(sisa::view_ok(a->q, a->pool.dtype) && sisa::view_ok(a->c, a->pool.dtype),
                 "sisa_prefix_decode: q and c rows must be 16-byte aligned");
    SISA_REQUIRE(a->gq.ptr && (a->fq.ptr == nullptr) == (a->pool.f.ptr == nullptr),
                 "sisa_prefix_decode: gq must be given, and fq where the pool has f");
    const Plan p = plan_of(a->B, a->pool.heads, a->M, a->G, a->max_len, a->max_shared);
    SISA_REQUIRE(workgroups(p, a->pool.heads) * 64 * NW <= sisa::MAX_THREADS && (int64_t)a->B * a->M * a->pool.heads * 64 <= sisa::MAX_THREADS - 64 * NW,
                 "sisa_prefix_decode: too large for one launch");
    hipStream_t st = (hipStream_t)stream;
    switch (a->pool.dtype) {
        case SISA_BF16: return launch<__bf16>(a, p, st);
        case SISA_F16: return launch<_Float16>(a, p, st);
        default: return launch<float>(a, p, st);
    }
}
