// Attention of the new positions of sequences that share their first positions, for gfx950 (include/sisa_hip_branch.h).
//
//   s_mj = q_m.k_j / 8 + lam exp(g_m - g_j) (c_m.b_j) + (F_m - F_j);   out_m = softmax_j(s_mj) v_j
//
// The softmax over a sequence's positions is joined from its parts: the common positions, which the query rows of a group see
// alike and which are read once for 16 NR of them, and its own. Both parts are the same work: up to 16 NR query rows against
// a range of positions in the pages of one table row, 32 positions (a tile) of a wave at a time on the matrix cores.
//
// Scores are computed transposed (S^T = K Q^T), so that a lane has one query row's softmax and the weights are the operand of
// O^T += V^T P^T as they are. K and b~ go from memory to the operand registers, each used by one wave only; v passes through
// LDS, which transposes it. The weights enter their product as a sum of two (fp16) or three (bf16) operands, so that the
// result is an fp32 one: rounded once to bf16 they would be off by 2^-9.
#include "pages.h"
#include "sisa_hip_branch.h"

namespace {

constexpr int DH = 64, DS = 32;
constexpr int KT = 32;                // positions of a tile
constexpr int NW = 4;                 // waves of a workgroup
constexpr int MOST = 64;              // most parts of a range: the join has a lane for each

// How a call is cut into workgroups: the query rows of all groups into tiles of 16 NR, a group's common positions into `parts`
// workgroups, a sequence's own ones into `own_parts` waves.
struct Plan {
    int nr;
    unsigned tiles, own_tiles, parts, own_parts, own_rows;
    int64_t items, own_items;         // workgroups, waves
};

// Tile t of all groups' query rows: group r's tiles begin at r + first[r] M / (16 NR), which leaves room for each.
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

// Up to 16 NR query rows, counted from sequence n0's first, against positions lo <= j < hi of a table row.
struct Work {
    int h, n0, r0, rows, lo, hi;
    const int32_t* row;
};

// What a wave loads of a tile: K and b~ as operands, v in 16-byte pieces, g and F of the position lane % 16 of either half.
template <class T>
struct Tile {
    static constexpr int E = 16 / (int)sizeof(T), CPR = DH / E, PASS = KT * CPR / 64;     // elements and pieces of a row
    frag8<T> k[2][2], b[2];
    u32x4 v[PASS];
    float g[2], f[2];
};

// 16-byte loads relative to a scalar base, 0 for the offset NOWHERE.
constexpr int NOWHERE = (int)0x80000000;
template <class V> SISA_DEV V load_at(const char* base, int voff, int soff) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(base, 0x7fffffff);
    if constexpr (sizeof(V) == 4) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b32(r, voff, soff, 0));
    else return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 0));
}
template <class T> SISA_DEV frag8<T> load_frag(const char* base, int voff, int soff) {
    if constexpr (sizeof(T) == 2) return load_at<frag8<T>>(base, voff, soff);
    else return join<T>(load_at<f32x4>(base, voff, soff), load_at<f32x4>(base, voff, soff + 16));
}

// A wave's view of the positions of one head: where the 16 from 16 i on begin in each tensor (lane i % 64), and what a lane
// adds to that.
template <class T>
struct Places {
    const sisa_page_pool* P;
    const int32_t* row;
    int W, shift, h, lo, hi, base;
    int page;                          // of 16-block base + lane; -1: none of the pool's
    int64_t k, v, b, g, f;
    int ok, ov, ob, og, of;            // byte offsets of the lane in a block of 16 positions

    SISA_DEV void init(const sisa_page_pool& pool, const Work& w, int W_, int shift_, int lane) {
        constexpr int es = sizeof(T);
        P = &pool;
        row = w.row, W = W_, shift = shift_, h = w.h, lo = w.lo, hi = w.hi;
        const int grp = lane >> 4, lc = lane & 15, ch = lane % Tile<T>::CPR, r = lane / Tile<T>::CPR;
        ok = (lc * (int)pool.k.sl + 8 * grp) * es;
        ob = (lc * (int)pool.b.sl + 8 * grp) * es;
        ov = (r * (int)pool.v.sl + Tile<T>::E * ch) * es;
        og = lc * (int)pool.g.sl * 4;
        of = lc * (int)pool.f.sl * 4;
    }
    SISA_DEV void look_up(int tile, int lane) {
        constexpr int es = sizeof(T);
        base = 2 * tile;
        const int j = 16 * (base + lane), slot = j & (P->page_size - 1);
        page = j < hi ? page_of(row, W, shift, P->pages, j) : -1;
        const int64_t at = page < 0 ? 0 : page;
        auto place = [&](const sisa_view& x, int size) { return (at * x.sb + h * x.sh + slot * x.sl) * size; };
        k = place(P->k, es);
        v = place(P->v, es);
        b = place(P->b, es);
        g = place(P->g, 4);
        f = place(P->f, 4);
    }
    SISA_DEV static const char* at(const void* p, int64_t place, int i) {
        const unsigned lo = __builtin_amdgcn_readlane((int)place, i), hi = __builtin_amdgcn_readlane((int)(place >> 32), i);
        return (const char*)p + (int64_t)((uint64_t)hi << 32 | lo);
    }
    // The tile of positions 32 tile ..
    SISA_DEV void load(int tile, int lane, Tile<T>& x) {
        if (2 * tile - base >= 64) look_up(tile, lane);
        const int lc = lane & 15, r = lane / Tile<T>::CPR;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int i = 2 * tile + kb - base, j0 = 16 * (2 * tile + kb);
            const bool there = __builtin_amdgcn_readlane(page, i) >= 0;
            const char *pk = at(P->k.ptr, k, i), *pv = at(P->v.ptr, v, i), *pb = at(P->b.ptr, b, i), *pg = at(P->g.ptr, g, i),
                       *pf = at(P->f.ptr, f, i);
            const bool in = there && j0 + lc >= lo && j0 + lc < hi;
            const int vk = in ? ok : NOWHERE, vb = in ? ob : NOWHERE;
            x.k[kb][0] = load_frag<T>(pk, vk, 0);
            x.k[kb][1] = load_frag<T>(pk, vk, 32 * (int)sizeof(T));
            x.b[kb] = load_frag<T>(pb, vb, 0);
            x.g[kb] = load_at<float>(pg, in ? og : NOWHERE, 0);
            x.f[kb] = load_at<float>(pf, in && P->f.ptr ? of : NOWHERE, 0);
            if (!there) x.f[kb] = __builtin_nanf("");
            constexpr int HALF = Tile<T>::PASS / 2, ROWS = 64 / Tile<T>::CPR;
#pragma unroll
            for (int p = 0; p < HALF; ++p) {
                const int jv = j0 + ROWS * p + r;
                x.v[HALF * kb + p] = load_at<u32x4>(pv, there && jv >= lo && jv < hi ? ov : NOWHERE,
                                                    ROWS * p * (int)P->v.sl * (int)sizeof(T));
            }
        }
    }
};

// The workgroups of the common parts, then those of the own ones, whose waves are on their own. Unnormalised outputs go to
// `part`, 16 NR rows an item, and `own`; each row's reference (log2) and sum to `stat` and `own_stat`.
template <class T, int NR>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2))) void prefix_part_kernel(sisa_prefix_decode_args a, Plan plan, int shift, f32x2* stat,
                                                              float* part, f32x2* own_stat, float* own_part) {
    constexpr int PER = 16 * NR, LOG = NR == 1 ? 4 : NR == 2 ? 5 : 6, LD = DH + 4;
    __shared__ WaveLds<T> lds[NW];
    __shared__ __attribute__((aligned(16))) float ms[NW][PER], ls[NW][PER], os[NW][16][LD];
    const int tid = threadIdx.x, lane = tid & 63, grp = lane >> 4, lc = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool own = blockIdx.x >= (unsigned)plan.items;
    const int64_t held = (int64_t)a.W << shift;
    const unsigned H = a.pool.heads;
    unsigned item = own ? (blockIdx.x - (unsigned)plan.items) * NW + w : blockIdx.x;
    Work k;
    Range t;                                             // the wave's tiles
    if (own) {
        if (item >= plan.own_items) return;
        const unsigned nm = item / H, pn = plan.own_tiles == 1 ? nm : nm / plan.own_tiles, p = pn / (unsigned)a.B, n = pn - p * a.B;
        k.h = item - nm * H;
        k.n0 = n;
        k.r0 = 16 * (nm - pn * plan.own_tiles);
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
        const unsigned ph = item / plan.tiles, tile = item - ph * plan.tiles, p = ph / H;
        k.h = ph - p * H;
        int r = 0;                                       // the last group whose tiles begin at or before this one
        if (a.G > 1) {
            r = -1;
            for (int i = 0; i < a.G; i += 64) r += __popcll(__ballot(i + lane < a.G && tile_base(a, i + lane, LOG) <= tile));
            if (r < 0) return;
        }
        const int f0 = a.first[r], f1 = a.first[r + 1];
        k.hi = common(a, held, r);
        if (f0 < 0 || f1 > a.B || f1 <= f0 || k.hi <= 0) return;
        const int64_t all = (int64_t)(f1 - f0) * a.M, nth = (int64_t)tile - tile_base(a, r, LOG), at = nth * PER;
        if (nth < 0 || at >= all) return;
        k.n0 = f0;
        k.r0 = at;
        k.rows = all - at < PER ? all - at : PER;
        k.lo = 0;
        const int n = (k.hi + KT - 1) / KT;
        if (part_of(n, plan.parts * NW, p * NW).from >= n) return;
        t = part_of(n, plan.parts * NW, p * NW + w);
    }
    k.row = a.table + k.n0 * a.s_table;
    const int nr = (k.rows + 15) >> 4;
    Places<T> at;
    at.init(a.pool, k, a.W, shift, lane);
    at.look_up(t.from, lane);

    // Query rows: lane i finds row i's; column lc of each group of 16 is a lane's, in all four groups of lanes.
    frag8<T> q[NR][2], c[NR];
    float gq[NR], fq[NR], m2[NR], l[NR];                 // l: the lane's part
    int lim[NR];                                         // positions below it are seen
    f32x4 o[NR][4];                                      // output features 16 db + 4 grp + i
    int least = k.hi;                                    // every row sees what lies before it
    {
        int n = k.n0, m = k.r0 + lane, seen = 0;
        if (!own) {
            const unsigned d = a.M == 1 ? m : (unsigned)m / (unsigned)a.M;
            n += d;
            m -= d * a.M;
        }
        float g = 0.f, f = 0.f;
        int64_t pq = 0, pc = 0;
        if (lane < k.rows) {
            g = ((const float*)a.gq.ptr)[n * a.gq.sb + k.h * a.gq.sh + m * a.gq.sl];
            if (a.fq.ptr) f = ((const float*)a.fq.ptr)[n * a.fq.sb + k.h * a.fq.sh + m * a.fq.sl];
            pq = n * a.q.sb + k.h * a.q.sh + m * a.q.sl;
            pc = n * a.c.sb + k.h * a.c.sh + m * a.c.sl;
            seen = visible(a, held, n, m);
            seen = seen < k.hi ? seen : k.hi;
            if (seen >= 0) least = seen;                 // the join answers for the others
        }
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) {
            const int y = __shfl_xor(least, s);
            least = y < least ? y : least;
        }
        least = __builtin_amdgcn_readfirstlane(least);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int from = 16 * i + lc;
            gq[i] = __shfl(g, from);
            fq[i] = __shfl(f, from);
            lim[i] = __shfl(seen, from);
            const T *rq = (const T*)a.q.ptr + lane_value(pq, from) + 8 * grp, *rc = (const T*)a.c.ptr + lane_value(pc, from) + 8 * grp;
            q[i][0] = q[i][1] = c[i] = zero8<T>();
            if (from < k.rows) q[i][0] = load8<T>(rq), q[i][1] = load8<T>(rq + 32), c[i] = load8<T>(rc);
            if (from >= k.rows) gq[i] = -__builtin_inff();
            l[i] = 0.f;
            m2[i] = LEAST;
#pragma unroll
            for (int db = 0; db < 4; ++db) o[i][db] = zero4();
        }
    }
    const float lam = a.lam[k.h * a.s_lam] * LOG2E;

    using X = Tile<T>;
    WaveLds<T>& sm = lds[w];
    X x;
    bool odd = false;
    for (int tile = t.from < t.to ? t.from - 1 : t.to; tile < t.to; ++tile) {
        const int jt = tile * KT;
        const bool mixed = jt + KT > least || jt < k.lo;               // some row does not see all of the tile
        frag8<T> kf[2][2], bf[2];
        bool fast = false;
        float ge = 0.f, fe = 0.f;
        if (tile >= t.from) {
            if (mixed) {
                // Values that are not finite, at positions that some row does not see: 0 in the product (0 times them would
                // be NaN there), and added to the rows that see them at the end.
                asm volatile("");      // a branch, not selects
#pragma unroll
                for (int i = 0; i < X::PASS; ++i) {
                    T e[X::E];
                    __builtin_memcpy(e, &x.v[i], 16);
#pragma unroll
                    for (int j = 0; j < X::E; ++j) {
                        const float y = (float)e[j];
                        if (!(y - y == 0.f)) e[j] = (T)0.f, odd = true;
                    }
                    __builtin_memcpy(&x.v[i], e, 16);
                }
            }
#pragma unroll
            for (int i = 0; i < X::PASS; ++i)
                *reinterpret_cast<u32x4*>(sm.v + toff<T, DH>((64 * i + lane) / X::CPR, lane % X::CPR)) = x.v[i];
            // Where every row sees the tile: exp(g_m - g_j) as exp(g_m - g_e) exp(g_e - g_j) and F_m - F_j as (F_m - F_e) +
            // (F_e - F_j), e the tile's last position, one factor a row and one a position. Both are at most 1 where g
            // falls; where it rises too far for them, or F_e is not finite, the tile is taken pair by pair.
            ge = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x.g[1]), 15));
            fe = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x.f[1]), 15));
            const float d0 = (ge - x.g[0]) * LOG2E, d1 = (ge - x.g[1]) * LOG2E;
            bool near = fabsf(d0) <= FACTORED && fabsf(d1) <= FACTORED && fe - fe == 0.f;
#pragma unroll
            for (int g = 0; g < NR; ++g) near = near && (gq[g] - ge) * LOG2E <= FACTORED;
            fast = !mixed && __ballot(!near) == 0;
            if (grp == 0) {
                sm.g[lc] = fast ? fast_exp2(d0) : x.g[0];
                sm.g[16 + lc] = fast ? fast_exp2(d1) : x.g[1];
                sm.f[lc] = fast ? (fe - x.f[0]) * LOG2E : x.f[0];
                sm.f[16 + lc] = fast ? (fe - x.f[1]) * LOG2E : x.f[1];
            }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) kf[kb][0] = x.k[kb][0], kf[kb][1] = x.k[kb][1], bf[kb] = x.b[kb];
        }
        if (tile + 1 < t.to) at.load(tile + 1, lane, x);               // under way meanwhile
        if (tile < t.from) continue;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int g = 0; g < NR; ++g) {
            if (g >= nr) break;
            f32x4 s[2];
            float more = 0.f;                            // to be added to the scores
            f32x4 qk[2], cb[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                qk[kb] = mma(kf[kb][1], q[g][1], mma(kf[kb][0], q[g][0], zero4()));
                cb[kb] = mma(bf[kb], c[g], zero4());
            }
            if (fast) {
                more = (fq[g] - fe) * LOG2E;
                const float rowf = lam * fast_exp2((gq[g] - ge) * LOG2E);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const f32x4 gk = lds4f(sm.g + 16 * kb + 4 * grp), fk = lds4f(sm.f + 16 * kb + 4 * grp);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[kb][e] = fmaf(cb[kb][e] * gk[e], rowf, fmaf(qk[kb][e], 0.125f * LOG2E, fk[e]));
                }
            } else {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const f32x4 gk = lds4f(sm.g + 16 * kb + 4 * grp), fk = lds4f(sm.f + 16 * kb + 4 * grp);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = jt + 16 * kb + 4 * grp + e;
                        const float dec = lam * fast_exp2((gq[g] - gk[e]) * LOG2E);
                        s[kb][e] = fmaf(fq[g] - fk[e], LOG2E, fmaf(qk[kb][e], 0.125f * LOG2E, dec * cb[kb][e]));
                        s[kb][e] = j >= k.lo && j < lim[g] ? s[kb][e] : -__builtin_inff();
                    }
                }
            }
            f32x4 p[2];
            float sum;
            auto weights = [&]() {
                const float off = more - m2[g] + UP<T>;
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
                const float to = group_max(over ? 1.f : 0.f) > 0.f ? fmaxf(m2[g], mx) : m2[g], corr = fast_exp2(m2[g] - to);
                m2[g] = to;
                l[g] *= corr;
#pragma unroll
                for (int db = 0; db < 4; ++db) o[g][db] *= corr;
                weights();
            }
            l[g] += sum;
#pragma unroll
            for (int i = 0; i < Split<T>::terms; ++i) {
                const frag8<T> pf = pack8<T>(p[0], p[1]);
#pragma unroll
                for (int db = 0; db < 4; ++db) o[g][db] = mma(frag_tr<T, DH>(sm.v, 16 * db, 0, lane), pf, o[g][db]);
                if (i + 1 < Split<T>::terms) {
                    const f32x8 back = __builtin_convertvector(pf, f32x8);
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[0][e] -= back[e], p[1][e] -= back[4 + e];
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();                 // the tile has been read
    }
    if (__ballot(odd)) {
        const int from = t.from * KT > k.lo ? t.from * KT : k.lo, to = t.to * KT < k.hi ? t.to * KT : k.hi;
        for (int j = from; j < to; ++j) {
            if ((j / KT + 1) * KT <= least && j / KT * KT >= k.lo) continue;       // its tile was taken whole
            const int page = page_of(k.row, a.W, shift, a.pool.pages, j);
            if (page < 0) continue;
            const T* v = (const T*)a.pool.v.ptr + page * a.pool.v.sb + k.h * a.pool.v.sh + (j & (a.pool.page_size - 1)) * a.pool.v.sl;
#pragma unroll 1
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = (float)v[16 * db + 4 * grp + e];
                    const bool bad = !(y - y == 0.f);
#pragma unroll
                    for (int g = 0; g < NR; ++g)
#pragma unroll
                        for (int d = 0; d < 4; ++d)
                            if (d == db && bad && j < lim[g]) o[g][d][e] += y;
                }
        }
    }

    if (own) {
        const float sum = group_sum(l[0]);
        if (lc >= k.rows) return;
        const int64_t to = (int64_t)item * plan.own_rows + lc;
        if (grp == 0) own_stat[to] = f32x2{m2[0] - UP<T>, sum};
#pragma unroll
        for (int db = 0; db < 4; ++db) *reinterpret_cast<f32x4*>(own_part + to * DH + 16 * db + 4 * grp) = o[0][db];
        return;
    }
    // the waves' parts of common positions joined, in order
#pragma unroll
    for (int g = 0; g < NR; ++g) {
        const float sum = group_sum(l[g]);
        if (grp == 0) ms[w][16 * g + lc] = m2[g] - UP<T>, ls[w][16 * g + lc] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < NR; ++g) {
        if (g >= nr) break;
        const int row = 16 * g + lc;
        float cm = ms[0][row];
#pragma unroll
        for (int i = 1; i < NW; ++i) cm = fmaxf(cm, ms[i][row]);
        auto factor = [&](float y) { return fast_exp2(y - cm); };
        const float mine = factor(ms[w][row]);
#pragma unroll
        for (int db = 0; db < 4; ++db) *reinterpret_cast<f32x4*>(&os[w][lc][16 * db + 4 * grp]) = o[g][db] * mine;
        __syncthreads();
        const int64_t to = (int64_t)item * PER + 16 * g;
        {
            static_assert(64 * NW == 16 * (DH / 4), "a thread per 4 features");
            const int rr = tid / (DH / 4), d = 4 * (tid % (DH / 4));
            f32x4 y = lds4f(&os[0][rr][d]);
#pragma unroll
            for (int i = 1; i < NW; ++i) y += lds4f(&os[i][rr][d]);
            if (16 * g + rr < k.rows) *reinterpret_cast<f32x4*>(part + (to + rr) * DH + d) = y;
        }
        if (w == 0 && grp == 0) {
            float cl = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) cl = fmaf(ls[i][row], factor(ms[i][row]), cl);
            stat[to + lc] = f32x2{cm, cl};
        }
        __syncthreads();
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
    TO* out = (TO*)a.out + (int64_t)row * DH + lane;
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
    const int nc = active(tiles, NW * each_of(tiles, plan.parts * NW), 0);
    const int no = vis > lo ? active(own_tiles, each_of(own_tiles, plan.own_parts), first) : 0;
    const int64_t at = (((int64_t)h * plan.tiles + tile) << log_per) + (mine & (per - 1)), step = ((int64_t)H * plan.tiles) << log_per;
    const int64_t own_at = (((int64_t)n * plan.own_tiles + (m >> 4)) * H + h) * plan.own_rows + (m & 15),
                  own_step = (int64_t)a.B * plan.own_tiles * H * plan.own_rows;
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
    p.nr = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    const int64_t per = 16 * p.nr;
    p.tiles = (unsigned)(max_shared > 0 ? G + B * M / per : 0);
    p.own_tiles = (unsigned)sisa::cdiv(M, 16);
    p.own_rows = (unsigned)(M < 16 ? M : 16);
    auto parts = [](int64_t items, int64_t total, int64_t positions, int64_t each) {
        const int64_t most = sisa::cdiv(positions, each), want = items > 0 ? sisa::cdiv(total, items) : 1;
        const int64_t n = want < most ? want : most;
        return (unsigned)(n < 1 ? 1 : n > MOST ? MOST : n);
    };
    p.parts = parts(p.tiles * H, 1024, max_shared, KT * NW);
    p.own_parts = parts(B * p.own_tiles * H, 4096, max_len, KT);
    p.items = (int64_t)p.parts * p.tiles * H;
    p.own_items = (int64_t)p.own_parts * B * p.own_tiles * H;
    return p;
}

struct Space {
    f32x2 *stat, *own_stat;
    float *part, *own;
    int64_t bytes;
};
Space space_of(char* base, const Plan& p) {
    const int64_t rows = p.items * 16 * p.nr, own = p.own_items * p.own_rows;
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

int64_t workgroups(const Plan& p) { return p.items + sisa::cdiv(p.own_items, NW); }

template <class T, class TO>
int launch_join(const sisa_prefix_decode_args* a, const Plan& p, int shift, const Space& ws, hipStream_t st) {
    const int64_t rows = (int64_t)a->B * a->pool.heads * a->M;
    const int log_per = p.nr == 1 ? 4 : p.nr == 2 ? 5 : 6;
    if (rows < 2048)
        prefix_join_kernel<TO, NW><<<(unsigned)rows, 64 * NW, 0, st>>>(*a, p, shift, log_per, ws.stat, ws.part, ws.own_stat, ws.own);
    else prefix_join_kernel<TO, 1><<<(unsigned)sisa::cdiv(rows, NW), 64 * NW, 0, st>>>(*a, p, shift, log_per, ws.stat, ws.part, ws.own_stat, ws.own);
    return sisa::launch_status("sisa_prefix_decode (join)");
}

template <class T>
int launch(const sisa_prefix_decode_args* a, const Plan& p, hipStream_t st) {
    const int shift = sisa::log2_of(a->pool.page_size);
    const Space ws = space_of((char*)a->workspace, p);
    const unsigned grid = (unsigned)workgroups(p);
    switch (p.nr) {
        case 1: prefix_part_kernel<T, 1><<<grid, 64 * NW, 0, st>>>(*a, p, shift, ws.stat, ws.part, ws.own_stat, ws.own); break;
        case 2: prefix_part_kernel<T, 2><<<grid, 64 * NW, 0, st>>>(*a, p, shift, ws.stat, ws.part, ws.own_stat, ws.own); break;
        default: prefix_part_kernel<T, 4><<<grid, 64 * NW, 0, st>>>(*a, p, shift, ws.stat, ws.part, ws.own_stat, ws.own);
    }
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
    return space_of(nullptr, plan_of(B, H, M, G, max_len, max_shared)).bytes;
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
    SISA_REQUIRE(a->table && a->lengths && a->first && a->group && a->shared && a->lam && a->out,
                 "sisa_prefix_decode: null pointer");
    SISA_REQUIRE(a->workspace && sisa::aligned16(a->workspace), "sisa_prefix_decode: null workspace, or not 16-byte aligned");
    SISA_REQUIRE(a->out_dtype == SISA_F32 || a->out_dtype == a->pool.dtype, "sisa_prefix_decode: out_dtype");
    SISA_REQUIRE(sisa::view_ok(a->q, a->pool.dtype) && sisa::view_ok(a->c, a->pool.dtype),
                 "sisa_prefix_decode: q and c rows must be 16-byte aligned");
    SISA_REQUIRE(a->gq.ptr && (a->fq.ptr == nullptr) == (a->pool.f.ptr == nullptr),
                 "sisa_prefix_decode: gq must be given, and fq where the pool has f");
    const Plan p = plan_of(a->B, a->pool.heads, a->M, a->G, a->max_len, a->max_shared);
    SISA_REQUIRE(workgroups(p) * 64 * NW <= sisa::MAX_THREADS && (int64_t)a->B * a->M * a->pool.heads * 64 <= sisa::MAX_THREADS - 64 * NW,
                 "sisa_prefix_decode: too large for one launch");
    hipStream_t st = (hipStream_t)stream;
    switch (a->pool.dtype) {
        case SISA_BF16: return launch<__bf16>(a, p, st);
        case SISA_F16: return launch<_Float16>(a, p, st);
        default: return launch<float>(a, p, st);
    }
}
