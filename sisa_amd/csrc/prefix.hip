// Attention of the new positions of sequences that share their first positions, for gfx950 (include/sisa_hip_branch.h).
//
//   s_mj = q_m.k_j / 8 + lam exp(g_m - g_j) (c_m.b_j) + (F_m - F_j);   out_m = softmax_j(s_mj) v_j
//
// The softmax over a sequence's positions is joined from its parts: the common positions, which the query rows of a group see
// alike and which are read once for 16 NR of them, and its own. Both parts are the same work: up to 16 NR query rows against
// a range of positions in the pages of one table row.
#include "pages.h"
#include "sisa_hip_branch.h"

namespace {

constexpr int DH = 64, DS = 32;
constexpr int KT = 32;                // positions of a wave's tile
constexpr int NW = 4;                 // waves of a workgroup, each with its own tiles
constexpr int SPLITS = 64;            // most parts of a range

// How a call is cut into workgroups: NR row groups of 16 to a tile of query rows, the tiles of all groups, the parts of a
// common range and of a sequence's own.
struct Plan {
    int nr, tiles, own_tiles, parts, own_parts;
    int64_t items, own_items;         // workgroups
};

// Tile t of all groups' query rows: group r's tiles begin at r + first[r] M / (16 NR), which leaves room for each.
SISA_DEV int64_t tile_base(const sisa_prefix_decode_args& a, int r, int per) {
    const int64_t n = a.first[r];
    return r + (n < 0 ? 0 : n > a.B ? a.B : n) * a.M / per;
}

// The tiles of KT positions that part p of a range of n tiles has: [from, to).
struct Range { int from, to; };
SISA_DEV Range part_of(int n, int parts, int p) {
    const int each = (n + parts - 1) / parts;
    const int from = each * p;
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

template <class T> struct Split;      // weights as a sum of operands: what is left of 24 bits is not seen in an fp32 sum
template <> struct Split<__bf16> { static constexpr int terms = 3; };
template <> struct Split<_Float16> { static constexpr int terms = 2; };
template <> struct Split<float> { static constexpr int terms = 1; };

template <class T, int NR>
struct __attribute__((aligned(16))) Lds {
    T v[NW][KT * DH];
    float g[NW][KT], f[NW][KT];
    float o[NW][16][DH + 4];
    float m[NW][16 * NR], l[NW][16 * NR];
};

// A workgroup of `items` common parts, then of own ones. part: unnormalised outputs (16 NR, 64) an item, stat: the row's
// reference (log2) and sum.
template <class T, int NR>
__global__ __launch_bounds__(64 * NW) void prefix_part_kernel(sisa_prefix_decode_args a, Plan plan, int shift, f32x2* stat,
                                                              float* part) {
    constexpr int PER = 16 * NR;
    __shared__ Lds<T, NR> sm;
    const int tid = threadIdx.x, lane = tid & 63, grp = lane >> 4, lc = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const sisa_page_pool& P = a.pool;
    const int H = P.heads, M = a.M;
    const int64_t held = (int64_t)a.W << shift;
    const int item = blockIdx.x;
    const bool own = item >= plan.items;
    int64_t i = own ? item - plan.items : item;
    const int h = i % H;
    i /= H;
    // query rows: r0 .. r0 + rows - 1 counted from sequence n0's first
    int n0, r0, rows, lo, hi;
    Range tiles;
    if (own) {
        const int mt = i % plan.own_tiles, n = i / plan.own_tiles % a.B, p = i / plan.own_tiles / a.B;
        const int r = a.group[n];
        if (r < 0 || r >= a.G) return;
        n0 = n;
        r0 = mt * PER;
        rows = M - r0 < PER ? M - r0 : PER;
        lo = common(a, held, r);
        hi = visible(a, held, n, r0 + rows - 1);
        if (lo < 0 || hi <= lo) return;
        const int first = lo / KT;
        tiles = part_of((hi + KT - 1) / KT - first, plan.own_parts, p);
        tiles.from += first;
        tiles.to += first;
    } else {
        const int tile = i % plan.tiles, p = i / plan.tiles;
        int r = -1;                                      // the last group whose tiles begin at or before this one
        for (int k = 0; k < a.G; k += 64) {
            const bool before = k + lane < a.G && tile_base(a, k + lane, PER) <= tile;
            r += __popcll(__ballot(before));
        }
        if (r < 0) return;
        const int f0 = a.first[r], f1 = a.first[r + 1];
        if (f0 < 0 || f1 > a.B || f1 <= f0) return;
        const int64_t all = (int64_t)(f1 - f0) * M, at = (int64_t)(tile - tile_base(a, r, PER)) * PER;
        if (at >= all) return;
        n0 = f0;
        r0 = at;
        rows = all - at < PER ? all - at : PER;
        lo = 0;
        hi = common(a, held, r);
        if (hi <= 0) return;
        tiles = part_of((hi + KT - 1) / KT, plan.parts, p);
    }
    if (tiles.from >= tiles.to) return;
    const int nr = (rows + 15) / 16;
    const int32_t* row = a.table + n0 * a.s_table;

    // the lane's query rows (column lc of each group of 16)
    frag8<T> qf[NR][2], cf[NR];
    float gq[NR], fq[NR], m2[NR], l[NR];
    int lim[NR];                                         // positions below it are seen
    f32x4 acc[NR][4];
    const bool has_f = P.f.ptr != nullptr;
    const float lam = a.lam[h * a.s_lam] * LOG2E;
    int least = hi;
#pragma unroll
    for (int g = 0; g < NR; ++g) {
        const int at = 16 * g + lc;
        const bool ok = at < rows;
        const int64_t n = n0 + (r0 + at) / M, m = (r0 + at) % M;
        qf[g][0] = qf[g][1] = cf[g] = zero8<T>();
        gq[g] = fq[g] = l[g] = 0.f;
        lim[g] = 0;
        m2[g] = -__builtin_inff();
        if (ok) {
            const T* q = (const T*)a.q.ptr + n * a.q.sb + h * a.q.sh + m * a.q.sl;
            qf[g][0] = load8<T>(q + 8 * grp);
            qf[g][1] = load8<T>(q + 32 + 8 * grp);
            cf[g] = load8<T>((const T*)a.c.ptr + n * a.c.sb + h * a.c.sh + m * a.c.sl + 8 * grp);
            gq[g] = ((const float*)a.gq.ptr)[n * a.gq.sb + h * a.gq.sh + m * a.gq.sl];
            if (has_f) fq[g] = ((const float*)a.fq.ptr)[n * a.fq.sb + h * a.fq.sh + m * a.fq.sl];
            const int vis = visible(a, held, n, m);
            lim[g] = vis < hi ? vis : hi;
            least = lim[g] < least ? lim[g] : least;
        }
#pragma unroll
        for (int db = 0; db < 4; ++db) acc[g][db] = zero4();
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        const int x = __shfl_xor(least, o);
        least = x < least ? x : least;
    }
    // every row of the tile sees the positions from lo to before `least`
    least = __builtin_amdgcn_readfirstlane(least);

    T* vs = sm.v[w];
    float *gs = sm.g[w], *fs = sm.f[w];
    for (int t = tiles.from + w; t < tiles.to; t += NW) {
        const int jt = t * KT;
        // 16 neighbours lie in one page
        int page[2];
        int64_t slot[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int j = jt + 16 * kb;
            page[kb] = j < hi ? page_of(row, a.W, shift, P.pages, j) : -1;
            slot[kb] = j & (P.page_size - 1);
        }
        const bool mixed = jt + KT > least;              // some row does not see all of the tile's positions below hi
        frag8<T> kf[2][2], bf[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int j = jt + 16 * kb + lc;
            kf[kb][0] = kf[kb][1] = bf[kb] = zero8<T>();
            if (page[kb] >= 0 && j >= lo && j < hi) {
                const T* k = (const T*)P.k.ptr + page[kb] * P.k.sb + h * P.k.sh + (slot[kb] + lc) * P.k.sl;
                kf[kb][0] = load8<T>(k + 8 * grp);
                kf[kb][1] = load8<T>(k + 32 + 8 * grp);
                bf[kb] = load8<T>((const T*)P.b.ptr + page[kb] * P.b.sb + h * P.b.sh + (slot[kb] + lc) * P.b.sl + 8 * grp);
            }
        }
        // v into LDS, 0 where there is none; values that are not finite and that some row does not see are added apart
        constexpr int E = 16 / (int)sizeof(T), CPR = DH / E, PASS = KT * CPR / 64;
        bool odd = false;
#pragma unroll
        for (int p = 0; p < PASS; ++p) {
            const int kb = p / (PASS / 2), r = (64 * p + lane) / CPR, ch = lane % CPR, j = jt + r;
            u32x4 x = {0, 0, 0, 0};
            if (page[kb] >= 0 && j >= lo && j < hi)
                x = *reinterpret_cast<const u32x4*>((const T*)P.v.ptr + page[kb] * P.v.sb + h * P.v.sh +
                                                    (slot[kb] + r - 16 * kb) * P.v.sl + E * ch);
            if (mixed && j >= least) {
                T e[E];
                __builtin_memcpy(e, &x, 16);
                bool fine = true;
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    const float y = (float)e[k];
                    if (!(y - y == 0.f)) e[k] = (T)0.f, fine = false;
                }
                odd |= !fine;
                __builtin_memcpy(&x, e, 16);
            }
            *reinterpret_cast<u32x4*>(vs + toff<T, DH>(r, ch)) = x;
        }
        if (lane < KT) {
            const int kb = lane >> 4, j = jt + lane;
            float g = 0.f, f = __builtin_nanf("");       // NaN for a page that is not there
            if (page[kb] >= 0 && j >= lo && j < hi) {
                g = ((const float*)P.g.ptr)[page[kb] * P.g.sb + h * P.g.sh + (slot[kb] + lc) * P.g.sl];
                f = has_f ? ((const float*)P.f.ptr)[page[kb] * P.f.sb + h * P.f.sh + (slot[kb] + lc) * P.f.sl] : 0.f;
            }
            gs[lane] = g;
            fs[lane] = f;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const uint64_t odds = mixed ? __ballot(odd) : 0;
#pragma unroll
        for (int g = 0; g < NR; ++g) {
            if (g >= nr) break;
            f32x4 s[2];
            float mx = -__builtin_inff();
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const f32x4 qk = mma(kf[kb][1], qf[g][1], mma(kf[kb][0], qf[g][0], zero4()));
                const f32x4 cb = mma(bf[kb], cf[g], zero4());
                const f32x4 gk = lds4f(gs + 16 * kb + 4 * grp), fk = lds4f(fs + 16 * kb + 4 * grp);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = jt + 16 * kb + 4 * grp + e;
                    const float dec = lam * fast_exp2((gq[g] - gk[e]) * LOG2E);
                    const float x = fmaf(qk[e], 0.125f * LOG2E, dec * cb[e]) + (fq[g] - fk[e]) * LOG2E;
                    s[kb][e] = j >= lo && j < lim[g] ? x : -__builtin_inff();
                    mx = fmaxf(mx, s[kb][e]);
                }
            }
            mx = fmaxf(group_max(mx), m2[g]);
            // fp16 weights have 2^12 at their largest, which keeps the low parts of small ones above the subnormals
            constexpr float UP = __is_same(T, _Float16) ? 12.f : 0.f;
            const float ref = mx == -__builtin_inff() ? 0.f : mx;
            const float corr = m2[g] == -__builtin_inff() ? 1.f : fast_exp2(m2[g] - ref);
            m2[g] = mx;
            l[g] *= corr;
            f32x4 p[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[kb][e] = fast_exp2(s[kb][e] - (ref - UP));
                    l[g] += p[kb][e];
                }
#pragma unroll
            for (int db = 0; db < 4; ++db) acc[g][db] *= corr;
            f32x4 x0 = p[0], x1 = p[1];
#pragma unroll
            for (int k = 0; k < Split<T>::terms; ++k) {
                const frag8<T> pf = pack8<T>(x0, x1);
#pragma unroll
                for (int db = 0; db < 4; ++db) acc[g][db] = mma(frag_tr<T, DH>(vs, 16 * db, 0, lane), pf, acc[g][db]);
                if (k + 1 < Split<T>::terms) {
                    const f32x8 back = __builtin_convertvector(pf, f32x8);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x0[e] -= back[e], x1[e] -= back[4 + e];
                }
            }
            if (odds) {                                  // p v of the values left out above, for the rows that see them
                for (int j = 0; j < KT; ++j) {
                    const int kb = j >> 4, from = (j >> 2 & 3) * 16 + lc;
                    if (page[kb] < 0 || jt + j < least || jt + j < lo || jt + j >= hi) continue;
                    float pj = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y = __shfl(kb ? p[1][e] : p[0][e], from);
                        pj = e == (j & 3) ? y : pj;
                    }
                    const T* v = (const T*)P.v.ptr + page[kb] * P.v.sb + h * P.v.sh + (slot[kb] + (j & 15)) * P.v.sl;
#pragma unroll
                    for (int db = 0; db < 4; ++db)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float y = (float)v[16 * db + 4 * grp + e];
                            if (!(y - y == 0.f) && jt + j < lim[g]) acc[g][db][e] = fmaf(pj, y, acc[g][db][e]);
                        }
                }
            }
        }
        __builtin_amdgcn_wave_barrier();                 // the tile has been read
    }

    // the waves' parts joined
    constexpr float UP = __is_same(T, _Float16) ? 12.f : 0.f;
#pragma unroll
    for (int g = 0; g < NR; ++g) {
        const float sum = group_sum(l[g]);
        if (grp == 0) sm.m[w][16 * g + lc] = m2[g] - UP, sm.l[w][16 * g + lc] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < NR; ++g) {
        if (g >= nr) break;
        const int r = 16 * g + lc;
        float cm = sm.m[0][r];
#pragma unroll
        for (int k = 1; k < NW; ++k) cm = fmaxf(cm, sm.m[k][r]);
        auto factor = [&](float x) { return x == -__builtin_inff() ? 1.f : fast_exp2(x - cm); };   // all -inf: sums of 0, or NaN
        const float mine = factor(sm.m[w][r]);
#pragma unroll
        for (int db = 0; db < 4; ++db) *reinterpret_cast<f32x4*>(&sm.o[w][lc][16 * db + 4 * grp]) = acc[g][db] * mine;
        __syncthreads();
        const int64_t at = (int64_t)item * PER + 16 * g;
        for (int e = tid; e < 16 * (DH / 4); e += 64 * NW) {
            const int rr = e / (DH / 4), d = 4 * (e % (DH / 4));
            f32x4 x = lds4f(&sm.o[0][rr][d]);
#pragma unroll
            for (int k = 1; k < NW; ++k) x += lds4f(&sm.o[k][rr][d]);
            *reinterpret_cast<f32x4*>(part + (at + rr) * DH + d) = x;
        }
        if (w == 0 && grp == 0) {
            float cl = 0.f;
#pragma unroll
            for (int k = 0; k < NW; ++k) cl = fmaf(sm.l[k][r], factor(sm.m[k][r]), cl);
            stat[at + lc] = f32x2{cm, cl};
        }
        __syncthreads();
    }
}

// A wave per query row: its parts, the common ones first, in order.
template <class TO>
__global__ __launch_bounds__(64 * NW) void prefix_join_kernel(sisa_prefix_decode_args a, Plan plan, int shift, const f32x2* stat,
                                                              const float* part) {
    const int lane = threadIdx.x & 63, H = a.pool.heads, M = a.M, PER = 16 * plan.nr;
    const int64_t row = (int64_t)blockIdx.x * NW + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= (int64_t)a.B * H * M) return;
    const int m = row % M, h = row / M % H, n = row / M / H;
    const int64_t held = (int64_t)a.W << shift;
    TO* out = (TO*)a.out + row * DH + lane;
    const int r = a.group[n], vis = visible(a, held, n, m);
    int lo = -1, f0 = 0, f1 = 0;
    if (r >= 0 && r < a.G) lo = common(a, held, r), f0 = a.first[r], f1 = a.first[r + 1];
    const int64_t mine = (int64_t)(n - f0) * M + m, tile = r >= 0 && r < a.G ? tile_base(a, r, PER) + mine / PER : -1;
    if (vis < 0 || lo < 0 || f0 < 0 || f1 > a.B || n < f0 || n >= f1 || (lo > 0 && (tile < 0 || tile >= plan.tiles))) {
        *out = cvt<TO>(__builtin_nanf(""));
        return;
    }
    float mx = -__builtin_inff(), l = 0.f, o = 0.f;
    auto add = [&](int64_t at) {
        const f32x2 s = stat[at];
        const float x = part[at * DH + lane];
        const float to = fmaxf(mx, s[0]), ref = to == -__builtin_inff() ? 0.f : to;
        const float fa = mx == -__builtin_inff() ? 1.f : fast_exp2(mx - ref), fb = s[0] == -__builtin_inff() ? 1.f : fast_exp2(s[0] - ref);
        l = fmaf(l, fa, s[1] * fb);
        o = fmaf(o, fa, x * fb);
        mx = to;
    };
    const int nt = (lo + KT - 1) / KT;
    for (int p = 0; p < plan.parts && vis > 0; ++p) {
        const Range t = part_of(nt, plan.parts, p);
        if (t.from >= t.to || t.from * KT >= vis) break;
        add((((int64_t)p * plan.tiles + tile) * H + h) * PER + mine % PER);
    }
    const int mt = m / PER, end = visible(a, held, n, (mt + 1) * PER - 1 < M - 1 ? (mt + 1) * PER - 1 : M - 1);
    const int first = lo / KT, nown = end > lo ? (end + KT - 1) / KT - first : 0;
    for (int p = 0; p < plan.own_parts && vis > lo; ++p) {
        const Range t = part_of(nown, plan.own_parts, p);
        if (t.from >= t.to || (first + t.from) * KT >= vis) break;
        add((plan.items + (((int64_t)p * a.B + n) * plan.own_tiles + mt) * H + h) * PER + m % PER);
    }
    *out = cvt<TO>(vis == 0 ? 0.f : o / l);
}

Plan plan_of(int64_t B, int64_t H, int64_t M, int64_t G, int64_t max_len, int64_t max_shared) {
    Plan p{};
    const int64_t rows = sisa::cdiv(B, G) * M;           // of a group, on average
    p.nr = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    const int64_t per = 16 * p.nr;
    p.tiles = (int)(max_shared > 0 ? G + B * M / per : 0);
    p.own_tiles = (int)sisa::cdiv(M, per);
    // about 2,048 workgroups of either kind, each with at least a tile for every wave
    auto parts = [](int64_t items, int64_t positions) {
        const int64_t most = sisa::cdiv(positions, KT * NW), want = items > 0 ? sisa::cdiv(2048, items) : 1;
        const int64_t n = want < most ? want : most;
        return (int)(n < 1 ? 1 : n > SPLITS ? SPLITS : n);
    };
    p.parts = parts(p.tiles * H, max_shared);
    p.own_parts = parts(B * p.own_tiles * H, max_len);
    p.items = (int64_t)p.parts * p.tiles * H;
    p.own_items = (int64_t)p.own_parts * B * p.own_tiles * H;
    return p;
}

struct Space {
    f32x2* stat;
    float* part;
    int64_t bytes;
};
Space space_of(char* base, const Plan& p) {
    const int64_t rows = (p.items + p.own_items) * 16 * p.nr;
    Space s{};
    s.stat = (f32x2*)base;
    s.part = (float*)(base + (rows * 8 + 255) / 256 * 256);
    s.bytes = (char*)s.part - base + rows * DH * 4;
    return s;
}

template <class T>
int launch(const sisa_prefix_decode_args* a, const Plan& p, hipStream_t st) {
    const int shift = sisa::log2_of(a->pool.page_size);
    const Space ws = space_of((char*)a->workspace, p);
    const unsigned grid = (unsigned)(p.items + p.own_items);
    switch (p.nr) {
        case 1: prefix_part_kernel<T, 1><<<grid, 64 * NW, 0, st>>>(*a, p, shift, ws.stat, ws.part); break;
        case 2: prefix_part_kernel<T, 2><<<grid, 64 * NW, 0, st>>>(*a, p, shift, ws.stat, ws.part); break;
        default: prefix_part_kernel<T, 4><<<grid, 64 * NW, 0, st>>>(*a, p, shift, ws.stat, ws.part);
    }
    const int rc = sisa::launch_status("sisa_prefix_decode");
    if (rc) return rc;
    const unsigned rows = (unsigned)sisa::cdiv((int64_t)a->B * a->pool.heads * a->M, NW);
    if (a->out_dtype == SISA_F32) prefix_join_kernel<float><<<rows, 64 * NW, 0, st>>>(*a, p, shift, ws.stat, ws.part);
    else prefix_join_kernel<T><<<rows, 64 * NW, 0, st>>>(*a, p, shift, ws.stat, ws.part);
    return sisa::launch_status("sisa_prefix_decode (join)");
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
    SISA_REQUIRE((p.items + p.own_items) * 64 * NW <= sisa::MAX_THREADS && (int64_t)a->B * a->M * a->pool.heads * 64 <= sisa::MAX_THREADS - 64 * NW,
                 "sisa_prefix_decode: too large for one launch");
    hipStream_t st = (hipStream_t)stream;
    switch (a->pool.dtype) {
        case SISA_BF16: return launch<__bf16>(a, p, st);
        case SISA_F16: return launch<_Float16>(a, p, st);
        default: return launch<float>(a, p, st);
    }
}
