// The attention weights that a prompt's positions receive, summed over its last queries, for gfx950
// (include/sisa_hip_cache.h): w_j = sum over i >= j in the window of exp(s_ij - lse_i).
//
//   s_ij = q_i.k_j / 8 + lam exp(g_i - g_j) (c_i.b_j) + (F_i - F_j)
//
// Two passes over the scores, neither of which keeps them: the queries' log-sum-exp over their keys, then every key's sum
// over its queries. Scores are 16x16 MFMA blocks with K = 64 (q.k) and 32 (c.b). A wave holds up to 64 queries (keys) in
// registers and streams 16 keys (queries) at a time, which L2 serves, the next 16 in LDS and those after them under way
// while the present ones are used; four or eight waves share the 64 and take every fourth or eighth of the 16s. In the first
// pass a lane owns one query per block (the keys are the block's rows), in the second one key: the running sums need no lane
// exchange before the end.
//
// Bound by the vector unit: the products of a block take 48 cycles of the matrix pipe, its 256 scores' exponentials alone
// 32 of issue. So blocks away from the diagonal factor the decay, exp(g_i - g_j) = exp(g_i - g_a) exp(g_a - g_j), and split
// the forget term, (F_i - F_a) + (F_a - F_j), at an anchor a between the two: the wave's first query in the first pass,
// its last key in the second. Where g and F do not rise, both factors are at most 1 and both terms at most 0, so nothing
// overflows and rounding grows with the differences of F, not with F. That leaves a product, two FMAs and one exponential for
// a score. Blocks that meet the diagonal or the end of the sequence take the formula as it stands; so does every block of a
// wave whose anchor is not finite, or on whose wrong side a g or F lies by more than RISE: the wave looks its gates through
// first.
#include "common.h"
#include "host.h"
#include "sisa_hip_cache.h"

namespace {

constexpr int DH = 64, DS = 32;
constexpr int FEW_ROWS = 256;         // query rows up to which, against four times as many keys, each wave has its own keys
constexpr int MAX_SPLITS = 32;        // of the keys in the first pass
constexpr float SCALE = LOG2E / 8;    // of q.k into log2 units
constexpr float RISE = 16.f;          // e^16 at most in a factor: what the other one loses below 2^-126 is less than e^-71

struct Rows {                         // queries of a sequence: first .. first + count - 1
    int n, first, count;
};

SISA_DEV Rows rows_of(const sisa_attn_weights_args& a, int b) {
    int n = a.lengths ? a.lengths[b] : a.L;
    n = n < 0 ? 0 : n > a.L ? a.L : n;
    const int count = a.window && a.window < n ? a.window : n;
    return Rows{n, n - count, count};
}

// 16 positions on their way into a wave's operands. They come from memory in whole rows (a lane takes 16 consecutive bytes,
// its neighbours the rest of the row) and pass through LDS that the wave has to itself: an operand's lanes next to each other
// belong to different rows, so that loading operands directly makes a cache access of every lane (287 accesses a tile; the
// L1 cache was what both passes waited for: 62 us each for 4 x 2,048 positions of 12 heads).
template <class T> struct Frags { frag8<T> x0, x1, s; };      // features 0..31, 32..63 and the state's 0..31
template <class T> struct Tile {
    Frags<T> x;
    f32x4 g, f, st;                               // of the lane's positions 4 grp .. + 3
};
template <class T> struct alignas(16) Buffer {
    T x[16 * DH], s[16 * DS];
    float gates[3 * 16];
};
template <class T> struct Raw {
    static constexpr int E = 16 / (int)sizeof(T), CX = DH / E, CS = DS / E, NX = 16 * CX / 64, NS = 16 * CS / 64;
    u32x4 x[NX], s[NS];
    float gate;
};

// Where a lane's pieces are: positions 0 .. 15 of a (batch, head), gates g (lanes 0..15), F (16..31), starts (32..47). Byte
// offsets within 16 positions are below 2^31 (checked by the host): a load takes a scalar base and one register.
template <class T> struct Stream {
    using R = Raw<T>;
    const char *x, *s;
    int64_t sx, ss;                               // bytes of a position
    const float* gate;
    int lane;
    bool starts;                                  // the lane reads starts

    SISA_DEV Stream(const sisa_view& vx, const sisa_view& vs, const sisa_attn_weights_args& a, int b, int h, const float* start,
                    int lane_) {
        lane = lane_;
        x = (const char*)((const T*)vx.ptr + b * vx.sb + h * vx.sh);
        s = (const char*)((const T*)vs.ptr + b * vs.sb + h * vs.sh);
        sx = vx.sl * (int)sizeof(T);
        ss = vs.sl * (int)sizeof(T);
        const float* g = (const float*)a.g.ptr + b * a.g.sb + h * a.g.sh;
        const float* f = a.f.ptr ? (const float*)a.f.ptr + b * a.f.sb + h * a.f.sh : g;
        starts = start && lane >= 32 && lane < 48;
        gate = (starts ? start : lane >= 16 && lane < 32 ? f : g) + (lane & 15);
    }
    SISA_DEV void go(int64_t positions) {
        x += positions * sx;
        s += positions * ss;
        gate += positions;
    }
    // the 16 positions from here, all of them there
    SISA_DEV R load() const {
        R r;
#pragma unroll
        for (int i = 0; i < R::NX; ++i) {
            const int p = lane + 64 * i;
            r.x[i] = *reinterpret_cast<const u32x4*>(x + (unsigned)((p / R::CX) * (int)sx + 16 * (p % R::CX)));
        }
#pragma unroll
        for (int i = 0; i < R::NS; ++i) {
            const int p = lane + 64 * i;
            r.s[i] = *reinterpret_cast<const u32x4*>(s + (unsigned)((p / R::CS) * (int)ss + 16 * (p % R::CS)));
        }
        r.gate = *gate;
        return r;
    }
    // the 16 positions from r0 (this stream is at 0), those from L on as the last one; the start of row r, which has its own
    // numbering and is padded to 16
    SISA_DEV R load_edge(int r0, int L, int r = 0) const {
        R o;
#pragma unroll
        for (int i = 0; i < R::NX; ++i) {
            const int p = lane + 64 * i, row = r0 + p / R::CX < L ? r0 + p / R::CX : L - 1;
            o.x[i] = *reinterpret_cast<const u32x4*>(x + row * sx + 16 * (p % R::CX));
        }
#pragma unroll
        for (int i = 0; i < R::NS; ++i) {
            const int p = lane + 64 * i, row = r0 + p / R::CS < L ? r0 + p / R::CS : L - 1;
            o.s[i] = *reinterpret_cast<const u32x4*>(s + row * ss + 16 * (p % R::CS));
        }
        const int g = r0 + (lane & 15) < L ? r0 : L - 1 - (lane & 15);
        o.gate = gate[starts ? r : g];
        return o;
    }
};

// Through the wave's own LDS; a wave's LDS accesses are carried out in their order.
template <class T, bool FORGET>
SISA_DEV Tile<T> turn(const Raw<T>& r, Buffer<T>* buf, int lane) {
    using R = Raw<T>;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < R::NX; ++i) {
        const int p = lane + 64 * i;
        *reinterpret_cast<u32x4*>(buf->x + toff<T, DH>(p / R::CX, p % R::CX)) = r.x[i];
    }
#pragma unroll
    for (int i = 0; i < R::NS; ++i) {
        const int p = lane + 64 * i;
        *reinterpret_cast<u32x4*>(buf->s + toff<T, DS>(p / R::CS, p % R::CS)) = r.s[i];
    }
    if (lane < 48) buf->gates[lane] = r.gate;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int grp = lane >> 4;
    return Tile<T>{Frags<T>{frag_rows<T, DH>(buf->x, 0, 0, lane), frag_rows<T, DH>(buf->x, 0, 1, lane),
                            frag_rows<T, DS>(buf->s, 0, 0, lane)},
                   lds4f(buf->gates + 4 * grp), FORGET ? lds4f(buf->gates + 16 + 4 * grp) : zero4(),
                   lds4f(buf->gates + 32 + 4 * grp)};
}

// Whether a wave's anchor (ga, fa) serves it. `off`: it does not for the lane's own gates. SIGN 1: the gates of the keys in
// `tiles` tiles from position `first` on, `step` positions from one to the next, must not lie below the anchor's; -1: those of
// queries not above. NaN needs no care, every score that meets it is NaN in either form. Each quarter of the wave looks at E
// tiles at a time. It costs 2 % of 4 x 2,048 positions of 12 heads and 3 % of the last 64 of 16,384 (76.6 -> 78.4 and 33.6 ->
// 34.7 us); watching the gates that the loops load anyway, whose registers then spill, 22 % of both.
template <int SIGN, bool FORGET, int E>
SISA_DEV bool anchored(const sisa_attn_weights_args& a, int b, int h, float ga, float fa, bool off, int first, int tiles, int step,
                       int lane) {
    const float* g = (const float*)a.g.ptr + b * a.g.sb + h * a.g.sh;
    const float* f = (const float*)a.f.ptr + b * a.f.sb + h * a.f.sh;
    float w = 0.f;
    for (int k = lane >> 4; k < tiles; k += 4 * E) {
        float x[E], y[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {                  // behind the last tile the last again; positions are below 2^30
            const unsigned at = first + step * (k + 4 * e < tiles ? k + 4 * e : tiles - 1) + (lane & 15);
            x[e] = *(const float*)((const char*)g + 4 * at);
            y[e] = FORGET ? *(const float*)((const char*)f + 4 * at) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) w = fmaxf(w, fmaxf(SIGN * (ga - x[e]), FORGET ? SIGN * (fa - y[e]) : 0.f));
    }
    const float inf = __builtin_inff();
    return !__any(off || w > RISE || !(fabsf(ga) < inf && (!FORGET || fabsf(fa) < inf)));
}

SISA_DEV float gate(const sisa_view& v, int b, int h, int r, int L) {
    return v.ptr ? ((const float*)v.ptr)[b * v.sb + h * v.sh + (r < L ? r : L - 1)] : 0.f;
}

// (m, l) of two parts of a row, log2 units
SISA_DEV void merge(float& m, float& l, float m2, float l2) {
    const float t = fmaxf(m, m2), ref = t == -__builtin_inff() ? 0.f : t;
    l = l * (m == -__builtin_inff() ? 1.f : fast_exp2(m - ref)) + l2 * (m2 == -__builtin_inff() ? 1.f : fast_exp2(m2 - ref));
    m = t;
}

// x of the lane whose number differs in bit 0 (0xB1) or bit 1 (0x4E).
template <int CTRL> SISA_DEV float in_quad(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}

// What the second pass starts its products from: -lse in units of q.k.
SISA_DEV float start_of(float m, float l) { return -(m + __log2f(l)) * (1.f / SCALE); }

// First pass. A block whose maximum exceeds the running one by less than 2^GROW leaves it as it is.
constexpr float GROW = 16.f;
// With `parts`, a row's maximum and sum over the split's keys are left for the second pass to join.
template <class T, bool FORGET, int U, int NW>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 ? 3 : 2) void weights_lse_kernel(sisa_attn_weights_args a, int R, int nsplit,
                                                                                     float* start, f32x2* parts) {
    constexpr int OWN = 16 * U;
    __shared__ float sm[NW][OWN], sl[NW][OWN];
    __shared__ Buffer<T> bufs[NW];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = lane >> 4, col = lane & 15, L = a.L, BH = a.B * a.H;
    // the longest blocks first, the heads side by side (with a multiple of 8 of them each stays on one XCD)
    const int bh = blockIdx.x % BH, rest = blockIdx.x / BH, split = rest % nsplit, h = bh % a.H, b = bh / a.H;
    const int r0 = ((R + OWN - 1) / OWN - 1 - rest / nsplit) * OWN;
    const Rows rows = rows_of(a, b);
    if (r0 >= rows.count) return;
    const int i0 = rows.first + r0;
    const float lam = a.lam[h * a.s_lam];
    Buffer<T>* buf = bufs + w;
    float gi[U], fi[U], md[U], ld[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        gi[u] = gate(a.g, b, h, i0 + 16 * u + col, L);
        fi[u] = gate(a.f, b, h, i0 + 16 * u + col, L);
        md[u] = -__builtin_inff();
        ld[u] = 0.f;
    }
    const int last = i0 + OWN < rows.n ? i0 + OWN : rows.n;          // keys 0 .. last - 1
    const int tiles = (last + 15) / 16;
    // split s takes a contiguous range of the tiles, wave w every NW-th; tiles up to `below` lie at or before i0
    const int per = (tiles + nsplit - 1) / nsplit;
    const int t0 = split * per, t1 = t0 + per < tiles ? t0 + per : tiles;
    const int below = (i0 + 1) / 16 < t1 ? (i0 + 1) / 16 : t1;
    int far = 0;                                                     // whole tiles that the wave takes as those on the diagonal
    Stream<T> keys(a.k, a.b, a, b, h, nullptr, lane);
    Frags<T> q[U];
    {
        const Stream<T> own(a.q, a.c, a, b, h, nullptr, lane);
        Raw<T> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = own.load_edge(i0 + 16 * u, L);
        if (below - 1 - w >= t0) {
            const float ga = gate(a.g, b, h, i0, L), fa = gate(a.f, b, h, i0, L);
            bool off = false;
#pragma unroll
            for (int u = 0; u < U; ++u) off |= i0 + 16 * u + col < rows.n && (gi[u] - ga > RISE || fi[u] - fa > RISE);
            const int whole = (below - 1 - t0 - w) / NW + 1;
            // (eight waves with 64 rows: the keys are split, a wave has few tiles)
            if (!anchored<1, FORGET, U == 4 && NW == 8 ? 2 : 8>(a, b, h, ga, fa, off, 16 * (below - 1 - w), whole, -16 * NW, lane))
                far = whole;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = turn<T, FORGET>(raw[u], buf, lane).x;
    }
    for (int n = -far;; ++n) {                                       // meeting the diagonal
        const int t = n < 0 ? below - 1 - w + NW * (n + 1) : (below > t0 ? below : t0) + w + NW * n;
        if (t >= t1) break;
        const Tile<T> k = turn<T, FORGET>(keys.load_edge(16 * t, L), buf, lane);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (16 * t > i0 + 16 * u + 15) continue;                 // all keys after all queries
            const f32x4 qk = mma(k.x.x1, q[u].x1, mma(k.x.x0, q[u].x0, zero4())), cb = mma(k.x.s, q[u].s, zero4());
            float x[4], mx = md[u];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float dec = lam * fast_exp2((gi[u] - k.g[e]) * LOG2E);
                x[e] = (fmaf(qk[e], 0.125f, dec * cb[e]) + (fi[u] - k.f[e])) * LOG2E;
                if (16 * t + 4 * grp + e > i0 + 16 * u + col) x[e] = -__builtin_inff();
                mx = fmaxf(mx, x[e]);
            }
            const float ref = mx == -__builtin_inff() ? 0.f : mx;
            ld[u] *= md[u] == -__builtin_inff() ? 1.f : fast_exp2(md[u] - ref);
#pragma unroll
            for (int e = 0; e < 4; ++e) ld[u] += fast_exp2(x[e] - ref);
            md[u] = mx;
        }
    }
    int left = (below - 1 - t0 - w) / NW + 1;                        // whole tiles of this wave, from the diagonal down
    if (far == 0 && below - 1 - w >= t0) {
        const float ga = gate(a.g, b, h, i0, L), fa = gate(a.f, b, h, i0, L);
        // y = 8 score - 8 (F_i - F_a); sums of 2^(y SCALE - ref), the maximum so far in mo
        float qg[U], mo[U], ref[U], lo[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            qg[u] = 8.f * lam * fast_exp2((gi[u] - ga) * LOG2E);
            mo[u] = -__builtin_inff();
            ref[u] = lo[u] = 0.f;
        }
        bool fresh = true;                                           // a maximum is still missing
        keys.go(16 * (int64_t)(below - 1 - w));
        auto add = [&](const Tile<T>& k) {
            f32x4 kg, kf;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                kg[e] = fast_exp2((ga - k.g[e]) * LOG2E);
                kf[e] = FORGET ? 8.f * (fa - k.f[e]) : 0.f;
            }
            f32x4 y[U];
            float mx = -__builtin_inff();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const f32x4 cb = mma(k.x.s, q[u].s, zero4());
                y[u] = mma(k.x.x1, q[u].x1, mma(k.x.x0, q[u].x0, kf));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[u][e] = fmaf(fmaf(cb[e] * kg[e], qg[u], y[u][e]), SCALE, -ref[u]);
                    mx = fmaxf(mx, y[u][e]);
                }
            }
            if (__any(fresh || mx > GROW)) {
                asm volatile("");                                    // rarely: not to be worked out beforehand
                fresh = false;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float to = fmaxf(mo[u], fmaxf(fmaxf(y[u][0], y[u][1]), fmaxf(y[u][2], y[u][3])) + ref[u]);
                    const float by = ref[u] - (to == -__builtin_inff() ? 0.f : to);
                    if (lo[u] != 0.f) lo[u] *= fast_exp2(by);
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[u][e] += by;
                    mo[u] = to;
                    ref[u] -= by;
                    fresh |= to == -__builtin_inff();
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) lo[u] += fast_exp2(y[u][e]);
        };
        // Two tiles ahead in memory, one in LDS; the last one's loads are its own again.
        auto next = [&]() {
            if (--left > 0) keys.go(-16 * NW);
            return keys.load();
        };
        Raw<T> raw = keys.load();
        Tile<T> even = turn<T, FORGET>(raw, buf, lane);
        raw = next();
        while (true) {
            const bool more = left > 0;
            const Tile<T> odd = turn<T, FORGET>(raw, buf, lane);
            raw = next();
            add(even);
            if (!more) break;
            const bool yet = left > 0;
            even = turn<T, FORGET>(raw, buf, lane);
            raw = next();
            add(odd);
            if (!yet) break;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            merge(md[u], ld[u], (mo[u] == -__builtin_inff() ? mo[u] : ref[u]) + (fi[u] - fa) * LOG2E, lo[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) merge(md[u], ld[u], __shfl_xor(md[u], o), __shfl_xor(ld[u], o));
        if (grp == 0) sm[w][16 * u + col] = md[u], sl[w][16 * u + col] = ld[u];
    }
    __syncthreads();
    const int r = r0 + lane;
    if (w != 0 || lane >= OWN || r >= rows.count) return;
    float mt = sm[0][lane], lt = sl[0][lane];
#pragma unroll
    for (int k = 1; k < NW; ++k) merge(mt, lt, sm[k][lane], sl[k][lane]);
    const int64_t at = (int64_t)bh * ((R + 15) / 16 * 16) + r;
    if (parts) parts[at * nsplit + split] = f32x2{mt, lt};
    else start[at] = start_of(mt, lt);
}

// Second pass. SHARE of a workgroup's NW waves have the same 64 keys and take every SHARE-th query tile: all of them, or one
// where so few queries are counted that the keys' loads weigh more (then the rows' parts from the first pass are joined here,
// in the order of the splits, by every workgroup: at most 256 rows of 32 parts).
template <class T, bool FORGET, int U, int NW, int SHARE>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 ? 3 : 2) void weights_sum_kernel(sisa_attn_weights_args a, int R, int nsplit,
                                                                                     const float* start, const f32x2* parts) {
    constexpr bool FEW = SHARE == 1;
    constexpr int OWN = 16 * U;
    __shared__ float part[NW][OWN];
    __shared__ float starts[FEW ? FEW_ROWS : 4];
    __shared__ Buffer<T> bufs[NW];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ws = w % SHARE;
    const int grp = lane >> 4, col = lane & 15, L = a.L, BH = a.B * a.H;
    const int bh = blockIdx.x % BH, h = bh % a.H, b = bh / a.H;
    const int j0 = (blockIdx.x / BH * (NW / SHARE) + w / SHARE) * OWN;
    const Rows rows = rows_of(a, b);
    const float lam = a.lam[h * a.s_lam];
    Buffer<T>* buf = bufs + w;
    const int Rp = (R + 15) / 16 * 16;
    Raw<T> raw[U];                                                   // the keys, under way while the rows' parts are joined
    {
        const Stream<T> own(a.k, a.b, a, b, h, nullptr, lane);
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = own.load_edge(j0 + 16 * u, L);
    }
    if constexpr (FEW) {
        // four lanes a row, all of their parts under way at once
        const int sub = threadIdx.x & 3;
        for (int r0 = 0; r0 < rows.count; r0 += 16 * NW) {
            const int r = r0 + threadIdx.x / 4;
            const f32x2* p = parts + ((int64_t)bh * Rp + (r < rows.count ? r : 0)) * nsplit;
            f32x2 x[MAX_SPLITS / 4];
            float m = -__builtin_inff(), l = 0.f;
#pragma unroll
            for (int k = 0; k < MAX_SPLITS / 4; ++k)
                x[k] = 4 * k < nsplit ? p[4 * k + sub < nsplit ? 4 * k + sub : 0] : f32x2{-__builtin_inff(), 0.f};
#pragma unroll
            for (int k = 0; k < MAX_SPLITS / 4; ++k) {
                if (4 * k + sub >= nsplit) x[k] = f32x2{-__builtin_inff(), 0.f};
                m = fmaxf(m, x[k][0]);
            }
            m = fmaxf(m, in_quad<0xB1>(m));
            m = fmaxf(m, in_quad<0x4E>(m));
            const float ref = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
            for (int k = 0; k < MAX_SPLITS / 4; ++k)
                if (4 * k < nsplit) l += x[k][1] * (x[k][0] == -__builtin_inff() ? 1.f : fast_exp2(x[k][0] - ref));
            l += in_quad<0xB1>(l);
            l += in_quad<0x4E>(l);
            if (sub == 0 && r < rows.count) starts[r] = start_of(m, l);
        }
        __syncthreads();
    }
    float sum[U] = {};
    // 16-query tiles of the window from the first that reaches j0: those that meet the diagonal, whole ones, the last one
    const int from = j0 > rows.first ? (j0 - rows.first) / 16 : 0, tiles = (rows.count + 15) / 16;
    if (j0 < rows.n && from < tiles) {
        Stream<T> queries(a.q, a.c, a, b, h, FEW ? nullptr : start + (int64_t)bh * Rp, lane);
        Frags<T> k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) k[u] = turn<T, FORGET>(raw[u], buf, lane).x;
        float gj[U], fj[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            gj[u] = gate(a.g, b, h, j0 + 16 * u + col, L);
            fj[u] = gate(a.f, b, h, j0 + 16 * u + col, L);
        }
        const int clear = j0 + OWN - 1 - rows.first;                 // the first row that sees every key of the block
        int w0 = clear > 0 ? (clear + 15) / 16 : 0, w1 = rows.count / 16;
        w0 = w0 < from ? from : w0 < tiles ? w0 : tiles;
        w1 = w1 < w0 ? w0 : w1;
        int left = w0 + ws < w1 ? (w1 - 1 - w0 - ws) / SHARE + 1 : 0;
        int far = 0;                                                 // whole tiles that the wave takes as those on the edges
        const float ga = gate(a.g, b, h, j0 + OWN - 1, L), fa = gate(a.f, b, h, j0 + OWN - 1, L);
        if (left > 0) {
            bool off = false;
#pragma unroll
            for (int u = 0; u < U; ++u) off |= ga - gj[u] > RISE || fa - fj[u] > RISE;
            if (!anchored<-1, FORGET, FEW ? 2 : 8>(a, b, h, ga, fa, off, rows.first + 16 * (w0 + ws), left, 16 * SHARE, lane))
                far = left, left = 0;
        }
        const int edges = w0 - from + tiles - w1;
        for (int e0 = ws - SHARE * far; e0 < edges; e0 += SHARE) {
            const int t = e0 < 0 ? w0 + e0 + SHARE * far : e0 < w0 - from ? from + e0 : w1 + e0 - (w0 - from);
            const int i0 = rows.first + 16 * t;
            Tile<T> q = turn<T, FORGET>(queries.load_edge(i0, L, 16 * t), buf, lane);
            if constexpr (FEW) q.st = lds4f(starts + 16 * t + 4 * grp);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (j0 + 16 * u > i0 + 15) continue;                 // all keys after all queries
                const f32x4 qk = mma(q.x.x1, k[u].x1, mma(q.x.x0, k[u].x0, zero4())), cb = mma(q.x.s, k[u].s, zero4());
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = i0 + 4 * grp + e;
                    const float dec = lam * fast_exp2((q.g[e] - gj[u]) * LOG2E);
                    const float x = fmaf(qk[e], 0.125f, dec * cb[e]) + (q.f[e] - fj[u]);
                    const float p = fast_exp2(fmaf(x, LOG2E, q.st[e] * SCALE));
                    sum[u] += i >= j0 + 16 * u + col && i < rows.n ? p : 0.f;
                }
            }
        }
        if (left > 0) {
            float kg[U], kf[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                kg[u] = lam * LOG2E * fast_exp2((ga - gj[u]) * LOG2E);
                kf[u] = (fa - fj[u]) * LOG2E;
            }
            queries.go(rows.first + 16 * (int64_t)(w0 + ws));
            if (queries.starts) queries.gate -= rows.first;
            const float* st = starts + 16 * (w0 + ws) + 4 * grp;      // of the tile that is used next
            auto add = [&](Tile<T> q) {
                if constexpr (FEW) q.st = lds4f(st), st += 16 * SHARE;
                f32x4 rg, rc;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    rg[e] = fast_exp2((q.g[e] - ga) * LOG2E);
                    rc[e] = FORGET ? fmaf(q.f[e] - fa, 8.f, q.st[e]) : q.st[e];
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const f32x4 qk = mma(q.x.x1, k[u].x1, mma(q.x.x0, k[u].x0, rc)), cb = mma(q.x.s, k[u].s, zero4());
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[u] += fast_exp2(fmaf(cb[e] * kg[u], rg[e], fmaf(qk[e], SCALE, kf[u])));
                }
            };
            // two tiles ahead in memory, one in LDS; the last one's loads are its own again
            auto next = [&]() {
                if (--left > 0) queries.go(16 * SHARE);
                return queries.load();
            };
            Raw<T> raw = queries.load();
            Tile<T> even = turn<T, FORGET>(raw, buf, lane);
            raw = next();
            while (true) {
                const bool more = left > 0;
                const Tile<T> odd = turn<T, FORGET>(raw, buf, lane);
                raw = next();
                add(even);
                if (!more) break;
                const bool yet = left > 0;
                even = turn<T, FORGET>(raw, buf, lane);
                raw = next();
                add(odd);
                if (!yet) break;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) sum[u] += __shfl_xor(sum[u], o);
        if (grp == 0) part[w][16 * u + col] = sum[u];
    }
    __syncthreads();
    const int j = j0 + lane;
    if (ws || lane >= OWN || j >= L) return;
    float s = part[w][lane];
#pragma unroll
    for (int k = 1; k < SHARE; ++k) s += part[w + k][lane];
    a.out[(int64_t)bh * L + j] = j < rows.n ? s : 0.f;
}

// How a call is laid out. Waves hold 64 queries (keys), four share them, where such blocks of all the queries are many. Where
// they are fewer, less: `groups` counts them, and both passes together took (us)
//                              16 rows, 8 waves   32 rows, 8   32 rows, 4   64 rows, 4
//   1 x 512 x 12 heads,  96          13.7            13.8         14.9         17.6
//   1 x 1,024 x 12,     192          22.5            18.5         21.0         25.1
//   2 x 920 x 12,       360          32.1            26.4         21.5         25.8
//   1 x 2,048 x 16,     512          65              44.8         41.2         44.8
//   4 x 1,024 x 12,     768          64              45.7         37.3         33.1
// Where few rows are counted against many keys, the keys of the first pass are split (256 keys at least, 32 splits at most),
// the second joins the parts, and there each wave has its own keys (the last 64 of 16,384 positions of 16 heads: 43 -> 35.5 us,
// 35 with four lanes to a row's join; 512 to 2,048 workgroups of splits in place of 256: first pass 15.6 -> 17 to 20.9). From
// FEW_ROWS + 1 rows on nothing is split: the last 256 of 16,384 positions of 4 heads take 29 us, the last 257 80.
struct Plan {
    int R, nsplit;
    bool few;
    int64_t groups, Rp, bytes;
};

Plan plan_of(int32_t B, int32_t H, int32_t L, int32_t window) {
    Plan p{};
    p.R = window && window < L ? window : L;
    p.Rp = (p.R + 15) / 16 * 16;
    p.few = p.R <= FEW_ROWS && L / 4 >= p.R;
    const int64_t BH = (int64_t)B * H;
    p.groups = BH * sisa::cdiv(p.R, 64);
    p.nsplit = 1;
    if (p.few && p.groups < 256) {
        const int64_t want = 256 / p.groups, most = sisa::cdiv(L, 256);
        p.nsplit = (int)(want < most ? want : most);
        p.nsplit = p.nsplit < MAX_SPLITS ? p.nsplit : MAX_SPLITS;
    }
    p.bytes = BH * p.Rp * (p.few ? 8 * (int64_t)p.nsplit : 4);
    return p;
}

// U blocks of 16 queries, NW waves in the first pass; U2 of keys, NW2 waves of which SHARE have the same in the second.
template <class T, bool FORGET, int U, int NW, int U2, int NW2, int SHARE>
int launch_weights(const sisa_attn_weights_args* a, const Plan& p, hipStream_t st) {
    const int64_t BH = (int64_t)a->B * a->H;
    float* start = p.few ? nullptr : (float*)a->workspace;
    f32x2* parts = p.few ? (f32x2*)a->workspace : nullptr;
    const int64_t rows = BH * sisa::cdiv(p.R, 16 * U) * p.nsplit, keys = BH * sisa::cdiv(a->L, 16 * U2 * (NW2 / SHARE));
    SISA_REQUIRE(rows <= sisa::MAX_THREADS / (64 * NW) && keys <= sisa::MAX_THREADS / (64 * NW2),
                 "sisa_attn_weights: B*H*L too large for one launch");
    weights_lse_kernel<T, FORGET, U, NW><<<(unsigned)rows, 64 * NW, 0, st>>>(*a, p.R, p.nsplit, start, parts);
    const int rc = sisa::launch_status("sisa_attn_weights (rows)");
    if (rc) return rc;
    weights_sum_kernel<T, FORGET, U2, NW2, SHARE><<<(unsigned)keys, 64 * NW2, 0, st>>>(*a, p.R, p.nsplit, start, parts);
    return sisa::launch_status("sisa_attn_weights");
}

template <class T, bool FORGET>
int launch_weights(const sisa_attn_weights_args* a, hipStream_t st) {
    const Plan p = plan_of(a->B, a->H, a->L, a->window);
    if (p.few) return launch_weights<T, FORGET, 4, 8, 4, 4, 1>(a, p, st);
    if (p.groups < 128) return launch_weights<T, FORGET, 1, 8, 1, 8, 8>(a, p, st);
    if (p.groups < 256) return launch_weights<T, FORGET, 2, 8, 2, 8, 8>(a, p, st);
    if (p.groups < 640) return launch_weights<T, FORGET, 2, 4, 2, 4, 4>(a, p, st);
    return launch_weights<T, FORGET, 4, 4, 4, 4, 4>(a, p, st);
}

template <class T>
int launch_weights(const sisa_attn_weights_args* a, hipStream_t st) {
    return a->f.ptr ? launch_weights<T, true>(a, st) : launch_weights<T, false>(a, st);
}

}  // namespace

extern "C" int64_t sisa_attn_weights_workspace_bytes(int32_t B, int32_t H, int32_t L, int32_t window) {
    if (B < 1 || H < 1 || L < 1 || window < 0) return 0;
    return plan_of(B, H, L, window).bytes;
}

extern "C" int sisa_attn_weights(const sisa_attn_weights_args* a, void* stream) {
    SISA_REQUIRE(a != nullptr, "sisa_attn_weights: null args");
    SISA_REQUIRE(a->B >= 0 && a->H >= 1 && a->L >= 0 && a->L <= (1 << 30) && a->window >= 0,
                 "sisa_attn_weights: bad shape B=%d H=%d L=%d window=%d", a->B, a->H, a->L, a->window);
    SISA_REQUIRE(a->dtype == SISA_BF16 || a->dtype == SISA_F16 || a->dtype == SISA_F32, "sisa_attn_weights: dtype %d",
                 a->dtype);
    if (a->B == 0 || a->L == 0) return SISA_OK;
    SISA_REQUIRE(sisa::view_ok(a->q, a->dtype) && sisa::view_ok(a->k, a->dtype) && sisa::view_ok(a->c, a->dtype) &&
                     sisa::view_ok(a->b, a->dtype),
                 "sisa_attn_weights: q, k, c and b rows must be 16-byte aligned");
    const sisa_view* rows[] = {&a->q, &a->k, &a->c, &a->b};
    for (const sisa_view* v : rows)
        SISA_REQUIRE(v->sl >= 0 && v->sl < SISA_ATTN_WEIGHTS_MAX_STRIDE,
                     "sisa_attn_weights: position strides must be in 0 .. %d elements", SISA_ATTN_WEIGHTS_MAX_STRIDE - 1);
    SISA_REQUIRE(a->g.ptr && a->lam && a->out && a->workspace && ((uintptr_t)a->workspace & 15) == 0,
                 "sisa_attn_weights: null pointer, or workspace not 16-byte aligned");
    SISA_REQUIRE(a->g.sl == 1 && (!a->f.ptr || a->f.sl == 1), "sisa_attn_weights: g and f must be contiguous along positions");
    hipStream_t st = (hipStream_t)stream;
    switch (a->dtype) {
        case SISA_BF16: return launch_weights<__bf16>(a, st);
        case SISA_F16: return launch_weights<_Float16>(a, st);
        default: return launch_weights<float>(a, st);
    }
}
