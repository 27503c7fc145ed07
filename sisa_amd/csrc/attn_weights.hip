// The attention weights that a prompt's positions receive, summed over its last queries, for gfx950
// (include/sisa_hip_cache.h): w_j = sum over i >= j in the window of exp(s_ij - lse_i).
//
//   s_ij = q_i.k_j / 8 + lam exp(g_i - g_j) (c_i.b_j) + (F_i - F_j)
//
// Two passes over the scores, neither of which keeps them: the queries' log-sum-exp over their keys, then every key's sum
// over its queries. Scores are 16x16 MFMA blocks with K = 64 (q.k) and 32 (c.b). A wave holds 64 queries (keys) in
// registers and streams 16 keys (queries) at a time straight from memory, which L2 serves, the next 16 loaded before the
// present ones are used; four waves share the 64 and take every fourth of the 16s. In the first pass a lane owns one query
// per block (the keys are the block's rows), in the second one key: the running sums need no lane exchange before the end.
//
// Bound by the vector unit: the products of a block take 48 cycles of the matrix pipe, its 256 scores' exponentials alone
// 32 of issue. So blocks away from the diagonal factor the decay, exp(g_i - g_j) = exp(g_i - g_a) exp(g_a - g_j), and split
// the forget term, (F_i - F_a) + (F_a - F_j), at an anchor a between the two: the first query of the 64 in the first pass,
// the last key in the second. Both factors are at most 1 and both terms at most 0 there, so nothing overflows and rounding
// grows with the differences of F, not with F. That leaves a product, two FMAs and one exponential for a score. Blocks
// that meet the diagonal or the end of the sequence take the formula as it stands.
#include "common.h"
#include "host.h"
#include "sisa_hip_cache.h"

namespace {

constexpr int DH = 64, DS = 32;
constexpr int WG = 4;                 // waves per workgroup
constexpr int OWN = 64;               // queries (keys) that a wave holds: four blocks of 16
constexpr float SCALE = LOG2E / 8;    // of q.k into log2 units

struct Rows {                         // queries of a sequence: first .. first + count - 1
    int n, first, count;
};

SISA_DEV Rows rows_of(const sisa_attn_weights_args& a, int b) {
    int n = a.lengths ? a.lengths[b] : a.L;
    n = n < 0 ? 0 : n > a.L ? a.L : n;
    const int count = a.window && a.window < n ? a.window : n;
    return Rows{n, n - count, count};
}

// The operand of 16 positions, r0 + lane % 16, features 0..31 and 32..63 and the state's 0..31; positions beyond the last
// of the view as the last one.
template <class T> struct Frags { frag8<T> x0, x1, s; };
template <class T>
SISA_DEV Frags<T> frags(const sisa_view& x, const sisa_view& s, int b, int h, int r0, int L, int lane) {
    const int row = r0 + (lane & 15) < L ? r0 + (lane & 15) : L - 1, f = 8 * (lane >> 4);
    const T* p = (const T*)x.ptr + b * x.sb + h * x.sh + row * x.sl;
    const T* q = (const T*)s.ptr + b * s.sb + h * s.sh + row * s.sl;
    return Frags<T>{load8<T>(p + f), load8<T>(p + 32 + f), load8<T>(q + f)};
}

SISA_DEV float gate(const sisa_view& v, int b, int h, int r, int L) {
    return v.ptr ? ((const float*)v.ptr)[b * v.sb + h * v.sh + (int64_t)(r < L ? r : L - 1) * v.sl] : 0.f;
}

// Four positions r .. r + 3, one load where they are neighbours in memory (at any alignment); 0 without a forget term.
struct __attribute__((packed, aligned(4))) Floats4 { f32x4 v; };
SISA_DEV f32x4 gates4(const sisa_view& v, int b, int h, int r, int L) {
    if (!v.ptr) return zero4();
    const float* p = (const float*)v.ptr + b * v.sb + h * v.sh;
    if (v.sl == 1 && r + 4 <= L) return reinterpret_cast<const Floats4*>(p + r)->v;
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = p[(int64_t)(r + e < L ? r + e : L - 1) * v.sl];
    return x;
}

// (m, l) of two parts of a row, log2 units
SISA_DEV void merge(float& m, float& l, float m2, float l2) {
    const float t = fmaxf(m, m2), ref = t == -__builtin_inff() ? 0.f : t;
    l = l * (m == -__builtin_inff() ? 1.f : fast_exp2(m - ref)) + l2 * (m2 == -__builtin_inff() ? 1.f : fast_exp2(m2 - ref));
    m = t;
}

// 16 streamed positions from r0: operands, g and F of the lane's four
template <class T> struct Tile {
    Frags<T> x;
    f32x4 g, f;
};
template <class T>
SISA_DEV Tile<T> load_tile(const sisa_attn_weights_args& a, bool keys, int b, int h, int r0, int lane) {
    const int r = r0 + 4 * (lane >> 4);
    return Tile<T>{keys ? frags<T>(a.k, a.b, b, h, r0, a.L, lane) : frags<T>(a.q, a.c, b, h, r0, a.L, lane),
                   gates4(a.g, b, h, r, a.L), gates4(a.f, b, h, r, a.L)};
}

// First pass. Keys go from the diagonal down, so that the running maximum is right early: a block whose maximum exceeds it
// by less than 2^GROW leaves it as it is.
constexpr float GROW = 16.f;
template <class T>
__global__ __launch_bounds__(64 * WG) void weights_lse_kernel(sisa_attn_weights_args a, int R, int nsplit, float* lse) {
    __shared__ float sm[WG][OWN], sl[WG][OWN];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = lane >> 4, col = lane & 15, L = a.L, BH = a.B * a.H;
    // the longest blocks first, the heads side by side (with a multiple of 8 of them each stays on one XCD)
    const int bh = blockIdx.x % BH, rest = blockIdx.x / BH, split = rest % nsplit, h = bh % a.H, b = bh / a.H;
    const int r0 = ((R + OWN - 1) / OWN - 1 - rest / nsplit) * OWN;
    const Rows rows = rows_of(a, b);
    if (r0 >= rows.count) return;
    const int i0 = rows.first + r0;
    const float lam = a.lam[h * a.s_lam];
    Frags<T> q[4];
    float gi[4], fi[4], md[4], ld[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        q[u] = frags<T>(a.q, a.c, b, h, i0 + 16 * u, L, lane);
        gi[u] = gate(a.g, b, h, i0 + 16 * u + col, L);
        fi[u] = gate(a.f, b, h, i0 + 16 * u + col, L);
        md[u] = -__builtin_inff();
        ld[u] = 0.f;
    }
    const float ga = gate(a.g, b, h, i0, L), fa = gate(a.f, b, h, i0, L);
    const int last = i0 + OWN < rows.n ? i0 + OWN : rows.n;          // keys 0 .. last - 1
    const int tiles = (last + 15) / 16, below = (i0 + 1) / 16;       // tiles 0 .. below - 1 lie at or before i0
    // tiles from the last down; split s takes a contiguous range of them, wave w every fourth
    const int per = (tiles + nsplit - 1) / nsplit;
    const int t0 = tiles - 1 - split * per, t1 = t0 - per > -1 ? t0 - per : -1;
    int t = t0 - w;
    if (t > t1) {
        Tile<T> now = load_tile<T>(a, true, b, h, 16 * t, lane);
        for (; t > t1 && t >= below; t -= WG) {                      // meeting the diagonal
            const int tn = t - WG > 0 ? t - WG : 0;
            const Tile<T> next = load_tile<T>(a, true, b, h, 16 * tn, lane);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (16 * t > i0 + 16 * u + 15) continue;             // all keys after all queries
                const f32x4 qk = mma(now.x.x1, q[u].x1, mma(now.x.x0, q[u].x0, zero4())), cb = mma(now.x.s, q[u].s, zero4());
                float x[4], mx = md[u];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float dec = lam * fast_exp2((gi[u] - now.g[e]) * LOG2E);
                    x[e] = (fmaf(qk[e], 0.125f, dec * cb[e]) + (fi[u] - now.f[e])) * LOG2E;
                    if (16 * t + 4 * grp + e > i0 + 16 * u + col) x[e] = -__builtin_inff();
                    mx = fmaxf(mx, x[e]);
                }
                const float ref = mx == -__builtin_inff() ? 0.f : mx;
                ld[u] *= md[u] == -__builtin_inff() ? 1.f : fast_exp2(md[u] - ref);
#pragma unroll
                for (int e = 0; e < 4; ++e) ld[u] += fast_exp2(x[e] - ref);
                md[u] = mx;
            }
            now = next;
        }
        if (t > t1) {
            // y = 8 score - 8 (F_i - F_a), the reference mo in log2 units
            float qg[4], mo[4], lo[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                qg[u] = 8.f * lam * fast_exp2((gi[u] - ga) * LOG2E);
                mo[u] = -__builtin_inff();
                lo[u] = 0.f;
            }
            for (; t > t1; t -= WG) {
                const int tn = t - WG > 0 ? t - WG : 0;
                const Tile<T> next = load_tile<T>(a, true, b, h, 16 * tn, lane);
                f32x4 kg, kf;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    kg[e] = fast_exp2((ga - now.g[e]) * LOG2E);
                    kf[e] = 8.f * (fa - now.f[e]);
                }
                f32x4 y[4];
                bool grow = false;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const f32x4 cb = mma(now.x.s, q[u].s, zero4());
                    y[u] = mma(now.x.x1, q[u].x1, mma(now.x.x0, q[u].x0, kf));
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[u][e] = fmaf(cb[e] * kg[e], qg[u], y[u][e]);
                    const float mx = fmaxf(fmaxf(y[u][0], y[u][1]), fmaxf(y[u][2], y[u][3]));
                    grow |= mx * SCALE > mo[u] + GROW;
                }
                if (__any(grow)) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const float mx = SCALE * fmaxf(fmaxf(y[u][0], y[u][1]), fmaxf(y[u][2], y[u][3]));
                        const float to = fmaxf(mo[u], mx);
                        lo[u] *= mo[u] == -__builtin_inff() ? 1.f : fast_exp2(mo[u] - to);
                        mo[u] = to;
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float ref = mo[u] == -__builtin_inff() ? 0.f : mo[u];
#pragma unroll
                    for (int e = 0; e < 4; ++e) lo[u] += fast_exp2(fmaf(y[u][e], SCALE, -ref));
                }
                now = next;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) merge(md[u], ld[u], mo[u] + (fi[u] - fa) * LOG2E, lo[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) merge(md[u], ld[u], __shfl_xor(md[u], o), __shfl_xor(ld[u], o));
        if (grp == 0) sm[w][16 * u + col] = md[u], sl[w][16 * u + col] = ld[u];
    }
    __syncthreads();
    const int r = r0 + lane;
    if (w != 0 || r >= rows.count) return;
    float mt = sm[0][lane], lt = sl[0][lane];
#pragma unroll
    for (int k = 1; k < WG; ++k) merge(mt, lt, sm[k][lane], sl[k][lane]);
    const int Rp = (R + 15) / 16 * 16;
    if (nsplit == 1) {
        lse[(int64_t)bh * Rp + r] = mt + __log2f(lt);
    } else {
        float* part = lse + (int64_t)BH * Rp + 2 * (((int64_t)bh * Rp + r) * nsplit + split);
        part[0] = mt;
        part[1] = lt;
    }
}

// lse of rows whose keys were split: a wave per row, split k with lane k mod 64, the lanes in a fixed tree
__global__ __launch_bounds__(256) void weights_merge_kernel(int64_t rows, int nsplit, float* lse) {
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (r >= rows) return;
    const float* part = lse + rows + 2 * r * nsplit;
    float m = -__builtin_inff(), l = 0.f;
    for (int k = lane; k < nsplit; k += 64) merge(m, l, part[2 * k], part[2 * k + 1]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) merge(m, l, __shfl_xor(m, o), __shfl_xor(l, o));
    if (lane == 0) lse[r] = m + __log2f(l);
}

// Second pass. SHARE waves of a workgroup have the same 64 keys and take every SHARE-th query tile; four, or one where so
// few queries are counted that the keys' loads weigh more.
template <class T, int SHARE>
__global__ __launch_bounds__(64 * WG) void weights_sum_kernel(sisa_attn_weights_args a, int R, const float* lse) {
    __shared__ float part[WG][OWN];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = lane >> 4, col = lane & 15, L = a.L, BH = a.B * a.H;
    const int bh = blockIdx.x % BH, h = bh % a.H, b = bh / a.H;
    const int j0 = (blockIdx.x / BH * (WG / SHARE) + w / SHARE) * OWN;
    const Rows rows = rows_of(a, b);
    const float lam = a.lam[h * a.s_lam];
    const float* le0 = lse + (int64_t)bh * ((R + 15) / 16 * 16) + 4 * grp;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const int from = j0 > rows.first ? (j0 - rows.first) / 16 : 0, tiles = (rows.count + 15) / 16;
    int t = from + w % SHARE;
    if (j0 < rows.n && t < tiles) {
        Tile<T> now = load_tile<T>(a, false, b, h, rows.first + 16 * t, lane);
        f32x4 le = *reinterpret_cast<const f32x4*>(le0 + 16 * t);
        Frags<T> k[4];
        float gj[4], fj[4], kg[4], kf[4];
        const float ga = gate(a.g, b, h, j0 + OWN - 1, L), fa = gate(a.f, b, h, j0 + OWN - 1, L);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            k[u] = frags<T>(a.k, a.b, b, h, j0 + 16 * u, L, lane);
            gj[u] = gate(a.g, b, h, j0 + 16 * u + col, L);
            fj[u] = gate(a.f, b, h, j0 + 16 * u + col, L);
            kg[u] = lam * LOG2E * fast_exp2((ga - gj[u]) * LOG2E);
            kf[u] = (fa - fj[u]) * LOG2E;
        }
        for (; t < tiles; t += SHARE) {
            const int i0 = rows.first + 16 * t, tn = t + SHARE < tiles ? t + SHARE : t;
            const Tile<T> next = load_tile<T>(a, false, b, h, rows.first + 16 * tn, lane);
            const f32x4 le_next = *reinterpret_cast<const f32x4*>(le0 + 16 * tn);
            if (i0 >= j0 + OWN - 1 && i0 + 16 <= rows.n) {
                f32x4 rg, rc;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    rg[e] = fast_exp2((now.g[e] - ga) * LOG2E);
                    rc[e] = fmaf(now.f[e] - fa, LOG2E, -le[e]);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const f32x4 qk = mma(now.x.x1, k[u].x1, mma(now.x.x0, k[u].x0, zero4())), cb = mma(now.x.s, k[u].s, zero4());
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sum[u] += fast_exp2(fmaf(cb[e] * kg[u], rg[e], fmaf(qk[e], SCALE, kf[u])) + rc[e]);
                }
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (j0 + 16 * u > i0 + 15) continue;             // all keys after all queries
                    const f32x4 qk = mma(now.x.x1, k[u].x1, mma(now.x.x0, k[u].x0, zero4())), cb = mma(now.x.s, k[u].s, zero4());
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = i0 + 4 * grp + e;
                        const float dec = lam * fast_exp2((now.g[e] - gj[u]) * LOG2E);
                        const float x = fmaf(qk[e], 0.125f, dec * cb[e]) + (now.f[e] - fj[u]);
                        const float p = fast_exp2(fmaf(x, LOG2E, -le[e]));
                        sum[u] += i >= j0 + 16 * u + col && i < rows.n ? p : 0.f;
                    }
                }
            }
            now = next;
            le = le_next;
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) sum[u] += __shfl_xor(sum[u], o);
        if (grp == 0) part[w][16 * u + col] = sum[u];
    }
    __syncthreads();
    const int j = j0 + lane;
    if (w % SHARE || j >= L) return;
    float s = part[w][lane];
#pragma unroll
    for (int k = 1; k < SHARE; ++k) s += part[w + k][lane];
    a.out[(int64_t)bh * L + j] = j < rows.n ? s : 0.f;
}

int window_of(int32_t L, int32_t window) { return window && window < L ? window : L; }

int64_t pad16(int64_t R) { return (R + 15) / 16 * 16; }

// Splits of the keys in the first pass: enough workgroups for the chip where few queries are counted, of 256 keys at least.
int splits_of(int64_t BH, int32_t L, int32_t R) {
    const int64_t groups = BH * sisa::cdiv(R, OWN), most = sisa::cdiv(L, 256);
    const int64_t want = groups >= 1024 ? 1 : sisa::cdiv(1024, groups);
    return (int)(want < most ? want : most);
}

// Up to this many query tiles each wave of the second pass has keys of its own.
constexpr int FEW_TILES = 16;

template <class T>
int launch_weights(const sisa_attn_weights_args* a, hipStream_t st) {
    const int R = window_of(a->L, a->window);
    const int64_t BH = (int64_t)a->B * a->H;
    const int nsplit = splits_of(BH, a->L, R);
    float* lse = (float*)a->workspace;
    weights_lse_kernel<T><<<(unsigned)(BH * sisa::cdiv(R, OWN) * nsplit), 64 * WG, 0, st>>>(*a, R, nsplit, lse);
    int rc = sisa::launch_status("sisa_attn_weights (rows)");
    if (rc) return rc;
    if (nsplit > 1) {
        weights_merge_kernel<<<(unsigned)sisa::cdiv(BH * pad16(R), 4), 256, 0, st>>>(BH * pad16(R), nsplit, lse);
        rc = sisa::launch_status("sisa_attn_weights (merge)");
        if (rc) return rc;
    }
    if (R <= 16 * FEW_TILES) weights_sum_kernel<T, 1><<<(unsigned)(BH * sisa::cdiv(a->L, OWN * WG)), 64 * WG, 0, st>>>(*a, R, lse);
    else weights_sum_kernel<T, WG><<<(unsigned)(BH * sisa::cdiv(a->L, OWN)), 64 * WG, 0, st>>>(*a, R, lse);
    return sisa::launch_status("sisa_attn_weights");
}

}  // namespace

extern "C" int64_t sisa_attn_weights_workspace_bytes(int32_t B, int32_t H, int32_t L, int32_t window) {
    if (B < 1 || H < 1 || L < 1 || window < 0) return 0;
    const int R = window_of(L, window), nsplit = splits_of((int64_t)B * H, L, R);
    return (int64_t)B * H * pad16(R) * (nsplit > 1 ? 1 + 2 * nsplit : 1) * (int64_t)sizeof(float);
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
    SISA_REQUIRE(a->g.ptr && a->lam && a->out && a->workspace, "sisa_attn_weights: null pointer");
    const int64_t BH = (int64_t)a->B * a->H;
    SISA_REQUIRE(BH * sisa::cdiv(a->L, 64) < ((int64_t)1 << 26), "sisa_attn_weights: B*H*L too large for one launch");
    hipStream_t st = (hipStream_t)stream;
    switch (a->dtype) {
        case SISA_BF16: return launch_weights<__bf16>(a, st);
        case SISA_F16: return launch_weights<_Float16>(a, st);
        default: return launch_weights<float>(a, st);
    }
}
