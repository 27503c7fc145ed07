// The attention weights that a prompt's positions receive, summed over its last queries, for gfx950
// (include/sisa_hip_cache.h): w_j = sum over i >= j in the window of exp(s_ij - lse_i).
//
//   s_ij = q_i.k_j / 8 + lam exp(g_i - g_j) (c_i.b_j) + (F_i - F_j)
//
// Two passes over the scores, neither of which keeps them: the queries' log-sum-exp over their keys, then every key's sum
// over its queries. Scores are 16x16 MFMA blocks with K = 64 (q.k) and 32 (c.b). A wave holds 64 queries (keys) in
// registers and streams 16 keys (queries) at a time straight from memory, which L2 serves; the workgroup's four waves share
// the 64 and take every fourth of the 16s. In the first pass a lane owns one query per block (the keys are the block's
// rows), in the second one key, so that the running statistics need no lane exchange before the end. Log2 units throughout.
#include "common.h"
#include "host.h"
#include "sisa_hip_cache.h"

namespace {

constexpr int DH = 64, DS = 32;
constexpr int WG = 4;                 // waves per workgroup
constexpr int OWN = 64;               // queries (keys) that a workgroup owns: four blocks of 16

struct Rows {                         // queries of a sequence: first .. first + count - 1
    int n, first, count;
};

SISA_DEV Rows rows_of(const sisa_attn_weights_args& a, int b) {
    int n = a.lengths ? a.lengths[b] : a.L;
    n = n < 0 ? 0 : n > a.L ? a.L : n;
    const int count = a.window && a.window < n ? a.window : n;
    return Rows{n, n - count, count};
}

template <class T> struct Frags { frag8<T> x0, x1, s; };      // features 0..31, 32..63 and the state's 0..31

// The operand of 16 positions r0 .. (lane % 16), positions beyond the last one of the view as the last one.
template <class T>
SISA_DEV Frags<T> frags(const sisa_view& x, const sisa_view& s, int b, int h, int r0, int L, int lane) {
    const int row = r0 + (lane & 15) < L ? r0 + (lane & 15) : L - 1, f = 8 * (lane >> 4);
    const T* p = (const T*)x.ptr + b * x.sb + h * x.sh + row * x.sl;
    const T* q = (const T*)s.ptr + b * s.sb + h * s.sh + row * s.sl;
    return Frags<T>{load8<T>(p + f), load8<T>(p + 32 + f), load8<T>(q + f)};
}

SISA_DEV float gate(const sisa_view& v, int b, int h, int r, int L) {
    return ((const float*)v.ptr)[b * v.sb + h * v.sh + (int64_t)(r < L ? r : L - 1) * v.sl];
}

// (m, l) of two parts of a row, log2 units
SISA_DEV void merge(float& m, float& l, float m2, float l2) {
    const float t = fmaxf(m, m2), ref = t == -__builtin_inff() ? 0.f : t;
    l = l * (m == -__builtin_inff() ? 1.f : exp2f(m - ref)) + l2 * (m2 == -__builtin_inff() ? 1.f : exp2f(m2 - ref));
    m = t;
}

template <class T>
__global__ __launch_bounds__(64 * WG) void weights_lse_kernel(sisa_attn_weights_args a, int R, int nsplit, float* lse) {
    __shared__ float sm[WG][OWN], sl[WG][OWN];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = lane >> 4, col = lane & 15, L = a.L;
    const int blocks = (R + OWN - 1) / OWN;
    const int split = blockIdx.x % nsplit, rest = blockIdx.x / nsplit;
    const int r0 = (blocks - 1 - rest % blocks) * OWN, bh = rest / blocks, h = bh % a.H, b = bh / a.H;
    const Rows rows = rows_of(a, b);
    if (r0 >= rows.count) return;
    const int i0 = rows.first + r0;
    const bool has_f = a.f.ptr != nullptr;
    const float lam = a.lam[h * a.s_lam];
    Frags<T> q[4];
    float gi[4], fi[4], m[4], l[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        q[u] = frags<T>(a.q, a.c, b, h, i0 + 16 * u, L, lane);
        gi[u] = gate(a.g, b, h, i0 + 16 * u + col, L);
        fi[u] = has_f ? gate(a.f, b, h, i0 + 16 * u + col, L) : 0.f;
        m[u] = -__builtin_inff();
        l[u] = 0.f;
    }
    const int last = i0 + OWN < rows.n ? i0 + OWN : rows.n;    // keys 0 .. last - 1
    const int tiles = (last + 15) / 16, per = (tiles + nsplit - 1) / nsplit;
    const int t1 = (split + 1) * per < tiles ? (split + 1) * per : tiles;
    for (int t = split * per + w; t < t1; t += WG) {
        const Frags<T> k = frags<T>(a.k, a.b, b, h, 16 * t, L, lane);
        float gj[4], fj[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            gj[e] = gate(a.g, b, h, 16 * t + 4 * grp + e, L);
            fj[e] = has_f ? gate(a.f, b, h, 16 * t + 4 * grp + e, L) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const f32x4 qk = mma(k.x1, q[u].x1, mma(k.x0, q[u].x0, zero4())), cb = mma(k.s, q[u].s, zero4());
            float x[4], t4 = m[u];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float dec = lam * exp2f((gi[u] - gj[e]) * LOG2E);
                x[e] = (fmaf(qk[e], 0.125f, dec * cb[e]) + (fi[u] - fj[e])) * LOG2E;
                if (16 * t + 4 * grp + e > i0 + 16 * u + col) x[e] = -__builtin_inff();
                t4 = fmaxf(t4, x[e]);
            }
            const float ref = t4 == -__builtin_inff() ? 0.f : t4;
            l[u] *= m[u] == -__builtin_inff() ? 1.f : exp2f(m[u] - ref);
#pragma unroll
            for (int e = 0; e < 4; ++e) l[u] += exp2f(x[e] - ref);
            m[u] = t4;
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) merge(m[u], l[u], __shfl_xor(m[u], o), __shfl_xor(l[u], o));
        if (grp == 0) sm[w][16 * u + col] = m[u], sl[w][16 * u + col] = l[u];
    }
    __syncthreads();
    const int r = r0 + lane;
    if (w != 0 || r >= rows.count) return;
    float mt = sm[0][lane], lt = sl[0][lane];
#pragma unroll
    for (int k = 1; k < WG; ++k) merge(mt, lt, sm[k][lane], sl[k][lane]);
    if (nsplit == 1) {
        lse[(int64_t)bh * R + r] = mt + log2f(lt);
    } else {
        float* part = lse + (int64_t)a.B * a.H * R + 2 * (((int64_t)bh * R + r) * nsplit + split);
        part[0] = mt;
        part[1] = lt;
    }
}

// lse of rows whose keys were split, the splits in order
__global__ __launch_bounds__(256) void weights_merge_kernel(int64_t rows, int nsplit, float* lse) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    const float* part = lse + rows + 2 * r * nsplit;
    float m = part[0], l = part[1];
    for (int k = 1; k < nsplit; ++k) merge(m, l, part[2 * k], part[2 * k + 1]);
    lse[r] = m + log2f(l);
}

template <class T>
__global__ __launch_bounds__(64 * WG) void weights_sum_kernel(sisa_attn_weights_args a, int R, const float* lse) {
    __shared__ float part[WG][OWN];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = lane >> 4, col = lane & 15, L = a.L;
    const int blocks = (L + OWN - 1) / OWN;
    const int j0 = (blockIdx.x % blocks) * OWN, bh = blockIdx.x / blocks, h = bh % a.H, b = bh / a.H;
    const Rows rows = rows_of(a, b);
    const bool has_f = a.f.ptr != nullptr;
    const float lam = a.lam[h * a.s_lam];
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    if (j0 < rows.n) {
        Frags<T> k[4];
        float gj[4], fj[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            k[u] = frags<T>(a.k, a.b, b, h, j0 + 16 * u, L, lane);
            gj[u] = gate(a.g, b, h, j0 + 16 * u + col, L);
            fj[u] = has_f ? gate(a.f, b, h, j0 + 16 * u + col, L) : 0.f;
        }
        // 16-query tiles of the window from the first that reaches j0
        const int from = j0 > rows.first ? (j0 - rows.first) / 16 : 0, tiles = (rows.count + 15) / 16;
        for (int t = from + w; t < tiles; t += WG) {
            const int i0 = rows.first + 16 * t;
            const Frags<T> q = frags<T>(a.q, a.c, b, h, i0, L, lane);
            float gi[4], fi[4], le[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 16 * t + 4 * grp + e;
                gi[e] = gate(a.g, b, h, i0 + 4 * grp + e, L);
                fi[e] = has_f ? gate(a.f, b, h, i0 + 4 * grp + e, L) : 0.f;
                le[e] = lse[(int64_t)bh * R + (r < rows.count ? r : rows.count - 1)];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const f32x4 qk = mma(q.x1, k[u].x1, mma(q.x0, k[u].x0, zero4())), cb = mma(q.s, k[u].s, zero4());
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = i0 + 4 * grp + e;
                    const float dec = lam * exp2f((gi[e] - gj[u]) * LOG2E);
                    const float x = fmaf(qk[e], 0.125f, dec * cb[e]) + (fi[e] - fj[u]);
                    const float p = exp2f(fmaf(x, LOG2E, -le[e]));
                    sum[u] += i >= j0 + 16 * u + col && i < rows.n ? p : 0.f;
                }
            }
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
    if (w == 0 && j < L)
        a.out[(int64_t)bh * L + j] = j < rows.n ? (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]) : 0.f;
}

int window_of(int32_t L, int32_t window) { return window && window < L ? window : L; }

// Splits of the keys in the first pass: enough workgroups for the chip where few queries are counted, of 256 keys at least.
int splits_of(int64_t BH, int32_t L, int32_t R) {
    const int64_t groups = BH * sisa::cdiv(R, OWN), most = sisa::cdiv(L, 256);
    const int64_t want = groups >= 1024 ? 1 : sisa::cdiv(1024, groups);
    return (int)(want < most ? want : most);
}

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
        weights_merge_kernel<<<(unsigned)sisa::cdiv(BH * R, 256), 256, 0, st>>>(BH * R, nsplit, lse);
        rc = sisa::launch_status("sisa_attn_weights (merge)");
        if (rc) return rc;
    }
    weights_sum_kernel<T><<<(unsigned)(BH * sisa::cdiv(a->L, OWN)), 64 * WG, 0, st>>>(*a, R, lse);
    return sisa::launch_status("sisa_attn_weights");
}

}  // namespace

extern "C" int64_t sisa_attn_weights_workspace_bytes(int32_t B, int32_t H, int32_t L, int32_t window) {
    if (B < 1 || H < 1 || L < 1 || window < 0) return 0;
    const int R = window_of(L, window), nsplit = splits_of((int64_t)B * H, L, R);
    return (int64_t)B * H * R * (nsplit > 1 ? 1 + 2 * nsplit : 1) * (int64_t)sizeof(float);
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
