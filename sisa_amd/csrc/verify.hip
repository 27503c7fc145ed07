// Verification of drafted tokens for gfx950 (include/sisa_hip_branch.h).
//
//   accept draft i while u_i q_i(x_i) < p_i(x_i);  then  token = min { v : sum_{w <= v} t_w > r sum_w t_w },  t = max(p_i - q_i, 0)
//
// Two launches. In the first, every workgroup of a row decides its drafts side by side (two dependent loads), the first refused
// one ending them, and its waves sum up the weights of 1,024 tokens each, of the differences and of p alone. In the second a
// workgroup a row finds the 1,024 tokens whose sum passes r times the whole, and in them the token. Weights are fp64: exact
// differences, exact products in the decisions, and a token's border off by 2^-50 or so.
//
// A row on one CU, in one launch, was bound by the conversions to fp64: a row of 50,277 tokens 16.8 us, 64 rows 21.1, 200 rows
// of bf16 without q 14.0.
#include "common.h"
#include "host.h"
#include "sisa_hip_branch.h"

namespace {

constexpr int NW = 4, NTH = 64 * NW;
constexpr int E = 4;                   // tokens of a lane's load
constexpr int LOADS = 4;               // of a lane
constexpr int CHUNK = 64 * E * LOADS;  // tokens of a wave
static_assert(CHUNK == E * NTH, "the second launch has a load for each thread");

struct Sums { double rest, p; };       // of a chunk's weights max(p - q, 0), and of max(p, 0)

// Four neighbouring tokens, wherever a row begins: global memory takes loads of any alignment.
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Four { vec4<T> v; };
template <class T> SISA_DEV vec4<T> load_four(const T* row, int v, int V) {
    if (v + E <= V) return reinterpret_cast<const Four<T>*>(row + v)->v;
    vec4<T> x;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = v + e < V ? row[v + e] : (T)0.f;
    return x;
}
// max(x, 0), and what is not a number stays so
SISA_DEV double positive(double x) { return x > 0. || x != x ? x : 0.; }

SISA_DEV double shuffle_up(double x, int d) { return __shfl_up(x, d); }
// The sums over a wave up to each lane.
SISA_DEV double scan(double x, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double y = shuffle_up(x, o);
        if (lane >= o) x += y;
    }
    return x;
}

SISA_DEV int drafts_of(const sisa_verify_args& a, int64_t n) {
    const int given = a.counts ? a.counts[n] : a.K;
    return given < 0 ? 0 : given > a.K ? a.K : given;
}

template <class TP, class TQ>
__global__ __launch_bounds__(NTH) void verify_sum_kernel(sisa_verify_args a, unsigned groups, unsigned chunks, Sums* sums) {
    __shared__ int refused;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned n32 = blockIdx.x / groups, group = blockIdx.x - n32 * groups;
    const int64_t n = n32;
    const int V = a.V, count = drafts_of(a, n);
    if (tid == 0) refused = count;
    __syncthreads();
    for (int i = tid; i < count; i += NTH) {
        const int64_t x = a.drafts[n * a.d_b + i * a.d_k];
        const float u = a.u[n * a.u_b + i * a.u_k];
        bool took = false;
        if (x >= 0 && x < V) {
            const double p = (double)(float)((const TP*)a.p)[n * a.p_b + i * a.p_k + x];
            const double q = a.q ? (double)(float)((const TQ*)a.q)[n * a.q_b + i * a.q_k + x] : 1.;
            took = (double)u * q < p;
        }
        if (!took) atomicMin(&refused, i);
    }
    __syncthreads();
    const int i = refused;
    if (group == 0 && tid == 0) a.accepted[n] = i;
    const TP* p = (const TP*)a.p + n * a.p_b + i * a.p_k;
    const TQ* q = i < count && a.q ? (const TQ*)a.q + n * a.q_b + i * a.q_k : nullptr;
    const int64_t draft = i < count && !a.q ? a.drafts[n * a.d_b + i * a.d_k] : -1;
    const unsigned chunk = group * NW + w;
    if (chunk < chunks) {
        const int v0 = chunk * CHUNK + E * lane;
        vec4<TP> xp[LOADS];
        vec4<TQ> xq[LOADS];
#pragma unroll
        for (int k = 0; k < LOADS; ++k) {
            xp[k] = load_four<TP>(p, v0 + 64 * E * k, V);
            if (q) xq[k] = load_four<TQ>(q, v0 + 64 * E * k, V);
        }
        // what is not a number is found in fp32 and makes the sums NaN: fp64 comparisons cost as much as the sums
        Sums s{0., 0.};
        bool bad = false;
        if (q) {
#pragma unroll
            for (int k = 0; k < LOADS; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x = (float)xp[k][e], y = (float)xq[k][e];
                    bad |= x - y != x - y;               // of infinities on both sides, too
                    s.p += __builtin_fmax((double)x, 0.);
                    s.rest += __builtin_fmax((double)x - (double)y, 0.);
                }
        } else {
            double out = 0.;                             // the draft's own weight
#pragma unroll
            for (int k = 0; k < LOADS; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x = (float)xp[k][e];
                    const bool drafted = v0 + 64 * E * k + e == draft;
                    bad |= x != x;
                    s.rest += __builtin_fmax((double)(drafted ? 0.f : x), 0.);
                    if (drafted) out = __builtin_fmax((double)x, 0.);
                }
            s.p = s.rest + out;
        }
        if (bad) s.rest = s.p = __builtin_nan("");
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s.rest += __shfl_xor(s.rest, o), s.p += __shfl_xor(s.p, o);
        if (lane == 0) sums[n * chunks + chunk] = s;
    }
}

template <class TP, class TQ>
__global__ __launch_bounds__(NTH) void verify_find_kernel(sisa_verify_args a, unsigned chunks, const Sums* sums) {
    __shared__ double part[2][NW], before;
    __shared__ int owner, last;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t n = blockIdx.x;
    const int V = a.V, K = a.K, count = drafts_of(a, n), i = a.accepted[n];
    const double r = (double)a.u[n * a.u_b + K * a.u_k];
    // each thread's neighbouring chunks
    const unsigned each = (chunks + NTH - 1) / NTH, c0 = tid * each, c1 = c0 + each < chunks ? c0 + each : chunks;
    const Sums* S = sums + n * chunks;
    Sums mine{0., 0.};
    for (unsigned c = c0; c < c1; ++c) mine.rest += S[c].rest, mine.p += S[c].p;
    const TP* p = (const TP*)a.p + n * a.p_b + i * a.p_k;
    const TQ* q = i < count && a.q ? (const TQ*)a.q + n * a.q_b + i * a.q_k : nullptr;
    int64_t draft = i < count && !a.q ? a.drafts[n * a.d_b + i * a.d_k] : -1;
    double up = scan(mine.rest, lane);
    const double up_p = scan(mine.p, lane);
    if (lane == 63) part[0][w] = up, part[1][w] = up_p;
    if (tid == 0) owner = (int)chunks, last = -1;
    __syncthreads();
    double total = 0., total_p = 0., ahead = 0., ahead_p = 0.;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
        if (k == w) ahead = total, ahead_p = total_p;
        total += part[0][k], total_p += part[1][k];
    }
    const bool plain = total == 0.;                      // no weight is left of the differences
    if (plain) total = total_p, ahead = ahead_p, up = up_p, q = nullptr, draft = -1;
    int token = -1;
    if (total - total == 0. && total > 0.) {
        auto sum_of = [&](unsigned c) { return plain ? S[c].p : S[c].rest; };
        const double own = plain ? mine.p : mine.rest, goal = r * total < 0. ? 0. : r * total;
        // the first chunk that passes the goal; where none does (rounding, or r of 1 and more), the last with any weight
        if (ahead + up > goal && c0 < c1) {
            double run = ahead + up - own;
            for (unsigned c = c0; c < c1; ++c) {
                const double x = sum_of(c);
                if (x > 0. && run + x > goal) {
                    atomicMin(&owner, (int)c);
                    break;
                }
                run += x;
            }
        }
        for (unsigned c = c1; c > c0; --c)
            if (sum_of(c - 1) > 0.) {
                atomicMax(&last, (int)c - 1);
                break;
            }
        __syncthreads();
        const bool passes = owner < (int)chunks;
        const unsigned c = passes ? owner : last;
        if (c >= c0 && c < c1) {
            double run = ahead + up - own;
            for (unsigned k = c0; k < c; ++k) run += sum_of(k);
            before = run;
        }
        __syncthreads();
        const double run = before;
        __syncthreads();
        if (tid == 0) owner = V, last = -1;
        const int v = c * CHUNK + E * tid;
        double y[E], all = 0.;
        const vec4<TP> xp = load_four<TP>(p, v, V);
        vec4<TQ> xq;
        if (q) xq = load_four<TQ>(q, v, V);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            double x = (double)(float)xp[e];
            if (q) x -= (double)(float)xq[e];
            y[e] = v + e == draft ? 0. : positive(x);
            all += y[e];
        }
        const double upto = scan(all, lane);
        if (lane == 63) part[0][w] = upto;
        __syncthreads();
        double at = run + (upto - all);
#pragma unroll
        for (int k = 0; k < NW; ++k)
            if (k < w) at += part[0][k];
        int hit = V, has = -1;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            at += y[e];
            if (y[e] > 0.) {
                has = v + e;
                if (passes && at > goal && hit == V) hit = v + e;
            }
        }
        const uint64_t hits = __ballot(hit < V), some = __ballot(has >= 0);
        if (hits && lane == __builtin_ctzll(hits)) atomicMin(&owner, hit);
        if (some && lane == 63 - __builtin_clzll(some)) atomicMax(&last, has);
        __syncthreads();
        token = owner < V ? owner : last;
    }
    for (int k = tid; k <= K; k += NTH) a.tokens[n * (K + 1) + k] = k < i ? a.drafts[n * a.d_b + k * a.d_k] : k == i ? token : -1;
}

// Workgroups of a row: a chunk a wave (2,600 workgroups: 11.4 us, the same work in 1,200 12.0, in 600 14.3).
unsigned groups_of(int64_t chunks) { return (unsigned)sisa::cdiv(chunks, NW); }

template <class TP, class TQ>
int launch(const sisa_verify_args* a, hipStream_t st) {
    const unsigned chunks = (unsigned)sisa::cdiv(a->V, CHUNK), groups = groups_of(chunks);
    verify_sum_kernel<TP, TQ><<<(unsigned)a->B * groups, NTH, 0, st>>>(*a, groups, chunks, (Sums*)a->workspace);
    const int rc = sisa::launch_status("sisa_verify");
    if (rc) return rc;
    verify_find_kernel<TP, TQ><<<(unsigned)a->B, NTH, 0, st>>>(*a, chunks, (const Sums*)a->workspace);
    return sisa::launch_status("sisa_verify (token)");
}
template <class TP>
int launch(const sisa_verify_args* a, hipStream_t st) {
    if (!a->q || a->q_dtype == a->p_dtype) return launch<TP, TP>(a, st);
    switch (a->q_dtype) {
        case SISA_BF16: return launch<TP, __bf16>(a, st);
        case SISA_F16: return launch<TP, _Float16>(a, st);
        default: return launch<TP, float>(a, st);
    }
}

bool type_ok(int t) { return t == SISA_F32 || t == SISA_BF16 || t == SISA_F16; }

}  // namespace

extern "C" int64_t sisa_verify_workspace_bytes(int32_t B, int32_t V) {
    return B < 1 || V < 1 || V > SISA_VERIFY_MAX_V ? 0 : B * sisa::cdiv(V, CHUNK) * (int64_t)sizeof(Sums);
}

extern "C" int sisa_verify(const sisa_verify_args* a, void* stream) {
    SISA_REQUIRE(a != nullptr, "sisa_verify: null args");
    SISA_REQUIRE(a->B >= 0 && a->K >= 0 && a->V >= 1 && a->V <= SISA_VERIFY_MAX_V && a->B <= (1 << 21) && a->K <= (1 << 20),
                 "sisa_verify: bad shape B=%d K=%d V=%d (at most 2^21 rows, 2^20 drafts and 2^24 tokens)", a->B, a->K, a->V);
    if (a->B == 0) return SISA_OK;
    SISA_REQUIRE((int64_t)a->B * groups_of(sisa::cdiv(a->V, CHUNK)) * NTH <= sisa::MAX_THREADS, "sisa_verify: B=%d rows of V=%d: too large for one launch",
                 a->B, a->V);
    SISA_REQUIRE(a->workspace && sisa::aligned16(a->workspace), "sisa_verify: null workspace, or not 16-byte aligned");
    SISA_REQUIRE(type_ok(a->p_dtype) && (!a->q || type_ok(a->q_dtype)), "sisa_verify: p and q must be fp32, bf16 or fp16");
    SISA_REQUIRE(a->p && (a->drafts || a->K == 0) && a->u && a->tokens && a->accepted, "sisa_verify: null pointer");
    hipStream_t st = (hipStream_t)stream;
    switch (a->p_dtype) {
        case SISA_BF16: return launch<__bf16>(a, st);
        case SISA_F16: return launch<_Float16>(a, st);
        default: return launch<float>(a, st);
    }
}
