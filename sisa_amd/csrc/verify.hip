// Verification of drafted tokens for gfx950 (include/sisa_hip_branch.h).
//
// A workgroup per row: the drafts are decided side by side, the first refused one ends them; then the vocabulary of one
// position is gone through twice, for the sum of the weights and, in the wave whose part holds it, for the token.
#include "common.h"
#include "host.h"
#include "sisa_hip_branch.h"

namespace {

constexpr int NW = 16, NTH = 64 * NW;

template <class T> SISA_DEV double at(const void* p, int64_t i) { return (double)(float)((const T*)p)[i]; }

template <class TP, class TQ>
__global__ __launch_bounds__(NTH) void verify_kernel(sisa_verify_args a) {
    __shared__ int refused;
    __shared__ double sums[NW];
    __shared__ int found[NW];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = blockIdx.x, V = a.V, K = a.K;
    const int given = a.counts ? a.counts[n] : K, count = given < 0 ? 0 : given > K ? K : given;
    if (tid == 0) refused = count;
    __syncthreads();
    for (int i = tid; i < count; i += NTH) {
        const int64_t x = a.drafts[n * a.d_b + i * a.d_k];
        bool took = false;
        if (x >= 0 && x < V) {
            const double p = at<TP>(a.p, n * a.p_b + i * a.p_k + x), q = a.q ? at<TQ>(a.q, n * a.q_b + i * a.q_k + x) : 1.0;
            took = (double)a.u[n * a.u_b + i * a.u_k] * q < p;
        }
        if (!took) atomicMin(&refused, i);
    }
    __syncthreads();
    const int i = refused;
    const double r = (double)a.u[n * a.u_b + K * a.u_k];
    const int64_t draft = i < count ? a.drafts[n * a.d_b + i * a.d_k] : -1;
    const int64_t prow = n * a.p_b + i * a.p_k, qrow = n * a.q_b + i * a.q_k;
    const int seg = ((V + NW - 1) / NW + 63) / 64 * 64, from = w * seg < V ? w * seg : V, to = from + seg < V ? from + seg : V;
    int token = -1;
    for (int plain = i < count ? 0 : 1; plain < 2; ++plain) {        // the differences, then the probabilities
        auto weight = [&](int v) -> double {
            const double p = at<TP>(a.p, prow + v);
            if (plain) return p > 0. || p != p ? p : 0.;
            if (!a.q) return v == draft || !(p > 0. || p != p) ? 0. : p;
            const double d = p - at<TQ>(a.q, qrow + v);
            return d > 0. || d != d ? d : 0.;
        };
        double s = 0.;
        for (int v = from + lane; v < to; v += 64) s += weight(v);
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (lane == 0) sums[w] = s;
        __syncthreads();
        // the part whose sum passes r * total, or else (rounding, or r of 1 and more) every part: its last token counts
        double total = 0.;
        for (int k = 0; k < NW; ++k) total += sums[k];
        const bool fine = total - total == 0.;
        if (fine && total > 0.) {
            const double goal = r * total;
            int owner = -1;
            double run = 0., upto = 0.;
            for (int k = 0; k < NW; ++k) {
                if (owner < 0 && upto + sums[k] > goal) owner = k, run = upto;
                upto += sums[k];
            }
            int hit = -1;
            if (owner < 0 || owner == w) {
                int last = -1;
                for (int v0 = from; v0 < to && hit < 0; v0 += 64) {
                    const double x = v0 + lane < to ? weight(v0 + lane) : 0.;
                    double up = x;
                    for (int o = 1; o < 64; o <<= 1) {
                        const double y = __shfl_up(up, o);
                        if (lane >= o) up += y;
                    }
                    const uint64_t some = __ballot(x > 0.), over = __ballot(owner == w && x > 0. && run + up > goal);
                    if (over) hit = v0 + __builtin_ctzll(over);
                    if (some) last = v0 + 63 - __builtin_clzll(some);
                    run += __shfl(up, 63);
                }
                hit = hit >= 0 ? hit : last;
            }
            if (lane == 0) found[w] = hit;
            __syncthreads();
            for (int k = 0; k < NW; ++k) token = found[k] >= 0 ? found[k] : token;
            break;
        }
        if (!fine) break;
        __syncthreads();
    }
    for (int k = tid; k <= K; k += NTH)
        a.tokens[(int64_t)n * (K + 1) + k] = k < i ? a.drafts[n * a.d_b + k * a.d_k] : k == i ? token : -1;
    if (tid == 0) a.accepted[n] = i;
}

template <class TP, class TQ>
int launch(const sisa_verify_args* a, hipStream_t st) {
    verify_kernel<TP, TQ><<<(unsigned)a->B, NTH, 0, st>>>(*a);
    return sisa::launch_status("sisa_verify");
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

extern "C" int64_t sisa_verify_workspace_bytes(int32_t, int32_t) { return 0; }

extern "C" int sisa_verify(const sisa_verify_args* a, void* stream) {
    SISA_REQUIRE(a != nullptr, "sisa_verify: null args");
    SISA_REQUIRE(a->B >= 0 && a->K >= 0 && a->V >= 1 && a->V <= SISA_VERIFY_MAX_V && a->B <= (1 << 21) && a->K <= (1 << 20),
                 "sisa_verify: bad shape B=%d K=%d V=%d (at most 2^21 rows, 2^20 drafts and 2^24 tokens)", a->B, a->K, a->V);
    if (a->B == 0) return SISA_OK;
    SISA_REQUIRE(type_ok(a->p_dtype) && (!a->q || type_ok(a->q_dtype)), "sisa_verify: p and q must be fp32, bf16 or fp16");
    SISA_REQUIRE(a->p && (a->drafts || a->K == 0) && a->u && a->tokens && a->accepted, "sisa_verify: null pointer");
    hipStream_t st = (hipStream_t)stream;
    switch (a->p_dtype) {
        case SISA_BF16: return launch<__bf16>(a, st);
        case SISA_F16: return launch<_Float16>(a, st);
        default: return launch<float>(a, st);
    }
}
