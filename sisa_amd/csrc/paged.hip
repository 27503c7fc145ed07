// A generation cache in pages for gfx950: writing new positions, and the attention of new tokens over the pages, split
// over the positions and joined (include/sisa_hip_cache.h).
//
//   s_mj = q_m.k_j / 8 + lam exp(g_m - g_j) (c_m.b_j) + (F_m - F_j),  j <= n - M + m;   out_m = softmax_j(s_mj) v_j
//
// Both are bound by memory: (160 es + 8) bytes a position and head, 328 in 16 bits, read (and written) once.
#include "pages.h"

namespace {

constexpr int DH = 64, DS = 32;

// ------------------------------------------------------------------------------------------------ write
// A wave moves ROWS rows, numbered with the positions of a head as neighbours: a prompt's rows of a head become neighbours
// in a page.
template <class T, int ROWS>
__global__ __launch_bounds__(256) void paged_write_kernel(sisa_paged_write_args a, int shift) {
    const int lane = threadIdx.x & 63;
    const unsigned id = (blockIdx.x * 4 + (threadIdx.x >> 6)) * ROWS + lane, M = a.M, H = a.pool.heads;
    const unsigned m = id % M, nh = id / M, h = nh % H;
    const int64_t n = nh / H;
    int64_t pos = 0;
    int page = -1;
    if (lane < ROWS && n < a.B && (!a.count || (int)m < a.count[n])) {
        pos = (int64_t)a.start[n] + m;
        page = page_of(a.table + n * a.s_table, a.W, shift, a.pool.pages, pos);
    }
    move_rows<T, ROWS>(RowViews{a.k, a.v, a.b, a.g, a.f}, rows_of_pool(a.pool), page >= 0, n, page, h, m,
                       pos & (a.pool.page_size - 1), lane);
}

template <class T>
void launch_write(const sisa_paged_write_args* a, int64_t rows, hipStream_t st) {
    const int shift = sisa::log2_of(a->pool.page_size), per = 4 * sisa::rows_per_wave(rows);
    const unsigned grid = (unsigned)sisa::cdiv(rows, per);
    if (per == 256) paged_write_kernel<T, 64><<<grid, 256, 0, st>>>(*a, shift);
    else paged_write_kernel<T, 8><<<grid, 256, 0, st>>>(*a, shift);
}

// ------------------------------------------------------------------------------------------------ decode
constexpr int DW = 4;                 // waves per workgroup
constexpr int KCH = 64 * DW;          // positions per chunk (workgroup)
constexpr int PART = DH + 2;          // chunk partial: max, sum, out[64]
constexpr int PIECE = 1024;           // positions of tracked weights per workgroup of the join

// Positions that query row m of a sequence of n sees, or -1 for a length that the call does not take.
SISA_DEV int visible(int n, int max_len, int64_t held, int M, int m) {
    if (n < 0 || n > max_len || n > held) return -1;
    const int last = n - M + m + 1;
    return last > 0 ? last : 0;
}

// One workgroup per (query row, chunk of 256 positions), a wave per 64 of them; 8 neighbouring lanes share a position (8
// features each), so that every load covers whole 128-byte rows. A group of 8 positions lies in one page.
template <class T, bool TRACK>
__global__ __launch_bounds__(64 * DW) void paged_chunk_kernel(sisa_paged_decode_args a, int shift, int nchunk, float* part,
                                                             float* scores) {
    __shared__ float wm[DW], wl[DW], wo[DW][DH];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int fg = lane & 7, kq = lane >> 3;
    const int chunk = blockIdx.x % nchunk, row = blockIdx.x / nchunk;
    const int H = a.pool.heads, m = row % a.M, nh = row / a.M, h = nh % H, n = nh / H;
    const int vis = visible(a.lengths[n], a.max_len, (int64_t)a.W << shift, a.M, m);
    if (chunk * KCH >= vis) return;                    // nothing here: the join does not read this partial
    const int jw = chunk * KCH + w * 64;
    const int32_t* table = a.table + n * a.s_table;
    const sisa_page_pool& P = a.pool;
    const int mask = P.page_size - 1;
    // lane i < 8: the page of positions jw + 8 i .. + 7, -1 where there are none or no such page
    int pg = -1;
    if (lane < 8 && jw + 8 * lane < vis) pg = page_of(table, a.W, shift, P.pages, jw + 8 * lane);
    const T* Q = (const T*)a.q.ptr + n * a.q.sb + h * a.q.sh + m * a.q.sl;
    const T* C = (const T*)a.c.ptr + n * a.c.sb + h * a.c.sh + m * a.c.sl;
    const float gq = ((const float*)a.gq.ptr)[n * a.gq.sb + h * a.gq.sh + m * a.gq.sl];
    const bool has_f = P.f.ptr != nullptr;
    const float fq = has_f ? ((const float*)a.fq.ptr)[n * a.fq.sb + h * a.fq.sh + m * a.fq.sl] : 0.f;
    const float lam = a.lam[h * a.s_lam];

    frag8<T> kr[8], vr[8], br[8];
    bool ok[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t page = __builtin_amdgcn_readlane(pg, i);
        const int j = jw + 8 * i + kq;
        ok[i] = page >= 0 && j < vis;
        if (ok[i]) {
            const int64_t slot = j & mask;
            kr[i] = load8<T>((const T*)P.k.ptr + page * P.k.sb + h * P.k.sh + slot * P.k.sl + 8 * fg);
            vr[i] = load8<T>((const T*)P.v.ptr + page * P.v.sb + h * P.v.sh + slot * P.v.sl + 8 * fg);
            if (fg < DS / 8) br[i] = load8<T>((const T*)P.b.ptr + page * P.b.sb + h * P.b.sh + slot * P.b.sl + 8 * fg);
        }
    }
    // per-position scalars with lane = position: lam exp(g_m - g_j) and F_m - F_j; NaN for a page that is not there
    const int64_t mine = __shfl(pg, lane >> 3);
    float dec = 0.f, fd = 0.f;
    if (jw + lane < vis) {
        if (mine < 0) {
            fd = __builtin_nanf("");
        } else {
            const int64_t slot = (jw + lane) & mask;
            dec = lam * expf(gq - ((const float*)P.g.ptr)[mine * P.g.sb + h * P.g.sh + slot * P.g.sl]);
            if (has_f) fd = fq - ((const float*)P.f.ptr)[mine * P.f.sb + h * P.f.sh + slot * P.f.sl];
        }
    }
    const f32x8 qv = load_f32x8<T>(Q + 8 * fg);
    f32x8 cv;
    if (fg < DS / 8) cv = load_f32x8<T>(C + 8 * fg);

    float s[8], mx = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float di = __shfl(dec, kq + 8 * i), fi = __shfl(fd, kq + 8 * i);
        float qk = 0.f, cb = 0.f;
        if (ok[i]) {
            const f32x8 kv = __builtin_convertvector(kr[i], f32x8);
#pragma unroll
            for (int e = 0; e < 8; ++e) qk = fmaf(qv[e], kv[e], qk);
            if (fg < DS / 8) {
                const f32x8 bv = __builtin_convertvector(br[i], f32x8);
#pragma unroll
                for (int e = 0; e < 8; ++e) cb = fmaf(cv[e], bv[e], cb);
            }
        }
        float t = fmaf(qk, 0.125f, di * cb);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) t += __shfl_xor(t, o);
        s[i] = jw + 8 * i + kq < vis ? t + fi : -__builtin_inff();
        mx = fmaxf(mx, s[i]);
    }
    if constexpr (TRACK) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (fg == 0 && jw + 8 * i + kq < vis) scores[(int64_t)row * a.max_len + jw + 8 * i + kq] = s[i];
    }
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    const float ref = mx == -__builtin_inff() ? 0.f : mx;      // all -inf: the weights are 0, not NaN
    float p[8], l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        p[i] = expf(s[i] - ref);                               // 0 for positions that are not visible
        l += p[i];
    }
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) l += __shfl_xor(l, o);
    f32x8 acc;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (ok[i] && p[i] != 0.f) {
            const f32x8 vv = __builtin_convertvector(vr[i], f32x8);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = fmaf(p[i], vv[e], acc[e]);
        }
    }
#pragma unroll
    for (int o = 8; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor(acc[e], o);
    if (lane == 0) wm[w] = mx, wl[w] = l;
    if (kq == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) wo[w][8 * fg + e] = acc[e];
    }
    __syncthreads();
    if (w != 0) return;
    float cm = wm[0];
#pragma unroll
    for (int k = 1; k < DW; ++k) cm = fmaxf(cm, wm[k]);
    float cl = 0.f, co = 0.f;
#pragma unroll
    for (int k = 0; k < DW; ++k) {
        const float sc = wm[k] == -__builtin_inff() ? 1.f : expf(wm[k] - cm);      // all -inf: sums of 0, or NaN
        cl = fmaf(wl[k], sc, cl);
        co = fmaf(wo[k][lane], sc, co);
    }
    float* dst = part + ((int64_t)row * nchunk + chunk) * PART;
    dst[2 + lane] = co;
    if (lane == 0) dst[0] = cm, dst[1] = cl;
}

// The join: chunk c's factor exp(max_c - max) is formed by thread c mod 256, sums go in chunk order. A workgroup per
// query row; or, with tracked weights, per (sequence and head, 1,024 positions), whose rows are taken in order and whose
// first workgroup writes the outputs.
template <bool TRACK>
__global__ __launch_bounds__(256) void paged_join_kernel(sisa_paged_decode_args a, int shift, int nchunk, const float* part,
                                                         const float* scores) {
    __shared__ float red[2][4], wo[4][DH];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int pieces = TRACK ? (a.max_len + PIECE - 1) / PIECE : 1;
    const int piece = blockIdx.x % pieces, item = blockIdx.x / pieces;
    const int H = a.pool.heads, nh = TRACK ? item : item / a.M, h = nh % H, n = nh / H;
    const int len = a.lengths[n];
    const bool outs = piece == 0;
    float add[PIECE / 256] = {0.f, 0.f, 0.f, 0.f};
    for (int m = TRACK ? 0 : item % a.M; m < (TRACK ? a.M : item % a.M + 1); ++m) {
        const int64_t row = (int64_t)nh * a.M + m;
        const int vis = visible(len, a.max_len, (int64_t)a.W << shift, a.M, m);
        if (vis <= 0) {
            if (outs && tid < DH) a.out[row * DH + tid] = vis < 0 ? __builtin_nanf("") : 0.f;
            continue;
        }
        const float* P = part + row * nchunk * PART;
        const int nc = (vis + KCH - 1) / KCH;
        float mx = -__builtin_inff();
        for (int c = tid; c < nc; c += 256) mx = fmaxf(mx, P[(int64_t)c * PART]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        __syncthreads();
        if (lane == 0) red[0][w] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
        const float ref = mx == -__builtin_inff() ? 0.f : mx;
        float l = 0.f;
        for (int c = tid; c < nc; c += 256) {
            const float mc = P[(int64_t)c * PART];
            l = fmaf(P[(int64_t)c * PART + 1], mc == -__builtin_inff() ? 1.f : expf(mc - ref), l);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
        if (lane == 0) red[1][w] = l;
        __syncthreads();
        l = red[1][0] + red[1][1] + red[1][2] + red[1][3];
        const float inv = 1.f / l;
        if (outs) {
            float o = 0.f;
            for (int c = w; c < nc; c += 4) {
                const float mc = P[(int64_t)c * PART];
                o = fmaf(P[(int64_t)c * PART + 2 + lane], mc == -__builtin_inff() ? 1.f : expf(mc - ref), o);
            }
            wo[w][lane] = o;
            __syncthreads();
            if (tid < DH) a.out[row * DH + tid] = (wo[0][tid] + wo[1][tid] + wo[2][tid] + wo[3][tid]) * inv;
        }
        if constexpr (TRACK) {
#pragma unroll
            for (int i = 0; i < PIECE / 256; ++i) {
                const int j = piece * PIECE + 256 * i + tid;
                if (j < vis) add[i] += expf(scores[row * a.max_len + j] - ref) * inv;
            }
        }
    }
    if constexpr (TRACK) {
        if (len < 0 || len > a.max_len || len > ((int64_t)a.W << shift)) return;
#pragma unroll
        for (int i = 0; i < PIECE / 256; ++i) {
            const int64_t j = piece * PIECE + 256 * i + tid;
            if (j < len)
                ((float*)a.w_out.ptr)[n * a.w_out.sb + h * a.w_out.sh + j * a.w_out.sl] =
                    ((const float*)a.w_in.ptr)[n * a.w_in.sb + h * a.w_in.sh + j * a.w_in.sl] + add[i];
        }
    }
}

int64_t part_bytes(int64_t rows, int64_t max_len) {
    return (rows * sisa::cdiv(max_len, KCH) * PART * (int64_t)sizeof(float) + 255) / 256 * 256;
}

template <class T, bool TRACK>
int launch_decode(const sisa_paged_decode_args* a, hipStream_t st) {
    const int shift = sisa::log2_of(a->pool.page_size), nchunk = (int)sisa::cdiv(a->max_len, KCH);
    const int64_t rows = (int64_t)a->B * a->pool.heads * a->M;
    float* part = (float*)a->workspace;
    float* scores = (float*)((char*)a->workspace + part_bytes(rows, a->max_len));
    paged_chunk_kernel<T, TRACK><<<(unsigned)(rows * nchunk), 64 * DW, 0, st>>>(*a, shift, nchunk, part, scores);
    const int rc = sisa::launch_status("sisa_paged_decode");
    if (rc) return rc;
    const int64_t groups = TRACK ? rows / a->M * sisa::cdiv(a->max_len, PIECE) : rows;
    paged_join_kernel<TRACK><<<(unsigned)groups, 256, 0, st>>>(*a, shift, nchunk, part, scores);
    return sisa::launch_status("sisa_paged_decode (join)");
}

template <class T>
int launch_decode(const sisa_paged_decode_args* a, hipStream_t st) {
    return a->w_out.ptr ? launch_decode<T, true>(a, st) : launch_decode<T, false>(a, st);
}


}  // namespace

extern "C" int sisa_paged_write(const sisa_paged_write_args* a, void* stream) {
    SISA_REQUIRE(a != nullptr, "sisa_paged_write: null args");
    SISA_REQUIRE_POOL("sisa_paged_write", a->pool);
    SISA_REQUIRE(a->B >= 0 && a->M >= 0 && a->W >= 1, "sisa_paged_write: bad shape B=%d M=%d W=%d", a->B, a->M, a->W);
    if (a->B == 0 || a->M == 0) return SISA_OK;
    SISA_REQUIRE(a->table && a->start, "sisa_paged_write: table and start must be given");
    SISA_REQUIRE(sisa::view_ok(a->k, a->pool.dtype) && sisa::view_ok(a->v, a->pool.dtype) && sisa::view_ok(a->b, a->pool.dtype),
                 "sisa_paged_write: k, v and b rows must be 16-byte aligned");
    SISA_REQUIRE(a->g.ptr && (a->f.ptr == nullptr) == (a->pool.f.ptr == nullptr),
                 "sisa_paged_write: g must be given, and f where the pool has one");
    const int64_t rows = (int64_t)a->B * a->M * a->pool.heads;
    SISA_REQUIRE(rows < ((int64_t)1 << 31), "sisa_paged_write: B*M*H must be below 2^31");
    hipStream_t st = (hipStream_t)stream;
    switch (a->pool.dtype) {
        case SISA_BF16: launch_write<__bf16>(a, rows, st); break;
        case SISA_F16: launch_write<_Float16>(a, rows, st); break;
        default: launch_write<float>(a, rows, st);
    }
    return sisa::launch_status("sisa_paged_write");
}

extern "C" int64_t sisa_paged_decode_workspace_bytes(int32_t B, int32_t H, int32_t M, int32_t max_len, int32_t tracked) {
    if (B < 1 || H < 1 || M < 1 || max_len < 1) return 0;
    const int64_t rows = (int64_t)B * H * M;
    return part_bytes(rows, max_len) + (tracked ? rows * max_len * (int64_t)sizeof(float) : 0);
}

extern "C" int sisa_paged_decode(const sisa_paged_decode_args* a, void* stream) {
    SISA_REQUIRE(a != nullptr, "sisa_paged_decode: null args");
    SISA_REQUIRE_POOL("sisa_paged_decode", a->pool);
    SISA_REQUIRE(a->B >= 0 && a->M >= 1 && a->W >= 1 && a->max_len >= 1 &&
                     a->max_len <= (int64_t)a->W * a->pool.page_size && a->max_len <= (1 << 30),
                 "sisa_paged_decode: bad shape B=%d M=%d W=%d max_len=%d (at most W pages of %d, and 2^30)", a->B, a->M, a->W,
                 a->max_len, a->pool.page_size);
    if (a->B == 0) return SISA_OK;
    SISA_REQUIRE(a->table && a->lengths && a->lam && a->out && a->workspace, "sisa_paged_decode: null pointer");
    SISA_REQUIRE(sisa::view_ok(a->q, a->pool.dtype) && sisa::view_ok(a->c, a->pool.dtype),
                 "sisa_paged_decode: q and c rows must be 16-byte aligned");
    SISA_REQUIRE(a->gq.ptr && (a->fq.ptr == nullptr) == (a->pool.f.ptr == nullptr),
                 "sisa_paged_decode: gq must be given, and fq where the pool has f");
    SISA_REQUIRE((a->w_in.ptr == nullptr) == (a->w_out.ptr == nullptr),
                 "sisa_paged_decode: w_in and w_out must be given together");
    const int64_t rows = (int64_t)a->B * a->pool.heads * a->M;
    SISA_REQUIRE(rows * sisa::cdiv(a->max_len, KCH) < ((int64_t)1 << 31), "sisa_paged_decode: too many rows for one launch");
    hipStream_t st = (hipStream_t)stream;
    switch (a->pool.dtype) {
        case SISA_BF16: return launch_decode<__bf16>(a, st);
        case SISA_F16: return launch_decode<_Float16>(a, st);
        default: return launch_decode<float>(a, st);
    }
}
