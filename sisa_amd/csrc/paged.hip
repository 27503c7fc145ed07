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
template <class T, int ROWS, bool STREAM>
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
    move_rows<T, ROWS, STREAM>(RowViews{a.k, a.v, a.b, a.g, a.f}, rows_of_pool(a.pool), page >= 0, n, page, h, m,
                               pos & (a.pool.page_size - 1), lane);
}

template <class T>
void launch_write(const sisa_paged_write_args* a, int64_t rows, hipStream_t st) {
    const int shift = sisa::log2_of(a->pool.page_size), per = 4 * sisa::rows_per_wave(rows);
    const unsigned grid = (unsigned)sisa::cdiv(rows, per);
    if (per != 256) paged_write_kernel<T, 8, false><<<grid, 256, 0, st>>>(*a, shift);
    else if (2 * rows * sisa::row_bytes(a->pool.dtype) < STREAM_BYTES) paged_write_kernel<T, 64, false><<<grid, 256, 0, st>>>(*a, shift);
    else paged_write_kernel<T, 64, true><<<grid, 256, 0, st>>>(*a, shift);
}

// ------------------------------------------------------------------------------------------------ decode
// A wave takes 64 positions. Eight neighbouring lanes share a position, 8 features of its k and v row and 4 of its b row
// each, so that every load covers whole rows; lane (kq, fg) has positions kq + 8 i, i < 8. A group of eight lies in one page:
// the page's number is in a scalar register. The partial dot products are summed over a position's lanes by halving
// exchanges, which leave position kq + 8 fg with lane (kq, fg): every score, exponential and gate is worked out once.
//
// The chain of dependent loads is what a short cache costs: pages are looked up beside the length, not after it (entries
// behind the last are read within the table and then ignored).
constexpr int TILE = 64;              // positions of a wave
constexpr int DW = 4;                 // waves per workgroup where the positions are split
constexpr int KCH = TILE * DW;        // positions per chunk (workgroup)
constexpr int PIECE = 1024;           // positions of tracked weights per workgroup of the join

// Positions that query row m of a sequence of n sees, or -1 for a length that the call does not take.
SISA_DEV int visible(int n, int max_len, int64_t held, int M, int m) {
    if (n < 0 || n > max_len || n > held) return -1;
    const int last = n - M + m + 1;
    return last > 0 ? last : 0;
}

template <int CTRL> SISA_DEV float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}
constexpr int XOR1 = 0xB1, XOR2 = 0x4E, XOR7 = 0x141, XOR8 = 0x128;    // of a lane's number (8: a rotation of 16 lanes by 8)

// x[i] summed over the eight lanes that share lane / 8; lane 8 k + i gets the sum of x[i].
SISA_DEV float sum_scatter(const float (&x)[8], int fg) {
    float y[4], z[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (fg & 4 ? x[i + 4] : x[i]) + dpp<XOR7>(fg & 4 ? x[i] : x[i + 4]);
#pragma unroll
    for (int i = 0; i < 2; ++i) z[i] = (fg & 2 ? y[i + 2] : y[i]) + dpp<XOR2>(fg & 2 ? y[i] : y[i + 2]);
    return (fg & 1 ? z[1] : z[0]) + dpp<XOR1>(fg & 1 ? z[0] : z[1]);
}

// STREAM: 16-bit rows of a cache of 256 MB or more, loaded with the non-temporal hint as csrc/decode.hip does (516 MB 102 ->
// 90 us; 77 MB 21.0 -> 22.9).
//
// A workgroup of NW waves per (query row, chunk of 64 NW positions). Outputs are TO: float, or the pool's dtype for a layer
// step, whose next product reads them. ONE: one chunk, which writes the row's output, and its
// weights. Otherwise the chunk's largest score and sum go to stat, its unnormalised output to part, and with TRACK the
// scores to `scores`.
template <class T, class TO, int NW, bool ONE, bool TRACK, bool STREAM>
__global__ __launch_bounds__(64 * NW) void paged_chunk_kernel(sisa_paged_decode_args a, TO* out, int shift, int nchunk,
                                                              f32x2* stat, float* part, float* scores) {
    __shared__ float wm[NW], wl[NW], wo[NW][DH];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int fg = lane & 7, kq = lane >> 3;
    // chunk by chunk over the rows: the chunks behind the shorter sequences' ends come last and hold nothing up
    const int rows = a.B * a.pool.heads * a.M, chunk = ONE ? 0 : blockIdx.x / rows, row = ONE ? blockIdx.x : blockIdx.x % rows;
    const int H = a.pool.heads, m = row % a.M, nh = row / a.M, h = nh % H, n = nh / H;
    const sisa_page_pool& P = a.pool;
    const int jw = (chunk * NW + w) * TILE;
    // lane i < 8: the page of positions jw + 8 i .. + 7
    const int group = (jw + 8 * fg) >> shift;
    int pg = group < a.W ? a.table[n * a.s_table + group] : -1;
    const int len = a.lengths[n];
    const int vis = visible(len, a.max_len, (int64_t)a.W << shift, a.M, m);
    if (!ONE && chunk * KCH >= vis) return;            // nothing here: the join does not read this chunk's partial
    pg = pg >= 0 && pg < P.pages ? pg : -1;
    const int mask = P.page_size - 1;

    frag8<T> kr[8], vr[8];
    vec4<T> br[8];
    bool ok[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t page = __builtin_amdgcn_readlane(pg, i);
        const int j = jw + 8 * i + kq;
        ok[i] = page >= 0 && j < vis;
        if (ok[i]) {
            const int64_t slot = j & mask;
            kr[i] = load_hint<frag8<T>, STREAM>((const T*)P.k.ptr + (page * P.k.sb + h * P.k.sh) + slot * P.k.sl + 8 * fg);
            vr[i] = load_hint<frag8<T>, STREAM>((const T*)P.v.ptr + (page * P.v.sb + h * P.v.sh) + slot * P.v.sl + 8 * fg);
            br[i] = load_hint<vec4<T>, STREAM>((const T*)P.b.ptr + (page * P.b.sb + h * P.b.sh) + slot * P.b.sl + 4 * fg);
        }
    }
    const f32x8 qv = load_f32x8<T>((const T*)a.q.ptr + n * a.q.sb + h * a.q.sh + m * a.q.sl + 8 * fg);
    const f32x4 cv = __builtin_convertvector(load4<T>((const T*)a.c.ptr + n * a.c.sb + h * a.c.sh + m * a.c.sl + 4 * fg), f32x4);
    const bool has_f = P.f.ptr != nullptr;
    const float gq = ((const float*)a.gq.ptr)[n * a.gq.sb + h * a.gq.sh + m * a.gq.sl];
    const float fq = has_f ? ((const float*)a.fq.ptr)[n * a.fq.sb + h * a.fq.sh + m * a.fq.sl] : 0.f;
    const float lam = a.lam[h * a.s_lam];
    // the lane's own position kq + 8 fg: lam exp(g_m - g_j) and F_m - F_j, NaN for a page that is not there
    const int j = jw + 8 * fg + kq;                    // group fg's page is lane fg's, and every lane 8 k + fg's
    float dec = 0.f, fd = __builtin_nanf("");
    if (j < vis && pg >= 0) {
        const int64_t slot = j & mask;
        dec = lam * expf(gq - ((const float*)P.g.ptr)[pg * P.g.sb + h * P.g.sh + slot * P.g.sl]);
        fd = has_f ? fq - ((const float*)P.f.ptr)[pg * P.f.sb + h * P.f.sh + slot * P.f.sl] : 0.f;
    }
    float old = 0.f;
    if constexpr (ONE && TRACK)
        if (j < vis) old = ((const float*)a.w_in.ptr)[n * a.w_in.sb + h * a.w_in.sh + j * a.w_in.sl];

    float qk[8], cb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        qk[i] = cb[i] = 0.f;
        if (ok[i]) {
            const f32x8 kv = __builtin_convertvector(kr[i], f32x8);
            const f32x4 bv = __builtin_convertvector(br[i], f32x4);
#pragma unroll
            for (int e = 0; e < 8; ++e) qk[i] = fmaf(qv[e], kv[e], qk[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) cb[i] = fmaf(cv[e], bv[e], cb[i]);
        }
    }
    const float tq = sum_scatter(qk, fg), tc = sum_scatter(cb, fg);      // every lane takes part in the exchanges
    const float s = j < vis ? fmaf(tq, 0.125f, dec * tc) + fd : -__builtin_inff();
    if constexpr (TRACK && !ONE)
        if (j < vis) scores[(int64_t)row * a.max_len + j] = s;
    float mx = fmaxf(s, dpp<XOR1>(s));
    mx = fmaxf(mx, dpp<XOR2>(mx));
    mx = fmaxf(mx, dpp<XOR7>(mx));
    mx = group_max(fmaxf(mx, dpp<XOR8>(mx)));
    const float ref = mx == -__builtin_inff() ? 0.f : mx;      // all -inf: the weights are 0, not NaN
    const float p = expf(s - ref);                             // 0 for positions that are not visible
    float l = p + dpp<XOR1>(p);
    l += dpp<XOR2>(l);
    l += dpp<XOR7>(l);
    l = group_sum(l + dpp<XOR8>(l));
    f32x8 acc;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float pi = __shfl(p, (lane & 56) | i);
        if (ok[i] && pi != 0.f) {
            const f32x8 vv = __builtin_convertvector(vr[i], f32x8);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = fmaf(pi, vv[e], acc[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = group_sum(acc[e] + dpp<XOR8>(acc[e]));
    if (lane == 0) wm[w] = mx, wl[w] = l;
    if (kq == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) wo[w][8 * fg + e] = acc[e];
    }
    __syncthreads();
    if (!(ONE && TRACK) && w != 0) return;
    float cm = wm[0];
#pragma unroll
    for (int k = 1; k < NW; ++k) cm = fmaxf(cm, wm[k]);
    float cl = 0.f, co = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
        const float sc = wm[k] == -__builtin_inff() ? 1.f : expf(wm[k] - cm);      // all -inf: sums of 0, or NaN
        cl = fmaf(wl[k], sc, cl);
        co = fmaf(wo[k][lane], sc, co);
    }
    if constexpr (ONE) {
        if (w == 0) out[(int64_t)row * DH + lane] = cvt<TO>(vis < 0 ? __builtin_nanf("") : vis == 0 ? 0.f : co / cl);
        if constexpr (TRACK)
            if (j < vis)
                ((float*)a.w_out.ptr)[n * a.w_out.sb + h * a.w_out.sh + j * a.w_out.sl] =
                    old + expf(s - (cm == -__builtin_inff() ? 0.f : cm)) / cl;
    } else {
        const int64_t at = (int64_t)row * nchunk + chunk;
        part[at * DH + lane] = co;
        if (lane == 0) stat[at] = f32x2{cm, cl};
    }
}

// The join of a row's chunks, in a fixed order. A workgroup per query row; or, with tracked weights, per (sequence and head,
// 1,024 positions), whose rows are taken in order and whose first workgroup writes the outputs. What the weights need is
// loaded before the row's sum is known.
template <class TO, bool TRACK>
__global__ __launch_bounds__(256) void paged_join_kernel(sisa_paged_decode_args a, TO* out, int shift, int nchunk,
                                                         const f32x2* stat, const float* part, const float* scores) {
    __shared__ float red[2][4], wo[4][DH], ms[256];    // ms: up to 256 chunks' factors
    constexpr int PER = PIECE / 256, AHEAD = 8;        // partial outputs of a wave under way
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pieces = TRACK ? (a.max_len + PIECE - 1) / PIECE : 1;
    const int piece = blockIdx.x % pieces, item = blockIdx.x / pieces;
    const int H = a.pool.heads, nh = TRACK ? item : item / a.M, h = nh % H, n = nh / H;
    const int len = a.lengths[n];
    if (TRACK && piece > 0 && piece * PIECE >= len) return;
    const bool outs = piece == 0;
    float sum[PER];
    if constexpr (TRACK) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int64_t j = piece * PIECE + 256 * i + tid;
            sum[i] = j < len && j < a.max_len ? ((const float*)a.w_in.ptr)[n * a.w_in.sb + h * a.w_in.sh + j * a.w_in.sl] : 0.f;
        }
    }
    for (int m = TRACK ? 0 : item % a.M; m < (TRACK ? a.M : item % a.M + 1); ++m) {
        const int64_t row = (int64_t)nh * a.M + m;
        const int vis = visible(len, a.max_len, (int64_t)a.W << shift, a.M, m);
        if (vis <= 0) {
            if (outs && tid < DH) out[row * DH + tid] = cvt<TO>(vis < 0 ? __builtin_nanf("") : 0.f);
            continue;
        }
        float s[PER];
        if constexpr (TRACK) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int j = piece * PIECE + 256 * i + tid;
                s[i] = j < vis ? scores[row * a.max_len + j] : -__builtin_inff();
            }
        }
        const f32x2* S = stat + row * nchunk;
        const int nc = (vis + KCH - 1) / KCH;
        float mx = -__builtin_inff(), l = 0.f, m0 = 0.f;
        for (int c = tid; c < nc; c += 256) {
            const f32x2 x = S[c];
            if (c == tid) m0 = x[0];
            const float to = fmaxf(mx, x[0]), ref = to == -__builtin_inff() ? 0.f : to;
            l = l * (mx == -__builtin_inff() ? 1.f : expf(mx - ref)) + x[1] * (x[0] == -__builtin_inff() ? 1.f : expf(x[0] - ref));
            mx = to;
        }
        float wmx = mx;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) wmx = fmaxf(wmx, __shfl_xor(wmx, o));
        l *= mx == -__builtin_inff() ? 1.f : expf(mx - wmx);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
        __syncthreads();                               // the last row's sums have been read
        if (lane == 0) red[0][w] = wmx, red[1][w] = l;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
        const float ref = mx == -__builtin_inff() ? 0.f : mx;
        l = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) l = fmaf(red[1][k], red[0][k] == -__builtin_inff() ? 1.f : expf(red[0][k] - ref), l);
        const float inv = 1.f / l;
        if (outs) {
            float o = 0.f;
            auto factor = [&](float mc) { return mc == -__builtin_inff() ? 1.f : expf(mc - ref); };
            ms[tid] = factor(m0);
            __syncthreads();
            // every fourth chunk; behind the last the last again, which is left out
            const float* O = part + row * nchunk * DH + lane;
            auto add = [&](auto&& scale) {
                for (int c0 = w; c0 < nc; c0 += 4 * AHEAD) {
                    float x[AHEAD], by[AHEAD];
#pragma unroll
                    for (int k = 0; k < AHEAD; ++k) {
                        const int c = c0 + 4 * k < nc ? c0 + 4 * k : nc - 1;
                        x[k] = O[c * DH];
                        by[k] = scale(c);
                    }
#pragma unroll
                    for (int k = 0; k < AHEAD; ++k) o = c0 + 4 * k < nc ? fmaf(x[k], by[k], o) : o;
                }
            };
            if (nc <= 256) add([&](int c) { return ms[c]; });
            else add([&](int c) { return factor(S[c][0]); });
            wo[w][lane] = o;
            __syncthreads();
            if (tid < DH) out[row * DH + tid] = cvt<TO>(((wo[0][tid] + wo[1][tid]) + (wo[2][tid] + wo[3][tid])) * inv);
        }
        if constexpr (TRACK) {
#pragma unroll
            for (int i = 0; i < PER; ++i) sum[i] += expf(s[i] - ref) * inv;
        }
    }
    if constexpr (TRACK) {
        if (visible(len, a.max_len, (int64_t)a.W << shift, 1, 0) <= 0) return;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int64_t j = piece * PIECE + 256 * i + tid;
            if (j < len) ((float*)a.w_out.ptr)[n * a.w_out.sb + h * a.w_out.sh + j * a.w_out.sl] = sum[i];
        }
    }
}

// The waves of a workgroup that takes a query row whole, so that no join is needed; 0: the row is split. With tracked weights
// it must be the only row to add to them. 16 waves fill a CU alone: more rows than CUs are split (whole / split, us: 192 rows of
// 1,000 positions, tracked, 16.7 / 20.4, 576 of 1,000 49.8 / 43.9; with 8 waves 544 rows of 452 20.7 / 23.5, with 4 768 of 100
// 9.4 / 13.6; with 16 waves the last two 27.1 and 17.9).
int whole_waves(int64_t rows, int M, int64_t max_len, int elem, bool tracked) {
    if (tracked && M > 1) return 0;
    return max_len <= KCH ? DW : max_len <= 2 * KCH ? 8 : max_len <= 4 * KCH && elem == 2 && rows <= 256 ? 16 : 0;
}

bool fits(int64_t rows, int M, int64_t max_len, int elem, bool tracked) {
    const int waves = whole_waves(rows, M, max_len, elem, tracked);
    return rows <= sisa::MAX_THREADS / (waves ? 64 * waves : sisa::cdiv(max_len, KCH) * KCH);
}

struct DecodeSpace {
    f32x2* stat;
    float *part, *scores;
    int64_t bytes;
};

int64_t pad256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

DecodeSpace decode_space(char* base, int64_t rows, int64_t max_len, bool tracked) {
    const int64_t chunks = rows * sisa::cdiv(max_len, KCH);
    DecodeSpace s{};
    s.stat = (f32x2*)base;
    s.part = (float*)(base + pad256(chunks * 8));
    s.scores = (float*)((char*)s.part + pad256(chunks * DH * 4));
    s.bytes = (char*)s.scores - base + (tracked ? rows * max_len * 4 : 0);
    return s;
}

template <class T, class TO, int NW, bool TRACK>
int launch_whole(const sisa_paged_decode_args* a, TO* out, int64_t rows, hipStream_t st) {
    paged_chunk_kernel<T, TO, NW, true, TRACK, false><<<(unsigned)rows, 64 * NW, 0, st>>>(*a, out, sisa::log2_of(a->pool.page_size),
                                                                                         1, nullptr, nullptr, nullptr);
    return sisa::launch_status("sisa_paged_decode");
}

template <class T, class TO, bool TRACK>
int launch_decode(const sisa_paged_decode_args* a, TO* out, hipStream_t st) {
    const int shift = sisa::log2_of(a->pool.page_size), nchunk = (int)sisa::cdiv(a->max_len, KCH);
    const int64_t rows = (int64_t)a->B * a->pool.heads * a->M;
    const DecodeSpace ws = decode_space((char*)a->workspace, rows, a->max_len, TRACK);
    switch (whole_waves(rows, a->M, a->max_len, (int)sizeof(T), TRACK)) {
        case 4: return launch_whole<T, TO, 4, TRACK>(a, out, rows, st);
        case 8: return launch_whole<T, TO, 8, TRACK>(a, out, rows, st);
        case 16:
            if constexpr (sizeof(T) == 2) return launch_whole<T, TO, 16, TRACK>(a, out, rows, st);
    }
    const unsigned grid = (unsigned)(rows * nchunk);
    if (sizeof(T) == 2 && a->M == 1 && sisa::cache_bytes(a->pool, a->B, a->max_len) >= STREAM_BYTES)
        paged_chunk_kernel<T, TO, DW, false, TRACK, sizeof(T) == 2><<<grid, KCH, 0, st>>>(*a, out, shift, nchunk, ws.stat, ws.part,
                                                                                         ws.scores);
    else paged_chunk_kernel<T, TO, DW, false, TRACK, false><<<grid, KCH, 0, st>>>(*a, out, shift, nchunk, ws.stat, ws.part, ws.scores);
    const int rc = sisa::launch_status("sisa_paged_decode");
    if (rc) return rc;
    const int64_t groups = TRACK ? rows / a->M * sisa::cdiv(a->max_len, PIECE) : rows;
    paged_join_kernel<TO, TRACK><<<(unsigned)groups, 256, 0, st>>>(*a, out, shift, nchunk, ws.stat, ws.part, ws.scores);
    return sisa::launch_status("sisa_paged_decode (join)");
}

template <class T, class TO>
int launch_decode(const sisa_paged_decode_args* a, TO* out, hipStream_t st) {
    return a->w_out.ptr ? launch_decode<T, TO, true>(a, out, st) : launch_decode<T, TO, false>(a, out, st);
}

}  // namespace

namespace sisa {
namespace detail {
// The attention of 16-bit operands with the result rounded to their dtype, (B,H,M,64) contiguous (checked by the caller:
// sisa_step_paged), and whether its launches take one new position of each of `rows` sequences and heads.
__attribute__((visibility("hidden"))) bool paged_attn_fits(int64_t rows, int64_t max_len, bool tracked) {
    return fits(rows, 1, max_len, 2, tracked);
}
__attribute__((visibility("hidden"))) int paged_attn_out16(const sisa_paged_decode_args* a, void* out, hipStream_t st) {
    return a->pool.dtype == SISA_BF16 ? launch_decode<__bf16>(a, (__bf16*)out, st) : launch_decode<_Float16>(a, (_Float16*)out, st);
}
}  // namespace detail
}  // namespace sisa

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

extern "C" int64_t sisa_paged_decode_workspace_bytes(int32_t B, int32_t H, int32_t M, int32_t max_len, int32_t dtype,
                                                     int32_t tracked) {
    if (B < 1 || H < 1 || M < 1 || max_len < 1 || whole_waves((int64_t)B * H * M, M, max_len, sisa::elem_size(dtype), tracked != 0))
        return 0;
    return decode_space(nullptr, (int64_t)B * H * M, max_len, tracked != 0).bytes;
}

extern "C" int sisa_paged_decode(const sisa_paged_decode_args* a, void* stream) {
    SISA_REQUIRE(a != nullptr, "sisa_paged_decode: null args");
    SISA_REQUIRE_POOL("sisa_paged_decode", a->pool);
    SISA_REQUIRE(a->B >= 0 && a->M >= 1 && a->W >= 1 && a->max_len >= 1 &&
                     a->max_len <= (int64_t)a->W * a->pool.page_size && a->max_len <= (1 << 30),
                 "sisa_paged_decode: bad shape B=%d M=%d W=%d max_len=%d (at most W pages of %d, and 2^30)", a->B, a->M, a->W,
                 a->max_len, a->pool.page_size);
    if (a->B == 0) return SISA_OK;
    SISA_REQUIRE(a->table && a->lengths && a->lam && a->out, "sisa_paged_decode: null pointer");
    const int64_t rows = (int64_t)a->B * a->pool.heads * a->M;
    SISA_REQUIRE(whole_waves(rows, a->M, a->max_len, sisa::elem_size(a->pool.dtype), a->w_out.ptr != nullptr) ||
                     (a->workspace && sisa::aligned16(a->workspace)),
                 "sisa_paged_decode: null workspace, or not 16-byte aligned");
    SISA_REQUIRE(sisa::view_ok(a->q, a->pool.dtype) && sisa::view_ok(a->c, a->pool.dtype),
                 "sisa_paged_decode: q and c rows must be 16-byte aligned");
    SISA_REQUIRE(a->gq.ptr && (a->fq.ptr == nullptr) == (a->pool.f.ptr == nullptr),
                 "sisa_paged_decode: gq must be given, and fq where the pool has f");
    SISA_REQUIRE((a->w_in.ptr == nullptr) == (a->w_out.ptr == nullptr),
                 "sisa_paged_decode: w_in and w_out must be given together");
    SISA_REQUIRE(fits(rows, a->M, a->max_len, sisa::elem_size(a->pool.dtype), a->w_out.ptr != nullptr),
                 "sisa_paged_decode: B*H*M*max_len too large for one launch");
    hipStream_t st = (hipStream_t)stream;
    switch (a->pool.dtype) {
        case SISA_BF16: return launch_decode<__bf16>(a, a->out, st);
        case SISA_F16: return launch_decode<_Float16>(a, a->out, st);
        default: return launch_decode<float>(a, a->out, st);
    }
}
