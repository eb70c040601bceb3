// sparse.cu -- page-sparse attention: key bounds per page, page selection, attention over lists.
//
//  * msgl_kv_page_bounds        smallest / largest key of each page a step touched
//  * msgl_select_pages          per query token and kv head, the pages with the largest bound of
//                               their attention logits (plus forced first and last pages)
//  * msgl_paged_attention_pages softmax attention over the listed pages only
//
// For page j with key bounds lo, hi (elementwise), every key k of the page and query head g:
//   q_g . k <= s_g(j) = sum_d max(q_gd, 0) hi_d + min(q_gd, 0) lo_d.
// A kv head's query group shares one list, so its score is max_g s_g(j): the largest logit any
// head of the group can have in the page. Bounds are bf16 like the keys, hence exact, and 1/16 of
// the page's key and value bytes.
//
// The selection does not hang on the order the sums are taken in: scores are computed with bf16
// MMAs in fp32, and where the error bound leaves open which page is the k-th, the pages in question
// are scored again to 2^-46 or better.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "tmap.h"

namespace msgl {
namespace {

constexpr int kPage = 16;
constexpr int kHd = 128;
constexpr int kMaxPagesPerReq = 32768;  // context bound of the selection: 524288 tokens
constexpr int kMaxTopPages = 1024;
constexpr float kNegInf = -__builtin_huge_valf();

// ------------------------------------------------------------------ request window
// Context length and query rows of request r: row i sits at position L - qn + i.
struct Window {
    int L, qn, q0;
};

__device__ __forceinline__ Window request_window(int r, const int* seq_lens, const int* q_indptr,
                                                 int max_len, bool report, int* err) {
    Window w;
    w.L = seq_lens[r];
    if (w.L < 0 || w.L > max_len) {
        if (report) record_error(err, MSGL_ERR_BOUNDS, 800);
        w.L = w.L < 0 ? 0 : max_len;
    }
    w.q0 = q_indptr ? q_indptr[r] : r;
    w.qn = q_indptr ? q_indptr[r + 1] - w.q0 : 1;
    return w;
}

// ------------------------------------------------------------------ bounds
constexpr int kBoundWarps = 8;

__device__ __forceinline__ uint32_t min_nan2(uint32_t a, uint32_t b) {
    __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max_nan2(uint32_t a, uint32_t b) {
    __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
}

// One warp per (request, touched page, kv head): half-warps take alternate token rows, 16 bytes a
// lane, all eight row loads in flight. Rows at or behind the context's end are not read.
__global__ void __launch_bounds__(kBoundWarps * 32)
page_bounds_kernel(const __nv_bfloat16* __restrict__ k_pool, int pool_pages,
                   const int* __restrict__ page_table, int max_pages,
                   const int* __restrict__ seq_lens, const int* __restrict__ q_indptr, int max_q_len,
                   int hkv, int pages_per_req, int64_t total, __nv_bfloat16* __restrict__ bounds,
                   int* err) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t wid = static_cast<int64_t>(blockIdx.x) * kBoundWarps + (threadIdx.x >> 5);
    if (wid >= total) return;
    const int h = static_cast<int>(wid % hkv);
    const int64_t rp = wid / hkv;
    const int p = static_cast<int>(rp % pages_per_req), r = static_cast<int>(rp / pages_per_req);
    const bool report = p == 0 && h == 0 && lane == 0;
    Window w = request_window(r, seq_lens, q_indptr, max_pages * kPage, report, err);
    if (w.qn > max_q_len) {
        if (report) record_error(err, MSGL_ERR_BOUNDS, 801);
        w.qn = max_q_len;
    }
    if (w.qn <= 0 || w.L == 0) return;
    const int page = max(w.L - w.qn, 0) / kPage + p;
    if (page * kPage >= w.L) return;
    const int phys = page_table[static_cast<int64_t>(r) * max_pages + page];
    if (static_cast<unsigned>(phys) >= static_cast<unsigned>(pool_pages)) {
        if (h == 0 && lane == 0) record_error(err, MSGL_ERR_BOUNDS, 802);
        return;
    }
    const int rows = min(kPage, w.L - page * kPage);
    const int half = lane >> 4, col = (lane & 15) * 8;
    const int64_t stride = static_cast<int64_t>(hkv) * kHd;
    const __nv_bfloat16* src = k_pool + (static_cast<int64_t>(phys) * kPage) * stride + h * kHd + col;
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // a missing row repeats row 0
        const int row = 2 * i + half;
        v[i] = *reinterpret_cast<const uint4*>(src + (row < rows ? row : 0) * stride);
    }
    uint32_t lo[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
    uint32_t hi[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            lo[e] = min_nan2(lo[e], u[e]);
            hi[e] = max_nan2(hi[e], u[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        lo[e] = min_nan2(lo[e], __shfl_xor_sync(0xffffffffu, lo[e], 16));
        hi[e] = max_nan2(hi[e], __shfl_xor_sync(0xffffffffu, hi[e], 16));
    }
    __nv_bfloat16* dst = bounds + ((static_cast<int64_t>(phys) * hkv + h) * 2 + half) * kHd + col;
    *reinterpret_cast<uint4*>(dst) = half ? make_uint4(hi[0], hi[1], hi[2], hi[3])
                                          : make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// ------------------------------------------------------------------ scores
// Scores of `groups` x 64 pages (16 a warp and group) for a tile of one request's query rows. The bounds of 16 pages
// are the A operand (16 x 256: lo then hi) and stay in registers; the B operand is (min(q, 0),
// max(q, 0)) of 8 columns = 8 / G tokens x G query heads. Both are loaded straight from global
// memory as 16-byte pieces: lane (g, c) takes elements 32 i + 8 c .. + 7 of row g, which fixes one
// order of the 256 products for A and B alike.
constexpr int kScoreWarps = 4;
constexpr int kScorePages = kScoreWarps * 16;

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t abs2(uint32_t a) { return a & 0x7fff7fffu; }

struct SelectArgs {
    const __nv_bfloat16 *q, *bounds;
    int pool_pages;
    const int* page_table;
    int max_pages;
    const int *seq_lens, *q_indptr;
    int num_reqs, total_q, max_q_len, max_len;
    int hq, hkv, top, sink, recent;
    int t0, t1;        // query rows of this launch
    int stride;        // pages per score row
    float* scores;             // [rows][Hkv][stride]
    float* mags;               // [rows][Hkv][stride / 16]: in the request's first row of the launch
    unsigned long long* wide;  // [rows][Hkv][stride]: keys beyond fp32 where many scores are close
    int* page_ids;
    int* err;
};

// Single tokens take `groups` groups of pages one after the other, the next group's page ids loaded
// ahead, and go through a page's heads first: their bounds are neighbours in memory (64 requests at
// 4k to 32k: 72 -> 64 us). Chunks take one group for a tile of kScoreCols columns (query rows x G),
// whose queries lie in shared memory: the loop over them waited for L1 before (1.3k rows 113 -> 90 us).
// A lane takes half a line at a time: the hint brings the rest of the bounds into L2 with it (64 requests
// 173 -> 170 us).
__device__ __forceinline__ uint4 load_bounds(const __nv_bfloat16* p) {
    uint4 v;
    asm volatile("ld.global.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
constexpr int kScoreCols = 128;
constexpr int kScorePitch = kHd * 2 + 64;  // bytes a query: two rows of a quarter-warp in other banks

template <int G, bool CHUNK>
__global__ void __launch_bounds__(kScoreWarps * 32, 4)
page_scores_kernel(const SelectArgs a, int tiles, int page_tiles, int groups) {
    constexpr int kRows = CHUNK ? kScoreCols / G : 1;  // query rows of a tile
    constexpr int TPN = 8 / G;                         // query rows of an 8-column MMA tile
    __shared__ __align__(16) uint8_t sq[CHUNK ? kScoreCols * kScorePitch : 16];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    int64_t id = blockIdx.x;
    const int inner = CHUNK ? page_tiles : a.hkv, outer = CHUNK ? a.hkv : page_tiles;
    const int x = static_cast<int>(id % inner);
    id /= inner;
    const int y = static_cast<int>(id % outer);
    id /= outer;
    const int h = CHUNK ? y : x, pt = CHUNK ? x : y;
    const int tile = static_cast<int>(id % tiles), r = static_cast<int>(id / tiles);
    const bool report = pt == 0 && h == 0 && tile == 0 && threadIdx.x == 0;
    const Window w = request_window(r, a.seq_lens, a.q_indptr, a.max_len, report, a.err);
    if (report && (w.qn > a.max_q_len || w.qn < 0 || w.q0 < 0 || w.q0 + static_cast<int64_t>(w.qn) > a.total_q))
        record_error(a.err, MSGL_ERR_BOUNDS, 801);
    const int first = max(w.q0, a.t0);  // the request's first row of this launch: holds its mags
    const int i0 = max(tile * kRows, first - w.q0);
    const int i1 = min(min(w.qn, a.max_q_len), min((tile + 1) * kRows, a.t1 - w.q0));
    if (w.q0 < 0 || i0 >= i1) return;
    const int seen = (w.L - w.qn + i1 - 1) >> 4;  // pages before the last row's own page
    const int last = seen + 1 - a.recent;         // pages [sink, last) are scored
    // Pages up to those that the request's last row of this launch scores take part in the magnitudes:
    // every tile then finds the same for a group of pages that its own end cuts, and whichever of them
    // stores it last, no row works with a smaller one than its pages have.
    const int rows_end = min(min(w.qn, a.max_q_len), a.t1 - w.q0);
    const int cover = ((w.L - w.qn + rows_end - 1) >> 4) + 1 - a.recent;
    if (seen + 1 <= a.top) return;                // every row of the tile sees all its pages
    const int end = min(last, (pt + 1) * groups * kScorePages);
    int pg0 = pt * groups * kScorePages;
    if (pg0 >= end || (pt + 1) * groups * kScorePages <= a.sink) return;  // the whole CTA
    const __nv_bfloat16* q0 = a.q + (static_cast<int64_t>(w.q0 + i0) * a.hq + h * G) * kHd;
    if (CHUNK) {
        for (int p = threadIdx.x; p < (i1 - i0) * G * 16; p += kScoreWarps * 32) {
            const int col = p >> 4, piece = p & 15;
            cp_async16(smem_u32(sq + col * kScorePitch + piece * 16),
                       q0 + (static_cast<int64_t>(col / G) * a.hq + col % G) * kHd + piece * 8, true);
        }
        cp_async_commit();
    }
    pg0 += warp * 16;
    if (!CHUNK) {
        pg0 += max(0, (a.sink - pg0) / kScorePages) * kScorePages;  // groups of forced pages only
        if (pg0 >= end) return;
    }

    const int* table = a.page_table + static_cast<int64_t>(r) * a.max_pages;
    int next[2];  // physical pages of the next group
#pragma unroll
    for (int u = 0; u < 2; ++u) next[u] = pg0 + g + 8 * u < cover ? table[pg0 + g + 8 * u] : -1;
    do {
        uint32_t af[8][2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            int phys = next[u];
            if (pg0 + g + 8 * u < cover && static_cast<unsigned>(phys) >= static_cast<unsigned>(a.pool_pages)) {
                record_error(a.err, MSGL_ERR_BOUNDS, 802);
                phys = -1;
            }
            const __nv_bfloat16* src = a.bounds + (static_cast<int64_t>(max(phys, 0)) * a.hkv + h) * 2 * kHd + 8 * c;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (phys >= 0) v = load_bounds(src + 32 * i);
                af[i][u][0] = v.x; af[i][u][1] = v.y; af[i][u][2] = v.z; af[i][u][3] = v.w;
            }
        }
        if (!CHUNK) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int page = pg0 + kScorePages + g + 8 * u;
                next[u] = page < end ? table[page] : -1;  // (one row: cover is last)
            }
        }
        {   // largest 2-norm of max(|lo|, |hi|) among the 16 pages: what the scores' error scales with
            float m[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                m[u] = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t v = max_nan2(abs2(af[i][u][e]), abs2(af[4 + i][u][e]));
                        m[u] += bf16lo(v) * bf16lo(v) + bf16hi(v) * bf16hi(v);
                    }
                m[u] += __shfl_xor_sync(0xffffffffu, m[u], 1);
                m[u] += __shfl_xor_sync(0xffffffffu, m[u], 2);
            }
            const float most = sqrtf(warp_max(fmaxf(m[0], m[1])));
            if (lane == 0 && pg0 < end)
                a.mags[(static_cast<int64_t>(first - a.t0) * a.hkv + h) * (a.stride / 16) + pg0 / 16] = most;
        }
        if (CHUNK) {
            cp_async_wait<0>();
            __syncthreads();
            if (pg0 >= end) return;
        }

        // lane (g, c) stores page g (+ 8) of row i + 2 c / G (of columns 2 c and 2 c + 1 where G = 1)
        const int tt = 2 * c / G;
        const bool mine[2] = {(2 * c) % G == 0 && pg0 + g < last, (2 * c) % G == 0 && pg0 + g + 8 < last};
        const int64_t pitch = static_cast<int64_t>(a.hkv) * a.stride;
        float* out = a.scores + (w.q0 + i0 + tt - a.t0) * pitch + static_cast<int64_t>(h) * a.stride + pg0 + g;
        for (int i = 0; i < i1 - i0; i += TPN, out += TPN * pitch) {
            uint32_t qf[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint4 v = make_uint4(0, 0, 0, 0);
                const int col = i * G + g;
                if (col < (i1 - i0) * G)
                    v = CHUNK ? *reinterpret_cast<const uint4*>(sq + col * kScorePitch + 16 * c + 64 * k)
                              : *reinterpret_cast<const uint4*>(q0 + col * kHd + 8 * c + 32 * k);
                qf[k][0] = v.x; qf[k][1] = v.y; qf[k][2] = v.z; qf[k][3] = v.w;
            }
            float d0[4] = {0.f, 0.f, 0.f, 0.f}, d1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint32_t n0 = min_nan2(qf[k][2 * s], 0u), n1 = min_nan2(qf[k][2 * s + 1], 0u);
                    const uint32_t p0 = max_nan2(qf[k][2 * s], 0u), p1 = max_nan2(qf[k][2 * s + 1], 0u);
                    mma_bf16_16816(d0, af[k][0][2 * s], af[k][1][2 * s], af[k][0][2 * s + 1],
                                   af[k][1][2 * s + 1], n0, n1);
                    mma_bf16_16816(d1, af[4 + k][0][2 * s], af[4 + k][1][2 * s], af[4 + k][0][2 * s + 1],
                                   af[4 + k][1][2 * s + 1], p0, p1);
                }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float v0 = d0[2 * u] + d1[2 * u], v1 = d0[2 * u + 1] + d1[2 * u + 1];
                if (G == 1) {
                    if (mine[u] && i + tt < i1 - i0) out[8 * u] = v0;
                    if (mine[u] && i + tt + 1 < i1 - i0) out[pitch + 8 * u] = v1;
                } else {
                    float m = max_nan(v0, v1);
                    if (G >= 4) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    if (G >= 8) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
                    if (mine[u] && i + tt < i1 - i0) out[8 * u] = m;
                }
            }
        }
        pg0 += kScorePages;
    } while (!CHUNK && pg0 < end);
}

// ------------------------------------------------------------------ selection
// Order-preserving integer keys; NaN ranks highest, the two zeros are one value. No key is 0.
__device__ __forceinline__ uint32_t key_of(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t b = __float_as_uint(v + 0.f);
    return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kInfKey = 0xff800000u;  // key_of(+inf): above it only NaN
__device__ __forceinline__ unsigned long long key_of(double v) {
    if (v != v) return ~0ull;
    const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

// Score key of one page and query head beyond fp32, by each group of eight lanes (every lane of the
// group gets it; all lanes of the warp call it). bounds_row: lo then hi of the page.
// A term is q (q > 0 ? hi : lo) plus zero times the other bound (NaN where that is infinite or NaN).
// With `narrow` (scores well inside the fp32 range) the products of two bf16 values are exact in
// fp32 and are summed as an unevaluated pair of fp32 values (Knuth's two-sum, about 2^-46 relative),
// several times faster here than in fp64, which takes the rest. Equal bounds give equal keys. The
// loops stay rolled: few rows come here, and most of what a long body would cost them is fetching it.
template <bool NARROW>
__device__ __noinline__ unsigned long long exact_key(const __nv_bfloat16* __restrict__ bounds_row,
                                                     const __nv_bfloat16* __restrict__ q, int lane) {
    const int d = 16 * (lane & 7);
    float sum = 0.f, rest = 0.f;
    double wide = 0.0;
    // (sum, rest) += (t, r); the same bits whichever side is which
    const auto add = [&](float t, float r) {
        const float n = __fadd_rn(sum, t), z = __fadd_rn(n, -sum);
        const float err = __fadd_rn(__fadd_rn(sum, -__fadd_rn(n, -z)), __fadd_rn(t, -z));
        rest = __fadd_rn(__fadd_rn(rest, r), err);
        sum = n;
    };
#pragma unroll 1
    for (int i = 0; i < 16; i += 8) {
        const uint4 xv = *reinterpret_cast<const uint4*>(q + d + i);
        const uint4 lv = *reinterpret_cast<const uint4*>(bounds_row + d + i);
        const uint4 hv = *reinterpret_cast<const uint4*>(bounds_row + kHd + d + i);
        const uint32_t x[4] = {xv.x, xv.y, xv.z, xv.w};
        const uint32_t lo[4] = {lv.x, lv.y, lv.z, lv.w};
        const uint32_t hi[4] = {hv.x, hv.y, hv.z, hv.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float f = e & 1 ? bf16hi(x[e >> 1]) : bf16lo(x[e >> 1]);
            const float l = e & 1 ? bf16hi(lo[e >> 1]) : bf16lo(lo[e >> 1]);
            const float h = e & 1 ? bf16hi(hi[e >> 1]) : bf16lo(hi[e >> 1]);
            const float mine = f > 0.f ? h : l, other = __fmul_rn(0.f, f > 0.f ? l : h);
            if constexpr (NARROW) add(__fmul_rn(f, mine), other);
            else wide += static_cast<double>(f) * mine + other;
        }
    }
#pragma unroll 1
    for (int o = 4; o > 0; o >>= 1) {
        if constexpr (NARROW) {
            const float t = __shfl_xor_sync(0xffffffffu, sum, o);
            add(t, __shfl_xor_sync(0xffffffffu, rest, o));
        } else {
            wide += __shfl_xor_sync(0xffffffffu, wide, o);
        }
    }
    if constexpr (NARROW) {
        const float top = __fadd_rn(sum, rest), low = __fadd_rn(rest, -__fadd_rn(top, -sum));
        return static_cast<unsigned long long>(key_of(top)) << 32 | key_of(low);
    } else {
        return key_of(wide);
    }
}

// Bit number of the lane group's set bit: the group's index (0 .. 3) from the lowest, at most the last.
__device__ __forceinline__ int group_bit(unsigned m, int lane) {
    int b = __ffs(m) - 1;
#pragma unroll
    for (int e = 1; e < 4; ++e) {
        m &= m - 1;
        if (e <= (lane >> 3) && m) b = __ffs(m) - 1;
    }
    return b;
}

constexpr int kListCap = 32;    // candidates resolved by one warp, one a lane
constexpr int kListGoal = 16;   // the search stops at that many

// The W warps of one row. With W = 1 the CTA's warps hold rows of their own.
template <int W>
struct RowGroup {
    struct Shared {
        uint32_t red[2][32];
        unsigned long long red64[2][32];
        uint32_t key[kListCap];
        int page[kListCap];
        unsigned long long exact[kListCap];  // of the open pages
        int open[kListCap];
        int n, req, n_open;
    };
    Shared& sh;
    int warp, lane, turn;

    __device__ __forceinline__ void sync() const {
        if (W == 1) __syncwarp();
        else __syncthreads();
    }
    // Sums / minima / maxima over the row's threads, one barrier each (the slots alternate).
    template <class Op>
    __device__ __forceinline__ uint32_t reduce(uint32_t v, uint32_t none, Op op) {
        v = op(v);
        if (W == 1) return v;
        turn ^= 1;
        if (lane == 0) sh.red[turn][warp] = v;
        __syncthreads();
        return op(lane < W ? sh.red[turn][lane] : none);
    }
    __device__ __forceinline__ uint32_t sum(uint32_t v) {
        return reduce(v, 0u, [](uint32_t x) { return __reduce_add_sync(0xffffffffu, x); });
    }
    __device__ __forceinline__ uint32_t least(uint32_t v) {
        return reduce(v, 0xffffffffu, [](uint32_t x) { return __reduce_min_sync(0xffffffffu, x); });
    }
    __device__ __forceinline__ uint32_t most(uint32_t v) {
        return reduce(v, 0u, [](uint32_t x) { return __reduce_max_sync(0xffffffffu, x); });
    }
    template <bool MAX>
    __device__ __forceinline__ unsigned long long pick64(unsigned long long v) {
        const auto op = [](unsigned long long x) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const unsigned long long y = __shfl_xor_sync(0xffffffffu, x, o);
                x = MAX ? max(x, y) : min(x, y);
            }
            return x;
        };
        v = op(v);
        if (W == 1) return v;
        turn ^= 1;
        if (lane == 0) sh.red64[turn][warp] = v;
        __syncthreads();
        return op(lane < W ? sh.red64[turn][lane] : (MAX ? 0ull : ~0ull));
    }
    // The count of the warps before this one; v is uniform in a warp.
    __device__ __forceinline__ uint32_t before(uint32_t v) {
        if (W == 1) return 0;
        turn ^= 1;
        if (lane == 0) sh.red[turn][warp] = v;
        __syncthreads();
        return __reduce_add_sync(0xffffffffu, lane < warp ? sh.red[turn][lane] : 0u);
    }
};

// W warps per row, K pages per lane: lane l of warp w holds pages 32 (w K + i) + l, i < K, as keys
// in registers. R rows per CTA (W = 1 only). The k-th largest key is found by bisection of the
// key range (a count per step); once at most kListGoal keys are left between the bounds, the keys
// within two error bounds of them go to a list of one key a lane, which one warp resolves by
// ranks, scored again beyond fp32 where that cannot tell.
template <int W, int K, int R>
__global__ void __launch_bounds__(32 * W * R)
select_pages_kernel(const SelectArgs a, int num_rows) {
    __shared__ typename RowGroup<W>::Shared shared[R];
    __shared__ uint32_t picked[R][W * K];  // bits of listed pages that were taken
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int slot = W == 1 ? wid : 0;
    const int id = static_cast<int>(blockIdx.x) * R + slot;
    if (id >= num_rows) return;
    auto& sh = shared[slot];
    RowGroup<W> row{sh, W == 1 ? 0 : wid, lane, 0};
    const int tid = row.warp * 32 + lane;
    const int t = a.t0 + id / a.hkv, h = id % a.hkv;
    int r = t;
    if (a.q_indptr) {  // the request that owns row t
        if (tid == 0) sh.req = -1;
        row.sync();
        for (int i = tid; i < a.num_reqs; i += 32 * W)
            if (a.q_indptr[i] <= t && t < a.q_indptr[i + 1]) sh.req = i;
        row.sync();
        r = sh.req;
        if (r < 0) return;  // a row behind the last sequence: left as it was
    }
    const bool report = h == 0 && tid == 0;
    const Window w = request_window(r, a.seq_lens, a.q_indptr, a.max_len, report, a.err);
    int* out = a.page_ids + (static_cast<int64_t>(t) * a.hkv + h) * a.top;
    if (t - w.q0 >= a.max_q_len) {  // more rows than the caller announced
        if (report) record_error(a.err, MSGL_ERR_BOUNDS, 801);
        for (int i = tid; i < a.top; i += 32 * W) out[i] = -1;
        return;
    }
    const int pos = w.L - w.qn + (t - w.q0);
    const int seen = pos < 0 ? 0 : pos / kPage + 1;
    if (seen <= a.top) {
        for (int i = tid; i < a.top; i += 32 * W) out[i] = i < seen ? i : -1;
        return;
    }
    const int first = a.sink, last = seen - a.recent;  // candidates; forced pages outside
    const int need = a.top - a.sink - a.recent;
    const int G = a.hq / a.hkv;
    for (int i = tid; i < a.sink; i += 32 * W) out[i] = i;
    for (int i = tid; i < a.recent; i += 32 * W) out[a.top - a.recent + i] = last + i;
    if (need == 0) return;

    const int64_t srow = (static_cast<int64_t>(t - a.t0) * a.hkv + h) * a.stride;
    const float* mrow = a.mags + (static_cast<int64_t>(max(w.q0, a.t0) - a.t0) * a.hkv + h) * (a.stride / 16);
    const __nv_bfloat16* qrow = a.q + (static_cast<int64_t>(t) * a.hq + h * G) * kHd;
    const int base = row.warp * K * 32 + lane;
    // all loads first: scores, query rows, magnitudes
    uint32_t key[K];
    float mag = 0.f;
    {
        const float* __restrict__ scores = a.scores + srow;
        float v[K];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int j = base + 32 * i;
            v[i] = j >= first && j < last ? scores[j] : 0.f;
        }
        for (int j = first / 16 + tid; j <= (last - 1) / 16; j += 32 * W) mag = fmaxf(mag, mrow[j]);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int j = base + 32 * i;
            key[i] = j >= first && j < last ? key_of(v[i]) : 0u;
        }
    }
    for (int i = lane; i < K; i += 32) picked[slot][row.warp * K + i] = 0u;
    // |fp32 score - exact| <= 2^-15 sum |products|: a step of an MMA chain adds 16 products and the
    // partial sum, each cut at worst at one unit (2^-23) of the largest; 8 steps a chain, half the
    // products in each of two chains and one addition make 2^-15.9. sum |products| <= |q| |max(|lo|,
    // |hi|)| (2-norms; the margin left covers their own rounding).
    float norm = 0.f;  // four lanes a head
    if (lane >> 2 < G) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 u = *reinterpret_cast<const uint4*>(qrow + (lane >> 2) * kHd + 32 * i + 8 * (lane & 3));
            const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) norm += bf16lo(x[e]) * bf16lo(x[e]) + bf16hi(x[e]) * bf16hi(x[e]);
        }
    }
    norm += __shfl_xor_sync(0xffffffffu, norm, 1);
    norm += __shfl_xor_sync(0xffffffffu, norm, 2);
    norm = sqrtf(warp_max(norm != norm ? __builtin_huge_valf() : norm));
    if (tid == 0) sh.n = 0;
    row.sync();  // the cleared bits and count
    uint32_t lo = 0xffffffffu, hi = 0u;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        lo = min(lo, key[i] ? key[i] : 0xffffffffu);
        hi = max(hi, key[i]);
    }
    lo = row.least(lo);
    hi = row.most(hi);
    const float scale = norm * __uint_as_float(row.most(__float_as_uint(mag)));
    const bool bounded = scale < 1e37f;  // else fp32 may have overflowed: all pages again
    const bool narrow = scale > 1e-20f && scale < 1e37f;
    const float eps2 = 2.f * (scale * 3.0517578125e-5f + 1e-30f);  // two errors

    const auto count_from = [&](uint32_t v) {
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < K; ++i) c += key[i] >= v;
        return static_cast<int>(row.sum(c));
    };
    // count(key >= lo) = n_lo >= need > n_hi = count(key > hi)
    int n_lo = last - first, n_hi = 0;
    while (bounded && lo < hi && n_lo - n_hi > kListGoal) {
        const uint32_t mid = hi - ((hi - lo) >> 1);
        const int c = count_from(mid);
        if (c >= need) {
            lo = mid;
            n_lo = c;
        } else {
            hi = mid - 1;
            n_hi = c;
        }
    }
    // every key within two errors of the k-th largest lies in [low, high]
    uint32_t low = lo, high = hi;
    if (!bounded) {
        low = 1u;
        high = 0xffffffffu;
    } else {
        if (lo <= kInfKey) low = key_of(__fadd_rd(value_of(lo), -eps2));
        high = hi <= kInfKey ? key_of(__fadd_ru(value_of(hi), eps2)) : 0xffffffffu;
    }
    uint32_t above = 0, inside = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        above += key[i] > high;
        inside += key[i] >= low && key[i] <= high;
    }
    const uint32_t both = row.sum(above | inside << 16);
    const int want = need - static_cast<int>(both & 0xffffu), listed = static_cast<int>(both >> 16);
    const auto bounds_of = [&](int j) {
        int phys = a.page_table[static_cast<int64_t>(r) * a.max_pages + j];
        if (static_cast<unsigned>(phys) >= static_cast<unsigned>(a.pool_pages)) phys = 0;  // recorded
        return a.bounds + (static_cast<int64_t>(phys) * a.hkv + h) * 2 * kHd;
    };
    const auto again = [&](int j, int g) {
        const __nv_bfloat16* b = bounds_of(j);
        return narrow ? exact_key<true>(b, qrow + g * kHd, lane) : exact_key<false>(b, qrow + g * kHd, lane);
    };
    if (listed == want) {
        high = low - 1;  // all of them
    } else if (listed <= kListCap) {
        if (inside) {
            int p = atomicAdd(&sh.n, static_cast<int>(inside));
#pragma unroll
            for (int i = 0; i < K; ++i)
                if (key[i] >= low && key[i] <= high) {
                    sh.key[p] = key[i];
                    sh.page[p++] = base + 32 * i;
                }
        }
        row.sync();
        bool take = false, mine_open = false;
        int page = 0, left = 0;
        if (row.warp == 0) {
            const uint32_t mine = lane < listed ? sh.key[lane] : 0u;
            page = lane < listed ? sh.page[lane] : 0;
            int more = 0, same = 0;
#pragma unroll
            for (int o = 0; o < 32; ++o) {
                const uint32_t k = __shfl_sync(0xffffffffu, mine, o);
                more += k > mine;
                same += k == mine;
            }
            // the keys of rank `want` and `want + 1` (if listed)
            const unsigned is_kth = __ballot_sync(0xffffffffu, more < want && want <= more + same);
            const unsigned is_next = __ballot_sync(0xffffffffu, mine && more <= want && want < more + same);
            const uint32_t kth = __shfl_sync(0xffffffffu, mine, __ffs(is_kth) - 1);
            const uint32_t next = is_next ? __shfl_sync(0xffffffffu, mine, __ffs(is_next) - 1) : 0u;
            // A score more than two errors above the next one is larger than all from there on, one
            // more than two errors below the k-th smaller than k others; the rest is open.
            uint32_t top_key = 0xffffffffu, low_key = 1u;
            if (bounded) {
                low_key = kth > kInfKey ? kth : key_of(__fadd_rd(value_of(kth), -eps2));
                if (next == 0u) top_key = 0u;
                else if (next <= kInfKey) top_key = key_of(__fadd_ru(value_of(next), eps2));
            }
            take = mine > top_key && mine >= low_key;
            mine_open = mine && !take && mine >= low_key;
            const unsigned open = __ballot_sync(0xffffffffu, mine_open);
            left = want - __popc(__ballot_sync(0xffffffffu, take));
            if (__popc(open) <= left) {
                take = take || mine_open;
                mine_open = false;
                if (lane == 0) sh.n_open = 0;
            } else {
                if (lane == 0) sh.n_open = __popc(open);
                if (mine_open) {
                    const int i = __popc(open & ((1u << lane) - 1));
                    sh.open[i] = page;
                    sh.exact[i] = 0ull;
                }
            }
        }
        row.sync();
        const int n_open = sh.n_open;
        if (n_open) {  // scored again: a page and head per group of eight lanes, over all warps
            for (int i0 = row.warp * 4; i0 < n_open * G; i0 += 4 * W) {
                const int i = min(i0 + (lane >> 3), n_open * G - 1);
                const unsigned long long k = again(sh.open[i / G], i % G);
                if ((lane & 7) == 0) atomicMax(&sh.exact[i / G], k);
            }
            row.sync();
        }
        if (row.warp == 0) {
            if (mine_open) {
                unsigned long long k = 0ull;
                for (int o = 0; o < n_open; ++o)
                    if (sh.open[o] == page) k = sh.exact[o];
                int rank = 0;  // by (score, lower page)
                for (int o = 0; o < n_open; ++o)
                    rank += sh.exact[o] > k || (sh.exact[o] == k && sh.open[o] < page);
                take = rank < left;
            }
            if (take) atomicOr(&picked[slot][page >> 5], 1u << (page & 31));
        }
        row.sync();
    } else {
        // more than the list holds (equal pages, values beyond fp32): all of them scored again into
        // the workspace, bisection of those keys
        unsigned long long* wide = a.wide + srow;
#pragma unroll 1
        for (int i = 0; i < K; ++i) {
            const int j0 = base - lane + 32 * i;
            const uint32_t k = j0 + lane >= first && j0 + lane < last ? key_of(a.scores[srow + j0 + lane]) : 0u;
            unsigned m = __ballot_sync(0xffffffffu, k >= low && k <= high);
            while (m) {  // four pages at a time
                const int j = j0 + group_bit(m, lane);
                unsigned long long k = 0ull;
                for (int g = 0; g < G; ++g) k = max(k, again(j, g));
                wide[j] = k;
#pragma unroll
                for (int e = 0; e < 4; ++e) m &= m - 1;
            }
        }
        row.sync();  // (a warp reads back only what it wrote)
        const auto each = [&](auto f) {
#pragma unroll 1
            for (int i = 0; i < K; ++i) {
                const int j = base + 32 * i;
                const uint32_t k = j >= first && j < last ? key_of(a.scores[srow + j]) : 0u;
                const bool in = k >= low && k <= high;
                f(i, in ? __ldcg(wide + j) : 0ull, in);
            }
        };
        unsigned long long wlo = ~0ull, whi = 0ull;
        each([&](int, unsigned long long k, bool in) {
            if (in) wlo = min(wlo, k);
            whi = max(whi, k);
        });
        wlo = row.template pick64<false>(wlo);
        whi = row.template pick64<true>(whi);
        while (wlo < whi) {
            const unsigned long long mid = whi - ((whi - wlo) >> 1);
            uint32_t c = 0;
            each([&](int, unsigned long long k, bool in) { c += in && k >= mid; });
            if (static_cast<int>(row.sum(c)) >= want) wlo = mid;
            else whi = mid - 1;
        }
        uint32_t more = 0, same = 0;  // above the edge; at it, in this warp
        each([&](int, unsigned long long k, bool in) {
            more += in && k > wlo;
            same += __popc(__ballot_sync(0xffffffffu, in && k == wlo));
        });
        const int equal = want - static_cast<int>(row.sum(more));  // taken at the edge, lowest first
        int rank = static_cast<int>(row.before(same));
        each([&](int i, unsigned long long k, bool in) {
            const unsigned e = __ballot_sync(0xffffffffu, in && k == wlo);
            const bool take = in && (k > wlo || (k == wlo && rank + __popc(e & ((1u << lane) - 1)) < equal));
            const unsigned bits = __ballot_sync(0xffffffffu, take);
            if (lane == 0) picked[slot][row.warp * K + i] = bits;
            rank += __popc(e);
        });
        row.sync();
    }
    // ascending output between the sink and the recent pages: lane i writes out word i of the warp
    uint32_t bits = lane < K ? picked[slot][row.warp * K + lane] : 0u;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const uint32_t sure = __ballot_sync(0xffffffffu, key[i] > high);
        if (lane == i) bits |= sure;
    }
    int incl = __popc(bits);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    const int mine = __shfl_sync(0xffffffffu, incl, 31);
    int at = a.sink + static_cast<int>(row.before(mine)) + incl - __popc(bits);
    for (; bits; bits &= bits - 1) out[at++] = (row.warp * K + lane) * 32 + __ffs(bits) - 1;
}

// ------------------------------------------------------------------ attention over the lists
// A row's list is read as a set: the listed pages become bits (decode) or row masks (chunks) over
// the context's pages, and a scan over those gives one ascending list without repeats.
//
// A page's 16 keys are the 16 MMA rows and the 8 MMA columns are 8 / G query rows x the G query
// heads of one kv head: S^T = K Q^T and O^T = V^T P^T, 8 MMAs each per page. With the columns as
// MMA rows (16 of them) a single token fills at most half of the tile, and a tile of four tokens
// (G = 4) multiplies pages that only some of them listed: 32 MMAs a page and twice the registers.
constexpr int kAttWarps = 4;
constexpr int kAttThreads = kAttWarps * 32;
constexpr int kPageBytes = 2 * kPage * kHd * 2;  // K and V of one page and kv head

struct AttArgs {
    const __nv_bfloat16 *q, *k_pool, *v_pool;
    int pool_pages;
    const int* page_table;
    int max_pages;
    const int *seq_lens, *q_indptr;
    int total_q, max_q_len, max_len;
    const int* page_ids;
    int top, hq, hkv;
    float sl2e;
    __nv_bfloat16* out;
    int* err;
};

// Running state of a warp's online softmax. Lane (g, c) holds dims 16 j + g (+ 8) of columns 2 c and
// 2 c + 1, the columns' maxima and this lane's part of their sums.
struct Softmax {
    float o[8][4];
    float m[2], l[2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        m[0] = m[1] = kNegInf;
        l[0] = l[1] = 0.f;
    }
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// One page (16 keys) for one warp. K and V tiles: halves of 64 dims, rows of 128 bytes, 16-byte
// pieces swizzled by the row; with PADDED rows of kPadRow bytes, 16 more than they hold, which sets
// the rows of a fragment 16 bytes apart in the banks as well. qb: column g's query as the B operand. lim0 / lim1: last visible
// offset in the page for columns 2 c / 2 c + 1 (< 0: the page is not of that column). With PART,
// only columns whose own limit is >= 0 take the new sums (the others' P is zero, but zero times a
// NaN or infinite value of a page that is not theirs must not reach them), and V rows behind vlim
// count as zero for the same reason. The second term of P takes no infinite values, as it may be zero or
// of the other sign: in chunks only with PART, which a pass whose sums are not finite is followed by; in
// single rows always (a second pass with a loop of its own cost 1 us at 4k, this 0.3).
constexpr int kPadRow = kHd * 2 + 16;
constexpr int kPadTile = kPage * kPadRow;
template <bool PART, bool PADDED>
__device__ __forceinline__ void attend(uint32_t base, const uint32_t (&qb)[8][2], Softmax& st,
                                       int lim0, int lim1, int vlim, float sl2e, int lane) {
    const int mi = lane >> 3, g = lane >> 2, c = lane & 3;
    // The asm statements keep their order, so fragments are loaded some steps ahead of the MMAs that
    // take them: kAhead of K, then half of V before the softmax and the rest behind it.
    constexpr int kAhead = PADDED ? 6 : 8;  // chunks have 96 registers a thread
    uint32_t f[kAhead][4];
    const auto load_k = [&](int kk) {
        const int row = ((mi & 1) << 3) + (lane & 7);
        const int piece = ((kk & 3) << 1) + (mi >> 1);
        const uint32_t at = PADDED ? row * kPadRow + ((2 * kk + (mi >> 1)) << 4)
                                   : ((kk >> 2) << 11) + row * 128 + ((piece ^ (row & 7)) << 4);
        uint32_t(&x)[4] = f[kk % kAhead];
        ldsm_x4(base + at, x[0], x[1], x[2], x[3]);
    };
#pragma unroll
    for (int kk = 0; kk < kAhead; ++kk) load_k(kk);
    float s[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {  // two chains
        const uint32_t(&x)[4] = f[kk % kAhead];
        mma_bf16_16816(s[kk & 1], x[0], x[1], x[2], x[3], qb[kk][0], qb[kk][1]);
        if (kk + kAhead < 8) load_k(kk + kAhead);
    }
    const uint32_t vb = base + (PADDED ? kPadTile : kPageBytes / 2);
    const auto load_v = [&](int j) {
        const int row = ((mi >> 1) << 3) + (lane & 7);
        const int piece = ((j & 3) << 1) + (mi & 1);
        const uint32_t at = PADDED ? row * kPadRow + ((2 * j + (mi & 1)) << 4)
                                   : ((j >> 2) << 11) + row * 128 + ((piece ^ (row & 7)) << 4);
        uint32_t(&x)[4] = f[j % kAhead];
        ldsm_x4_t(vb + at, x[0], x[1], x[2], x[3]);
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) load_v(j);
    // p[e]: key g (e < 2) or g + 8, column 2 c + e % 2
    float p[4], old[2] = {st.m[0], st.m[1]};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        p[e] = g + (e >> 1) * 8 <= (e & 1 ? lim1 : lim0) ? (s[0][e] + s[1][e]) * sl2e : kNegInf;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        float mx = fmaxf(p[r], p[2 + r]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        st.m[r] = fmaxf(st.m[r], mx);
    }
    if (__any_sync(0xffffffffu, st.m[0] != old[0] || st.m[1] != old[1])) {  // a maximum rose: rescale
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float alpha = st.m[r] == kNegInf ? 1.f : exp2f(old[r] - st.m[r]);
            st.l[r] *= alpha;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                st.o[j][r] *= alpha;
                st.o[j][2 + r] *= alpha;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        p[e] = exp2f(p[e] - (st.m[e & 1] == kNegInf ? 0.f : st.m[e & 1]));
        st.l[e & 1] += p[e];
    }
    // P as two bf16 terms, which leaves 2^-16 of a weight out. One term leaves 2^-8 of each, which where
    // the values cancel is far more than the rounding of the result. (Selection and attention of 1.3k rows
    // of 64 pages: 460 us with one term, 494 with two; 64 requests 169.3 and 170.4.)
    const uint32_t h0 = pack_bf16x2(p[0], p[1]), h1 = pack_bf16x2(p[2], p[3]);
    const uint32_t b0 = transpose8x8(h0), b1 = transpose8x8(h1);
    const uint32_t r0 = transpose8x8(pack_bf16x2(p[0] - bf16lo(h0), p[1] - bf16hi(h0)));
    const uint32_t r1 = transpose8x8(pack_bf16x2(p[2] - bf16lo(h1), p[3] - bf16hi(h1)));
#pragma unroll
    for (int j = 4; j < kAhead; ++j) load_v(j);
    // V fragments hold keys (2c, 2c + 1) and (2c + 8, 2c + 9)
    uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
    if (PART) {
        keep0 = (2 * c <= vlim ? 0xffffu : 0u) | (2 * c + 1 <= vlim ? 0xffff0000u : 0u);
        keep1 = (2 * c + 8 <= vlim ? 0xffffu : 0u) | (2 * c + 9 <= vlim ? 0xffff0000u : 0u);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t(&x)[4] = f[j % kAhead];
        if (!PART) {
            const auto part = [](uint32_t v) { return PADDED ? v : finite2(v); };
            mma_bf16_16816(st.o[j], part(x[0]), part(x[1]), part(x[2]), part(x[3]), r0, r1);
            mma_bf16_16816(st.o[j], x[0], x[1], x[2], x[3], b0, b1);
        } else {
            const uint32_t y[4] = {x[0] & keep0, x[1] & keep0, x[2] & keep1, x[3] & keep1};
            float d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = st.o[j][e];
            mma_bf16_16816(d, finite2(y[0]), finite2(y[1]), finite2(y[2]), finite2(y[3]), r0, r1);
            mma_bf16_16816(d, y[0], y[1], y[2], y[3], b0, b1);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if ((e & 1 ? lim1 : lim0) >= 0) st.o[j][e] = d[e];
        }
        if (j + kAhead < 8) load_v(j + kAhead);
    }
}

__device__ __forceinline__ void dump_sums(const Softmax& st, float* m, float* l, int lane) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        float sum = st.l[r];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (g == 0) {
            m[2 * c + r] = st.m[r];
            l[2 * c + r] = sum;
        }
    }
}

// A warp's state into shared memory: o rows of kPad floats per column, m and l per column.
constexpr int kPad = kHd + 4;  // the four lanes of a dim fall into different banks
__device__ __forceinline__ void dump(const Softmax& st, float* o, float* m, float* l, int lane) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[(2 * c + (e & 1)) * kPad + 16 * j + g + (e >> 1) * 8] = st.o[j][e];
    dump_sums(st, m, l, lane);
}

// 8 dims of one column joined over `n` dumped states, `step` columns' worth apart: M and L of the
// column and its unnormalised values.
__device__ __forceinline__ void join(const float* o, const float* m, const float* l, int n, int step,
                                     float& M, float& L, float (&acc)[8]) {
    M = kNegInf;
    for (int k = 0; k < n; ++k) M = fmaxf(M, m[k * step]);
    L = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    for (int k = 0; k < n; ++k) {
        const float mk = m[k * step], lk = l[k * step];
        if (mk == kNegInf && lk == 0.f) continue;  // saw no key
        const float sc = exp2f(mk - M);
        L += lk * sc;
        const float4 u = *reinterpret_cast<const float4*>(o + k * step * kPad);
        const float4 v = *reinterpret_cast<const float4*>(o + k * step * kPad + 4);
        acc[0] += u.x * sc; acc[1] += u.y * sc; acc[2] += u.z * sc; acc[3] += u.w * sc;
        acc[4] += v.x * sc; acc[5] += v.y * sc; acc[6] += v.z * sc; acc[7] += v.w * sc;
    }
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8], float f) {
    return make_uint4(pack_bf16x2(v[0] * f, v[1] * f), pack_bf16x2(v[2] * f, v[3] * f),
                      pack_bf16x2(v[4] * f, v[5] * f), pack_bf16x2(v[6] * f, v[7] * f));
}

// ---- single rows: decode, and short chunks
// Lists attended one by one, also in chunks whose tiles would be half empty or too few (at most kRowsAlone
// rows a request, or kTotalAlone rows in all). Selection and attention, 64 of 512 pages, 32 / 8 heads: 8
// requests x 17 / 33 / 48 / 65 rows take 96 / 158 / 215 / 283 us this way and 96 / 164 / 168 / 222 in tiles,
// one of 129 / 257 / 513 rows 88 / 143 / 270 and 99 / 101 / 169. The rows at which the two cross move
// with the query group: 8 x 33 rows take 170 and 179 at 64 / 8 heads, 146 and 104 at 16 / 8.
// A cluster of up to 16 CTAs (decode_split) per (query row, kv head): each CTA
// takes a share of the listed pages, its four warps take its pages in turn, every warp with a ring
// of its own (cp.async, 16 bytes a lane, three pages) and an online softmax. The warps' results are
// joined in shared memory, the CTAs' through distributed shared memory, each CTA finishing a share
// of the output: no workspace, one launch, a fixed order.
constexpr int kRowsAlone = 32, kTotalAlone = 256;
constexpr int kDecStages = 3;
constexpr int kDecRing = kAttWarps * kDecStages * kPageBytes;

__global__ void __launch_bounds__(kAttThreads, 2)
attend_pages_decode_kernel(const AttArgs a, int num_reqs, int words) {
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* ring = smem;                                           // kDecRing
    uint32_t* bits = reinterpret_cast<uint32_t*>(smem + kDecRing);  // [words]
    int* list_phys = reinterpret_cast<int*>(bits + words);          // [top]
    int* list_page = list_phys + a.top;                             // [top]
    __shared__ int scan[32];
    __shared__ float cm[8], cl[8];  // joined maximum and sum per query head
    __shared__ int owner, listed;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int S = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
    for (int i = threadIdx.x; i < words; i += kAttThreads) bits[i] = 0;
    pdl_wait();
    pdl_trigger();
    const int id = static_cast<int>(blockIdx.x) / S;
    const int h = id % a.hkv, t = id / a.hkv;
    const int G = a.hq / a.hkv;
    // the loads that only the row decides, ahead of those of its request
    const int* ids = a.page_ids + (static_cast<int64_t>(t) * a.hkv + h) * a.top;
    const int id0 = static_cast<int>(threadIdx.x) < a.top ? ids[threadIdx.x] : -1;
    uint32_t qb[8][2];
    {
        const __nv_bfloat16* qr = a.q + (static_cast<int64_t>(t) * a.hq + h * G + g) * kHd;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
            qb[kk][0] = g < G ? *reinterpret_cast<const uint32_t*>(qr + 16 * kk + 2 * c) : 0u;
            qb[kk][1] = g < G ? *reinterpret_cast<const uint32_t*>(qr + 16 * kk + 8 + 2 * c) : 0u;
        }
    }
    if (threadIdx.x == 0) listed = 0;
    int r = t;
    if (a.q_indptr) {  // the request that owns row t
        if (threadIdx.x == 0) owner = -1;
        __syncthreads();
        for (int i = threadIdx.x; i < num_reqs; i += kAttThreads)
            if (a.q_indptr[i] <= t && t < a.q_indptr[i + 1]) owner = i;
        __syncthreads();
        r = owner;
        if (r < 0) return;  // a row behind the last request: left as it was (the whole cluster)
    }
    const bool report = h == 0 && rank == 0 && threadIdx.x == 0;
    const Window w = request_window(r, a.seq_lens, a.q_indptr, a.max_len, report, a.err);
    const bool fits = w.q0 >= 0 && w.qn <= a.max_q_len && w.q0 + static_cast<int64_t>(w.qn) <= a.total_q;
    if (report && !fits) record_error(a.err, MSGL_ERR_BOUNDS, 801);
    if (!fits) return;  // the whole cluster
    const int pos = w.L - w.qn + (t - w.q0);
    for (int i = threadIdx.x; i < a.top; i += kAttThreads) list_page[i] = i < kAttThreads ? id0 : ids[i];
    __syncthreads();
    // A list in ascending order, as selection writes it, is taken as it is; any other is put in order and
    // rid of repeats through a bitmap, 0.8 us more.
    bool other = false;
    for (int i = threadIdx.x; i < a.top; i += kAttThreads) {
        const int page = list_page[i], before = i ? list_page[i - 1] : -1;
        if (page < 0) continue;
        other = other || pos < 0 || page > pos / kPage || (i && (before < 0 || before >= page));
        if (i + 1 == a.top || list_page[i + 1] < 0) listed = i + 1;
    }
    const bool in_order = !__syncthreads_or(other);
    int total = listed;
    if (!in_order) {
        for (int i = threadIdx.x; i < a.top; i += kAttThreads) {
            const int page = ids[i];
            if (page < 0) continue;
            if (pos < 0 || page > pos / kPage) {
                if (rank == 0) record_error(a.err, MSGL_ERR_BOUNDS, 803);
                continue;
            }
            atomicOr(&bits[page >> 5], 1u << (page & 31));
        }
        __syncthreads();
        int per = 0;  // set bits of this thread's run of words
        const int run = (words + kAttThreads - 1) / kAttThreads;
        const int w_lo = min(words, static_cast<int>(threadIdx.x) * run), w_hi = min(words, w_lo + run);
        for (int i = w_lo; i < w_hi; ++i) per += __popc(bits[i]);
        int at = block_excl_scan(per, scan, total);
        for (int i = w_lo; i < w_hi; ++i)
            for (uint32_t b = bits[i]; b; b &= b - 1, ++at) list_page[at] = i * 32 + __ffs(b) - 1;
        __syncthreads();
    }
    const int lo = static_cast<int>(static_cast<int64_t>(total) * rank / S);  // this CTA's share
    const int count = static_cast<int>(static_cast<int64_t>(total) * (rank + 1) / S) - lo;
    list_page += lo;
    for (int i = threadIdx.x; i < count; i += kAttThreads) {  // all in flight together
        int phys = a.page_table[static_cast<int64_t>(r) * a.max_pages + list_page[i]];
        if (static_cast<unsigned>(phys) >= static_cast<unsigned>(a.pool_pages)) {
            record_error(a.err, MSGL_ERR_BOUNDS, 802);
            phys = 0;
        }
        list_phys[i] = phys;
    }
    __syncthreads();

    Softmax st;
    st.clear();
    const int mine = count > warp ? (count - warp + kAttWarps - 1) / kAttWarps : 0;
    const uint32_t ring0 = smem_u32(ring) + warp * kDecStages * kPageBytes;
    const int64_t stride = static_cast<int64_t>(a.hkv) * kHd;
    const auto issue = [&](int i) {
        const int e = warp + i * kAttWarps;
        const uint32_t dst = ring0 + (i % kDecStages) * kPageBytes;
        const int live = pos - list_page[e] * kPage;  // last row to load: zeros behind it
        const int64_t off = static_cast<int64_t>(list_phys[e]) * kPage * stride + h * kHd;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const int row = 2 * x + (lane >> 4), piece = lane & 15;
            const int64_t src = off + row * stride + piece * 8;
            const uint32_t d = dst + ((piece >> 3) << 11) + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
            cp_async16(d, a.k_pool + src, row <= live);
            cp_async16(d + kPageBytes / 2, a.v_pool + src, row <= live);
        }
    };
    for (int i = 0; i < kDecStages - 1; ++i) {
        if (i < mine) issue(i);
        cp_async_commit();
    }
    for (int i = 0; i < mine; ++i) {
        cp_async_wait<kDecStages - 2>();
        __syncwarp();
        if (i + kDecStages - 1 < mine) issue(i + kDecStages - 1);
        cp_async_commit();
        const int lim = pos - list_page[warp + i * kAttWarps] * kPage;
        attend<false, false>(ring0 + (i % kDecStages) * kPageBytes, qb, st, lim, lim, 0, a.sl2e, lane);
        __syncwarp();
    }

    // ---- join the warps' results (shared memory over the drained rings)
    cp_async_wait<0>();
    __syncthreads();
    float* mo = reinterpret_cast<float*>(ring);  // [4 warps][8][kPad]
    float* mm = mo + kAttWarps * 8 * kPad;       // [4][8]
    float* ml = mm + kAttWarps * 8;
    float* co = ml + kAttWarps * 8;              // [8][128]: joined, for the cluster
    dump(st, mo + warp * 8 * kPad, mm + warp * 8, ml + warp * 8, lane);
    __syncthreads();
    __nv_bfloat16* out = a.out + (static_cast<int64_t>(t) * a.hq + h * G) * kHd;
    for (int item = threadIdx.x; item < G * 16; item += kAttThreads) {
        const int head = item >> 4, d0 = (item & 15) * 8;
        float M, L, acc[8];
        join(mo + head * kPad + d0, mm + head, ml + head, kAttWarps, 8, M, L, acc);
        if (S == 1) {  // an empty list gives a zero row
            *reinterpret_cast<uint4*>(out + head * kHd + d0) = pack8(acc, L == 0.f ? 0.f : 1.f / L);
        } else {
            *reinterpret_cast<float4*>(co + head * kHd + d0) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            *reinterpret_cast<float4*>(co + head * kHd + d0 + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
            if (d0 == 0) {
                cm[head] = M;
                cl[head] = L;
            }
        }
    }
    if (S == 1) return;
    cluster_sync_all();
    // item (column, 8 dims) i of every S, its S parts loaded by as many neighbouring lanes
    const int part = threadIdx.x % S;
    for (int i0 = 0; i0 < G * 16; i0 += kAttThreads) {
        const int item = i0 + threadIdx.x / S * S + rank;
        const bool live = item < G * 16;
        const int head = live ? item >> 4 : 0, d0 = live ? (item & 15) * 8 : 0;
        const uint32_t src = mapa_shared(smem_u32(co + head * kHd + d0), part);
        const float mk = ld_dsmem_f32(mapa_shared(smem_u32(cm + head), part));
        const float lk = ld_dsmem_f32(mapa_shared(smem_u32(cl + head), part));
        const float4 u = ld_dsmem_v4(src), v = ld_dsmem_v4(src + 16);
        float M = mk;
        for (int o = 1; o < S; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        // parts that saw no key count nothing (their m may be the -inf that M is too)
        const float sc = mk == kNegInf && lk == 0.f ? 0.f : exp2f(mk - M);
        float L = lk * sc, acc[8] = {u.x * sc, u.y * sc, u.z * sc, u.w * sc, v.x * sc, v.y * sc, v.z * sc, v.w * sc};
        for (int o = 1; o < S; o <<= 1) {
            L += __shfl_xor_sync(0xffffffffu, L, o);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
        }
        if (live && part == 0)
            *reinterpret_cast<uint4*>(out + head * kHd + d0) = pack8(acc, L == 0.f ? 0.f : 1.f / L);
    }
    cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

// ---- chunks
// One CTA per (tile of one request's query rows, kv head): sixteen warps in RW row groups of TQ =
// 8 / G rows each (8 for G = 1, where that is 64 rows, else 16) times 16 / RW page groups, and a
// producer warp. The rows' lists are joined into one list of pages with a mask of the rows that asked
// for each, so a page that several neighbouring queries chose crosses from L2 once; a warp attends the
// pages that its own rows asked for, one in 16 / RW of them. Pages come by TMA (one 3-D box of K, one of
// V) through a ring shared by the warps, in stages of kStagePages: most warps skip most pages, and a
// barrier per page cost as much as the pages. Contexts longer than kWin pages are walked in windows
// of that many. A cluster of CTAs (chunk_split) shares a tile: each takes a share of every window's
// list, and the partial results are joined through distributed shared memory.
//
// Bound by shared memory: a warp's fragments of a page are 8 KB, 64 cycles of its port, and 5.3 of the
// 16 row groups want a page; with the write of the page 410 cycles, of some 580 that a page takes (1.3k
// rows of 32 heads over 64 pages each, 126k page loads: 371 us; a CTA's list and join are 8 of 70 us). With
// one bf16 term of P it was 525, and 338 us.
// A box is 16 rows of kPadRow bytes, wider than the tensor's rows: the rest is filled with zeros, which
// pads the rows. Boxes of swizzled half rows of 128 bytes took 225 cycles of the copy engine each and
// 36 us more in all. Slower ways to bring the same pages: cp.async from producer warps (it shares the
// path of the fragment loads), bulk copies of single rows, K by TMA and V by cp.async, tiles of 16
// rows on two CTAs per SM; 16 warps, the last to leave a stage filling it again, in place of the
// producer: 554 against 528 us.
//
// A masked weight is zero, but zero times a NaN or infinite value is NaN. Such values are looked
// for at the end instead of at every page: a row they reached is NaN from then on, so a tile
// without NaN or infinite sums was right, and any other is computed again with the masked values
// kept out (PART of attend).
constexpr int kChWarps = 16;
constexpr int kChThreads = (kChWarps + 1) * 32;
constexpr int kStagePages = 7;
constexpr int kChStages = 3;
constexpr int kStageBytes = kStagePages * 2 * kPadTile;
constexpr int kWin = 2048;
constexpr int kTileRows = 64;  // mask bits
constexpr int kChSmem = kChStages * kStageBytes + kWin * (8 + 4 + 2) + 1024;

__global__ void __launch_bounds__(kChThreads, 1)
attend_pages_chunk_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                          const AttArgs a, int tiles, int row_groups) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint32_t* masks = reinterpret_cast<uint32_t*>(ring + kChStages * kStageBytes);  // [2][kWin]: rows 0-31, 32-63
    int* list_phys = reinterpret_cast<int*>(masks + 2 * kWin);            // [kWin]
    uint16_t* list_page = reinterpret_cast<uint16_t*>(list_phys + kWin);  // [kWin], in the window
    __shared__ uint64_t full[kChStages], empty[kChStages];
    __shared__ int scan[32];
    __shared__ float sm[kChWarps * 8], sl[kChWarps * 8];

    if (threadIdx.x == 0) {
        for (int s = 0; s < kChStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], kChWarps);
        }
        fence_barrier_init();
        tma_prefetch_desc(&tk);
        tma_prefetch_desc(&tv);
    }
    for (int i = threadIdx.x; i < 2 * kWin; i += kChThreads) masks[i] = 0;
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int G = a.hq / a.hkv;
    const int lgG = 31 - __clz(G), TQ = 8 >> lgG;
    const int RW = row_groups, PW = kChWarps / RW, rg = warp % RW, pg = warp / RW;
    const int CS = static_cast<int>(cluster_nctarank()), rank = static_cast<int>(cluster_ctarank());
    int64_t id = static_cast<int>(blockIdx.x) / CS;
    const int h = static_cast<int>(id % a.hkv);
    id /= a.hkv;
    const int tile = static_cast<int>(id % tiles), r = static_cast<int>(id / tiles);
    const bool report = tile == 0 && h == 0 && rank == 0 && threadIdx.x == 0;
    const Window w = request_window(r, a.seq_lens, a.q_indptr, a.max_len, report, a.err);
    const bool fits = w.q0 >= 0 && w.qn >= 0 && w.qn <= a.max_q_len && w.q0 + static_cast<int64_t>(w.qn) <= a.total_q;
    if (report && !fits) record_error(a.err, MSGL_ERR_BOUNDS, 801);
    const int i0 = tile * RW * TQ;
    const int rows = min(RW * TQ, w.qn - i0);
    if (!fits || rows <= 0) return;  // the whole cluster
    const int pos0 = w.L - w.qn + i0;  // position of the tile's first row

    const int wrow = rg * TQ, wrows = max(0, min(TQ, rows - wrow));  // this warp's rows (may be none)
    const int row0 = (2 * c) >> lgG, row1 = (2 * c + 1) >> lgG;              // of columns 2 c, 2 c + 1, in the warp
    uint32_t qb[8][2];
    {
        const bool real = warp < kChWarps && (g >> lgG) < wrows;
        const __nv_bfloat16* qr =
            a.q + (static_cast<int64_t>(w.q0 + i0 + wrow + (g >> lgG)) * a.hq + h * G + (g & (G - 1))) * kHd;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
            qb[kk][0] = real ? *reinterpret_cast<const uint32_t*>(qr + 16 * kk + 2 * c) : 0u;
            qb[kk][1] = real ? *reinterpret_cast<const uint32_t*>(qr + 16 * kk + 8 + 2 * c) : 0u;
        }
    }
    Softmax st;
    const uint32_t wmask = warp < kChWarps ? (1u << wrows) - 1u : 0u;
    const int pages = (pos0 + rows - 1) < 0 ? 0 : (pos0 + rows - 1) / kPage + 1;
    bool ok = true;
    int done = 0;  // stages of earlier windows: ring slots and phases run on
    // One pass over the pages; true where a sum of this CTA is infinite or NaN. Two copies, so that the
    // registers of the careful one are not those of the other.
    const auto walk = [&](auto careful) {
        constexpr bool kCareful = decltype(careful)::value;
        st.clear();
        for (int w0 = 0; w0 < pages; w0 += kWin) {
            // Loads first, each kind together: the table of this thread's run of pages, then ids by fours.
            constexpr int kRun = kWin / (kChWarps * 32);
            const int run0 = static_cast<int>(threadIdx.x) * kRun;  // the producer warp has none
            int phys[kRun];
#pragma unroll
            for (int e = 0; e < kRun; ++e)
                phys[e] = warp < kChWarps && w0 + run0 + e < pages
                              ? a.page_table[static_cast<int64_t>(r) * a.max_pages + w0 + run0 + e] : 0;
            const int* ids = a.page_ids + (static_cast<int64_t>(w.q0 + i0) * a.hkv + h) * a.top;
            const int step_row = kChThreads / a.top, step_at = kChThreads % a.top;
            int row = threadIdx.x / a.top, at = threadIdx.x % a.top;
            int page[4], of[4];
            const auto load = [&] {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    page[e] = row < rows ? ids[static_cast<int64_t>(row) * a.hkv * a.top + at] : -1;
                    of[e] = row;
                    row += step_row;
                    at += step_at;
                    if (at >= a.top) {
                        at -= a.top;
                        ++row;
                    }
                }
            };
            load();
            __syncthreads();  // masks are zero
            for (;;) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (page[e] < 0) continue;
                    const int pos = pos0 + of[e];
                    if (pos < 0 || page[e] > pos / kPage) {
                        if (w0 == 0 && !kCareful && rank == 0) record_error(a.err, MSGL_ERR_BOUNDS, 803);
                        continue;
                    }
                    if (page[e] >= w0 && page[e] < w0 + kWin)
                        atomicOr(&masks[(of[e] >> 5) * kWin + page[e] - w0], 1u << (of[e] & 31));
                }
                if (row >= rows) break;
                load();
            }
            __syncthreads();
            uint32_t any[kRun];
            int per = 0;
#pragma unroll
            for (int e = 0; e < kRun; ++e) {
                any[e] = warp < kChWarps ? masks[run0 + e] | masks[kWin + run0 + e] : 0u;
                per += any[e] != 0;
            }
            int total;
            at = block_excl_scan(per, scan, total);
            const int lo = total * rank / CS, count = total * (rank + 1) / CS - lo;  // this CTA's share
            at -= lo;
#pragma unroll
            for (int e = 0; e < kRun; ++e) {
                if (!any[e]) continue;
                if (at >= 0 && at < count) {
                    if (static_cast<unsigned>(phys[e]) >= static_cast<unsigned>(a.pool_pages)) {
                        record_error(a.err, MSGL_ERR_BOUNDS, 802);
                        phys[e] = 0;
                    }
                    list_page[at] = static_cast<uint16_t>(run0 + e);
                    list_phys[at] = phys[e];
                }
                ++at;
            }
            __syncthreads();

            const int stages = (count + kStagePages - 1) / kStagePages;
            if (warp == kChWarps) {
                for (int i = 0; i < stages; ++i) {  // lane l loads K (even) or V of page l / 2
                    const int n = done + i, s = n % kChStages;
                    const int e0 = i * kStagePages, pages_in = min(kStagePages, count - e0);
                    const int y = lane < 2 * pages_in ? list_phys[e0 + lane / 2] * kPage : 0;
                    if (n >= kChStages)
                        ok = ok && __all_sync(0xffffffffu, mbar_wait(&empty[s], (n / kChStages - 1) & 1, a.err, 821));
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&full[s], pages_in * 2 * kPadTile);
                    __syncwarp();
                    if (lane < 2 * pages_in)
                        tma_load_3d(ring + s * kStageBytes + lane * kPadTile, lane & 1 ? &tv : &tk, &full[s], 0, h, y);
                    __syncwarp();
                }
            } else {
                for (int i = 0, mine = 0; i < stages; ++i) {
                    const int n = done + i, s = n % kChStages;
                    // lane e: page e of the stage, and which of this warp's rows want it
                    const int e = i * kStagePages + lane;
                    int page = 0;
                    uint32_t want = 0;
                    if (lane < kStagePages && e < count) {
                        page = list_page[e];
                        want = (masks[(wrow >> 5) * kWin + page] >> (wrow & 31)) & wmask;
                    }
                    unsigned some = __ballot_sync(0xffffffffu, want != 0);
                    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (n / kChStages) & 1, a.err, 820));
                    for (; some; some &= some - 1) {
                        const int x = __ffs(some) - 1;
                        if (!ok || (mine++ & (PW - 1)) != pg) continue;
                        const uint32_t mask = __shfl_sync(0xffffffffu, want, x);
                        const uint32_t base = smem_u32(ring) + s * kStageBytes + x * 2 * kPadTile;
                        // the first row's position in the page
                        const int rel = pos0 + wrow - (w0 + __shfl_sync(0xffffffffu, page, x)) * kPage;
                        if constexpr (!kCareful) {
                            attend<false, true>(base, qb, st, ((mask >> row0) & 1u) ? rel + row0 : -1,
                                          ((mask >> row1) & 1u) ? rel + row1 : -1, 0, a.sl2e, lane);
                        } else {
                            // rows that see the whole page go together, one that ends inside it alone
                            for (uint32_t left = mask; left;) {
                                const int row = __ffs(left) - 1;
                                const uint32_t now = rel + row >= kPage - 1 ? left : 1u << row;
                                left &= ~now;
                                attend<true, true>(base, qb, st, ((now >> row0) & 1u) ? rel + row : -1,
                                                   ((now >> row1) & 1u) ? rel + row : -1, rel + row, a.sl2e, lane);
                            }
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&empty[s]);
                }
            }
            done += stages;
            __syncthreads();
            for (int i = threadIdx.x; i < 2 * kWin; i += kChThreads) masks[i] = 0;  // of the next window
        }
        float sum = 0.f;  // NaN where a sum is infinite or NaN
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += 0.f * ((st.o[j][0] + st.o[j][1]) + (st.o[j][2] + st.o[j][3]));
        return __syncthreads_or(sum != sum) != 0;
    };
    if (walk(std::false_type{})) walk(std::true_type{});  // each CTA for itself

    // ---- join the page groups and the cluster's shares, normalise, store
    // A warp's state lies lane by lane, 16 bytes per 16 dims. The PW x CS warps of a row group each join
    // and store a share of the 128 dims, as MMA tiles.
    float4* mo = reinterpret_cast<float4*>(ring);  // [16 warps][8][32 lanes]
    if (warp < kChWarps) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            mo[(warp * 8 + j) * 32 + lane] = make_float4(st.o[j][0], st.o[j][1], st.o[j][2], st.o[j][3]);
        dump_sums(st, sm + warp * 8, sl + warp * 8, lane);
    }
    cluster_sync_all();
    const int parts = PW * CS, lgCS = 31 - __clz(CS);  // part p: page group p / CS of CTA p % CS
    const int self = pg * CS + rank, j0 = 8 * self / parts, j1 = 8 * (self + 1) / parts;
    if (warp < kChWarps && j0 < j1) {
        const auto at = [&](const void* x, int p) { return mapa_shared(smem_u32(x), p & (CS - 1)); };
        float M[2] = {kNegInf, kNegInf}, L[2] = {0.f, 0.f};
#pragma unroll 4
        for (int p = 0; p < parts; ++p) {
            const int col = ((p >> lgCS) * RW + rg) * 8 + 2 * c;
#pragma unroll
            for (int k = 0; k < 2; ++k) M[k] = fmaxf(M[k], ld_dsmem_f32(at(sm + col + k, p)));
        }
        const int tr = wrow + (g >> lgG);  // of column g, which this lane stores
        uint32_t* out = reinterpret_cast<uint32_t*>(
            a.out + (static_cast<int64_t>(w.q0 + i0 + tr) * a.hq + h * G + (g & (G - 1))) * kHd);
        float acc[8][4];
#pragma unroll
        for (int x = 0; x < 8; ++x) acc[x][0] = acc[x][1] = acc[x][2] = acc[x][3] = 0.f;
        for (int p = 0; p < parts; ++p) {  // a part's loads together
            const int from = (p >> lgCS) * RW + rg, col = from * 8 + 2 * c;
            float mk[2], lk[2];
            float4 o[8];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                mk[k] = ld_dsmem_f32(at(sm + col + k, p));
                lk[k] = ld_dsmem_f32(at(sl + col + k, p));
            }
            const uint32_t src = at(mo + (from * 8 + j0) * 32 + lane, p);
#pragma unroll
            for (int x = 0; x < 8; ++x)
                if (j0 + x < j1) o[x] = ld_dsmem_v4(src + x * 32 * 16);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (mk[k] == kNegInf && lk[k] == 0.f) continue;  // saw no key
                const float sc = exp2f(mk[k] - M[k]);
                L[k] += lk[k] * sc;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    if (j0 + x >= j1) continue;
                    acc[x][k] += (k ? o[x].y : o[x].x) * sc;
                    acc[x][2 + k] += (k ? o[x].w : o[x].z) * sc;
                }
            }
        }
        // an empty list gives a zero row
        const float f0 = L[0] == 0.f ? 0.f : 1.f / L[0], f1 = L[1] == 0.f ? 0.f : 1.f / L[1];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            if (j0 + x >= j1) break;
            const uint32_t lo = transpose8x8(pack_bf16x2(acc[x][0] * f0, acc[x][1] * f1));
            const uint32_t hi = transpose8x8(pack_bf16x2(acc[x][2] * f0, acc[x][3] * f1));
            if (tr < rows) {  // dims 16 j + 2 c, + 1 and those 8 further of column g
                out[8 * (j0 + x) + c] = lo;
                out[8 * (j0 + x) + 4 + c] = hi;
            }
        }
    }
    cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

// ------------------------------------------------------------------ host checks
int check_heads(int hq, int hkv, int head_dim, int page_size) {
    if (head_dim != kHd) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "sparse attention: head_dim must be 128");
    if (page_size != kPage) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "sparse attention: page_size must be 16");
    if (hkv <= 0 || hq <= 0 || hq % hkv) return set_error(MSGL_ERR_INVALID_ARG, "sparse attention: Hq % Hkv != 0");
    const int group = hq / hkv;
    if (group > 8 || (8 % group)) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "sparse attention: Hq/Hkv must be 1,2,4 or 8");
    return MSGL_OK;
}

int pages_of(int tokens) { return tokens / kPage + (tokens % kPage != 0); }

// Query rows of one launch pair: as many as keep the workspace (16 bytes per row, kv head and
// page) within 256 MB, so that the scores (a quarter of it) stay in L2 until they are read; at
// least 16. (1.3k rows of 1024 pages: 509 us in two passes of 128 MB, 494 in one.)
constexpr int64_t kSelectBytes = int64_t(256) << 20;
int slab_rows(int total_q, int stride, int hkv) {
    const int64_t rows = std::max<int64_t>(16, kSelectBytes / (int64_t(16) * stride * hkv));
    return static_cast<int>(std::min<int64_t>(total_q, rows));
}
// CTAs that share a list in decode: a power of two up to the largest cluster (16, above the portable
// 8), as many as two CTAs per SM hold, of at least 4 pages (one a warp) each.
int decode_split(int64_t lists, int top) {
    int s = 1;
    while (s < 16 && lists * s * 2 <= 2 * 148 && top >= 8 * s) s *= 2;
    return s;
}

// CTAs that share a tile of a chunk (up to 4): one SM holds one, and the rounds of 148 should be full.
// A share costs a list and a join of its own, about a tenth of a tile's time in twos and a third in
// fours. Selection and attention with tiles alone / in twos / in fours: 16 tiles 135 / 86 / 62 us, 136
// tiles 169 / 182 / 222, 344 tiles 508 / 494 / 621.
int chunk_split(int64_t tiles) {
    const double gain[3] = {1.0, 0.9, 0.63};
    int best = 1;
    double most = 0.0;
    for (int k = 0; k < 3; ++k) {
        const int64_t ctas = tiles << k, rounds = (ctas + 147) / 148;
        const double v = gain[k] * static_cast<double>(ctas) / static_cast<double>(148 * rounds);
        if (v > most) most = v, best = 1 << k;
    }
    return best;
}

// Opts the decode kernel in to clusters above the portable size, once per device.
cudaError_t large_clusters() {
    static std::atomic<bool> done[kMaxDevices];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool cached = dev >= 0 && dev < kMaxDevices;
    if (cached && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
    e = cudaFuncSetAttribute(attend_pages_decode_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && cached) done[dev].store(true, std::memory_order_release);
    return e;
}

int score_stride(int max_seq_len) { return std::max(16, (pages_of(max_seq_len) + 15) / 16 * 16); }

}  // namespace
}  // namespace msgl

using namespace msgl;

extern "C" {

int msgl_kv_page_bounds(const void* k_pool, int64_t num_slots, const int* page_table, int max_pages,
                        const int* seq_lens, const int* q_indptr, int num_reqs, int max_q_len,
                        int num_kv_heads, int head_dim, int page_size, void* bounds,
                        msgl_stream_t stream) {
    if (head_dim != kHd) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "kv_page_bounds: head_dim must be 128");
    if (page_size != kPage) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "kv_page_bounds: page_size must be 16");
    if (num_kv_heads <= 0 || num_reqs < 0 || max_q_len < 0 || max_pages <= 0 || max_pages > INT32_MAX / kPage ||
        num_slots <= 0 || num_slots % kPage || num_slots / kPage > INT32_MAX)
        return set_error(MSGL_ERR_INVALID_ARG, "kv_page_bounds: bad sizes");
    if (!q_indptr && max_q_len != 1)
        return set_error(MSGL_ERR_INVALID_ARG, "kv_page_bounds: max_q_len must be 1 without q_indptr");
    if (num_reqs == 0 || max_q_len == 0) return MSGL_OK;
    if (!k_pool || !page_table || !seq_lens || !bounds || !aligned16(k_pool) || !aligned16(bounds))
        return set_error(MSGL_ERR_INVALID_ARG, "kv_page_bounds: null or unaligned pointer");
    int* err = device_error_word();
    if (!err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    const int per = std::min<int64_t>((int64_t(max_q_len) + 14) / kPage + 1, max_pages);
    const int64_t total = int64_t(num_reqs) * per * num_kv_heads;
    const int64_t blocks = (total + kBoundWarps - 1) / kBoundWarps;
    if (blocks > INT32_MAX) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "kv_page_bounds: batch too large");
    launch_pdl(page_bounds_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kBoundWarps * 32), 0, stream,
               static_cast<const __nv_bfloat16*>(k_pool), static_cast<int>(num_slots / kPage), page_table,
               max_pages, seq_lens, q_indptr, max_q_len, num_kv_heads, per, total,
               static_cast<__nv_bfloat16*>(bounds), err);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

size_t msgl_select_pages_workspace_size(int total_q, int max_seq_len, int num_kv_heads) {
    if (total_q <= 0 || max_seq_len <= 0 || num_kv_heads <= 0 || pages_of(max_seq_len) > kMaxPagesPerReq) return 0;
    // never less for fewer rows or a shorter context: one allocation serves all calls below its own
    const int64_t row = int64_t(16) * num_kv_heads * score_stride(max_seq_len);
    return static_cast<size_t>(std::min(total_q * row, std::max(kSelectBytes, 16 * row)));
}

int msgl_select_pages(const void* q, const void* bounds, int64_t num_pages, const int* page_table,
                      int max_pages, const int* seq_lens, const int* q_indptr, int num_reqs,
                      int total_q, int max_q_len, int max_seq_len, int num_q_heads, int num_kv_heads,
                      int head_dim, int page_size, int top_pages, int sink_pages, int recent_pages,
                      int* page_ids, void* workspace, size_t workspace_bytes, msgl_stream_t stream) {
    int rc = check_heads(num_q_heads, num_kv_heads, head_dim, page_size);
    if (rc) return rc;
    if (num_reqs < 0 || total_q < 0 || max_q_len < 0 || max_seq_len < 0 || max_pages <= 0 || num_pages <= 0 ||
        num_pages > INT32_MAX)
        return set_error(MSGL_ERR_INVALID_ARG, "select_pages: bad sizes");
    if (!q_indptr && (max_q_len != 1 || total_q != num_reqs))
        return set_error(MSGL_ERR_INVALID_ARG, "select_pages: one query row per request without q_indptr");
    if (top_pages <= 0 || sink_pages < 0 || recent_pages < 1 || sink_pages > top_pages - recent_pages)
        return set_error(MSGL_ERR_INVALID_ARG, "select_pages: need recent_pages >= 1 and sink_pages + recent_pages <= top_pages");
    if (top_pages > kMaxTopPages) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "select_pages: top_pages > 1024");
    if (pages_of(max_seq_len) > max_pages)
        return set_error(MSGL_ERR_INVALID_ARG, "select_pages: max_seq_len exceeds page-table width");
    if (pages_of(max_seq_len) > kMaxPagesPerReq)
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "select_pages: max_seq_len > 524288");
    if (num_reqs == 0 || total_q == 0 || max_q_len == 0) return MSGL_OK;
    if (!q || !bounds || !page_table || !seq_lens || !page_ids || !aligned16(q) || !aligned16(bounds))
        return set_error(MSGL_ERR_INVALID_ARG, "select_pages: null or unaligned pointer");
    if (!workspace || !aligned16(workspace) ||
        workspace_bytes < msgl_select_pages_workspace_size(total_q, max_seq_len, num_kv_heads))
        return set_error(MSGL_ERR_WORKSPACE, "select_pages: workspace missing, unaligned or too small");
    SelectArgs a = {};
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.bounds = static_cast<const __nv_bfloat16*>(bounds);
    a.pool_pages = static_cast<int>(num_pages);
    a.page_table = page_table;
    a.max_pages = max_pages;
    a.seq_lens = seq_lens;
    a.q_indptr = q_indptr;
    a.num_reqs = num_reqs;
    a.total_q = total_q;
    a.max_q_len = max_q_len = std::min(max_q_len, total_q);  // no request can own more rows
    a.max_len = max_seq_len;
    a.hq = num_q_heads;
    a.hkv = num_kv_heads;
    a.top = top_pages;
    a.sink = sink_pages;
    a.recent = recent_pages;
    a.page_ids = page_ids;
    a.err = device_error_word();
    if (!a.err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    a.stride = score_stride(max_seq_len);
    const int slab = slab_rows(total_q, a.stride, num_kv_heads);
    a.wide = static_cast<unsigned long long*>(workspace);
    a.scores = reinterpret_cast<float*>(a.wide + int64_t(slab) * num_kv_heads * a.stride);
    a.mags = a.scores + int64_t(slab) * num_kv_heads * a.stride;

    const int G = num_q_heads / num_kv_heads;
    const bool chunk = max_q_len > 1;
    using Score = void (*)(SelectArgs, int, int, int);
    const Score score = chunk ? (G == 1   ? Score(page_scores_kernel<1, true>)
                                 : G == 2 ? Score(page_scores_kernel<2, true>)
                                 : G == 4 ? Score(page_scores_kernel<4, true>) : Score(page_scores_kernel<8, true>))
                              : (G == 1   ? Score(page_scores_kernel<1, false>)
                                 : G == 2 ? Score(page_scores_kernel<2, false>)
                                 : G == 4 ? Score(page_scores_kernel<4, false>) : Score(page_scores_kernel<8, false>));
    const int tile_rows = chunk ? kScoreCols / G : 1;
    const int tiles = (max_q_len + tile_rows - 1) / tile_rows;
    // Single tokens: a few groups of pages a warp, whose page ids are loaded a group ahead, as long as
    // some eight CTAs per SM are left.
    const int64_t heads = int64_t(num_reqs) * tiles * num_kv_heads;
    const int all_groups = (pages_of(max_seq_len) + kScorePages - 1) / kScorePages;
    int groups = 1;
    while (!chunk && groups < 8 && heads * all_groups >= 32 * 148 * groups) groups *= 2;
    const int page_tiles = (all_groups + groups - 1) / groups;
    const int64_t blocks = heads * page_tiles;
    const int64_t sel_blocks = int64_t(slab) * num_kv_heads;
    if (blocks > INT32_MAX || sel_blocks > INT32_MAX)
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "select_pages: batch too large");
    // Up to 1024 pages a warp holds a row; with too few rows to fill the GPU, and for longer
    // rows, more warps share one. Few warps that hold many scores beat many that hold few, whose
    // counts meet at a barrier in every step: 8192 pages, one request, 8 warps 27.0 us for
    // selection and attention, 16 warps 28.4; 2048 pages, 64 requests, 4 warps 170, 8 warps 172,
    // 16 warps 183. At 512 pages the order turns: 4 warps 14.7 us, 2 warps 15.0.
    using Select = void (*)(SelectArgs, int);
    const int pages = pages_of(max_seq_len);
    const bool many = sel_blocks >= 4 * 148;
    int warps, rows;  // per row, per CTA
    Select select;
    if (pages <= 256 && many) { select = select_pages_kernel<1, 8, 4>; warps = 1; rows = 4; }
    else if (pages <= 1024 && many) { select = select_pages_kernel<1, 32, 4>; warps = 1; rows = 4; }
    else if (pages <= 512) { select = select_pages_kernel<4, 4, 1>; warps = 4; rows = 1; }
    else if (pages <= 2048) { select = select_pages_kernel<4, 16, 1>; warps = 4; rows = 1; }
    else if (pages <= 8192) { select = select_pages_kernel<8, 32, 1>; warps = 8; rows = 1; }
    else { select = select_pages_kernel<32, 32, 1>; warps = 32; rows = 1; }
    for (int t0 = 0; t0 < total_q; t0 += slab) {
        a.t0 = t0;
        a.t1 = std::min(total_q, t0 + slab);
        if (page_tiles > 0 && pages_of(max_seq_len) > top_pages) {
            launch_pdl(score, dim3(static_cast<unsigned>(blocks)), dim3(kScoreWarps * 32), 0, stream, a,
                       tiles, page_tiles, groups);
            MSGL_LAUNCH_CHECK();
        }
        const int n = (a.t1 - t0) * num_kv_heads;
        launch_pdl(select, dim3((n + rows - 1) / rows), dim3(32 * warps * rows), 0, stream, a, n);
        MSGL_LAUNCH_CHECK();
    }
    return MSGL_OK;
}

int msgl_paged_attention_pages(const void* q, const void* k_pool, const void* v_pool,
                               int64_t num_slots, const int* page_table, int max_pages,
                               const int* seq_lens, const int* q_indptr, int num_reqs, int total_q,
                               int max_q_len, int max_seq_len, const int* page_ids, int top_pages,
                               int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                               float scale, void* out, msgl_stream_t stream) {
    int rc = check_heads(num_q_heads, num_kv_heads, head_dim, page_size);
    if (rc) return rc;
    if (num_reqs < 0 || total_q < 0 || max_q_len < 0 || max_seq_len < 0 || max_pages <= 0 || num_slots <= 0 ||
        num_slots % kPage || num_slots / kPage > INT32_MAX || top_pages <= 0)
        return set_error(MSGL_ERR_INVALID_ARG, "attention_pages: bad sizes");
    if (!q_indptr && (max_q_len != 1 || total_q != num_reqs))
        return set_error(MSGL_ERR_INVALID_ARG, "attention_pages: one query row per request without q_indptr");
    if (top_pages > kMaxTopPages) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "attention_pages: top_pages > 1024");
    if (pages_of(max_seq_len) > max_pages)
        return set_error(MSGL_ERR_INVALID_ARG, "attention_pages: max_seq_len exceeds page-table width");
    if (pages_of(max_seq_len) > kMaxPagesPerReq)
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "attention_pages: max_seq_len > 524288");
    if (num_reqs == 0 || total_q == 0 || max_q_len == 0) return MSGL_OK;
    if (!q || !k_pool || !v_pool || !page_table || !seq_lens || !page_ids || !out || !aligned16(q) ||
        !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out))
        return set_error(MSGL_ERR_INVALID_ARG, "attention_pages: null or unaligned pointer");
    AttArgs a = {};
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.k_pool = static_cast<const __nv_bfloat16*>(k_pool);
    a.v_pool = static_cast<const __nv_bfloat16*>(v_pool);
    a.pool_pages = static_cast<int>(num_slots / kPage);
    a.page_table = page_table;
    a.max_pages = max_pages;
    a.seq_lens = seq_lens;
    a.q_indptr = q_indptr;
    a.total_q = total_q;
    a.max_q_len = max_q_len = std::min(max_q_len, total_q);  // no request can own more rows
    a.max_len = max_seq_len;
    a.page_ids = page_ids;
    a.top = top_pages;
    a.hq = num_q_heads;
    a.hkv = num_kv_heads;
    a.sl2e = scale * 1.4426950408889634f;
    a.out = static_cast<__nv_bfloat16*>(out);
    a.err = device_error_word();
    if (!a.err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    const int G = num_q_heads / num_kv_heads;
    if (max_q_len > kRowsAlone && total_q > kTotalAlone) {
        CUtensorMap tk, tv;  // {dims, kv heads, token rows}: one page of one kv head a box, its rows padded
        const uint64_t row = uint64_t(num_kv_heads) * kHd * 2;
        rc = make_tmap_3d_bf16(&tk, k_pool, kHd, num_kv_heads, num_slots, kHd * 2, row, kPadRow / 2, 1, kPage, false);
        if (!rc) rc = make_tmap_3d_bf16(&tv, v_pool, kHd, num_kv_heads, num_slots, kHd * 2, row, kPadRow / 2, 1, kPage, false);
        if (rc) return rc;
        const int tq = 8 / G;
        const int row_groups = std::min(kChWarps, kTileRows / tq);
        const int tiles = (max_q_len + row_groups * tq - 1) / (row_groups * tq);
        const int64_t blocks = int64_t(num_reqs) * tiles * num_kv_heads;
        // tiles that hold rows: every request ends with a part of one
        const int64_t held = (total_q / (row_groups * tq) + (num_reqs + 1) / 2) * num_kv_heads;
        const int split = chunk_split(std::min(blocks, std::max<int64_t>(1, held)));
        if (blocks * split > INT32_MAX) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "attention_pages: batch too large");
        static std::atomic<int> optin[kMaxDevices];
        cudaError_t e = smem_optin(attend_pages_chunk_kernel, kChSmem, optin);
        if (e == cudaSuccess)
            e = launch_cluster(attend_pages_chunk_kernel, blocks * split, kChThreads, split,
                               kChSmem, stream, tk, tv, a, tiles, row_groups);
        if (e != cudaSuccess) return set_error(MSGL_ERR_CUDA, cudaGetErrorString(e));
        MSGL_LAUNCH_CHECK();
        return MSGL_OK;
    }
    const int words = pages_of(max_seq_len) / 32 + 1;
    const size_t smem = kDecRing + size_t(words) * 4 + size_t(top_pages) * 8;
    const int64_t lists = int64_t(total_q) * num_kv_heads;
    if (lists * 16 > INT32_MAX) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "attention_pages: batch too large");
    const int split = decode_split(lists, top_pages);
    static std::atomic<int> optin[kMaxDevices];
    cudaError_t e = smem_optin(attend_pages_decode_kernel, smem, optin);
    if (e == cudaSuccess && split > 8) e = large_clusters();
    if (e != cudaSuccess) return set_error(MSGL_ERR_CUDA, cudaGetErrorString(e));
    e = launch_cluster(attend_pages_decode_kernel, lists * split, kAttThreads, split, smem, stream, a, num_reqs, words);
    if (e != cudaSuccess) return set_error(MSGL_ERR_CUDA, cudaGetErrorString(e));
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

}  // extern "C"
