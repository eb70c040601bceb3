// lora.cu -- low-rank adapters of many requests at once beside a shared projection.
//
//  * msgl_lora_add      out[t] = y[t] + scale[a] * B[a] (A[a] x[t])      (bf16)
//  * msgl_lora_partial  part[t] = scale[a] * B[a] (A[a] x[t])            (fp32: one more split-K
//                       partial of the projection, summed by the kernel that follows it)
// with a = adapter_ids[r] of the request r that owns row t (none: the product is zero).
//
// h = A[a] x has rank values a row; the second product multiplies it by B[a]. Both are bound by
// what they stream (x and A; B, y and out). The order of the products of a dot product is free, so
// operands go straight from global memory into MMA fragments as 8- or 16-byte pieces wherever a
// value is used once, the same piece of a lane on both operands.
//
//  * Up to 16 rows a request (decode): one launch, a cluster of CTAs per request or per adapter. Its warps
//    split K for the first product, its CTAs exchange their sums through distributed shared memory
//    and split N for the second. Token rows are the MMA's 16 rows; one token leaves 15 of them
//    empty, which costs nothing while the weights are what is streamed.
//  * Longer chunks: `shrink` writes h, `expand` reads it. Both take 64 rows of one request a CTA and
//    bring what several warps share (A, x, B, h) into shared memory.
//
// h is summed in fp32. For the fp32 partial it enters the second product as three bf16 terms (what is
// left of h: 2^-24 of it), for the bf16 result as two (2^-16). One term (2^-8 of each of the rank's h)
// is not enough: the result is off by as much of sum |B h|, which where those terms cancel, or cancel
// y, is far more than the rounding of the result itself. (4.5k rows, 4096 -> 6144, on the device: 43 us
// with one term and 50 with two at rank 64, 65 and 79 at rank 128, no difference at rank 16.) The terms
// behind the first take infinite and NaN weights as zero: what is left of an h that is a bf16 value is
// zero, and zero times an infinite weight would be NaN.
#include <algorithm>

#include "common.cuh"

namespace msgl {
namespace {

constexpr int kLoraWarps = 4;
constexpr int kMaxRank = 128;

struct LoraArgs {
    const __nv_bfloat16* x;
    int64_t ldx;
    const __nv_bfloat16 *a, *b;
    const float* scales;
    int num_adapters;
    const int *ids, *q_indptr;
    int max_q_len;
    const __nv_bfloat16* y;
    int64_t ldy;
    void* out;
    int64_t ldo;
    int T, N, K, R;
    __nv_bfloat16* h;  // workspace: h of long chunks
    int tiles;         // 64-row tiles per request
    int* err;
};

struct LoraTile {
    int adapter, t0, rows;  // first row of the tile and its row count
};

// Tile `tile` (of `per` rows) of request r. Rows outside [0, T) are never touched.
__device__ __forceinline__ LoraTile lora_tile(const LoraArgs& a, int r, int tile, int per, bool report) {
    LoraTile o;
    // from L2: `expand` reads these before its wait
    const int q0 = a.q_indptr ? __ldcg(a.q_indptr + r) : r;
    int qn = a.q_indptr ? __ldcg(a.q_indptr + r + 1) - q0 : 1;
    if (q0 < 0 || qn < 0 || qn > a.max_q_len || q0 + static_cast<int64_t>(qn) > a.T) {
        if (report) record_error(a.err, MSGL_ERR_BOUNDS, 811);
        qn = 0;
    }
    o.adapter = __ldcg(a.ids + r);
    if (o.adapter >= a.num_adapters) {
        if (report) record_error(a.err, MSGL_ERR_BOUNDS, 810);
        o.adapter = -1;
    }
    o.t0 = q0 + tile * per;
    o.rows = min(per, qn - tile * per);
    return o;
}

// What a bf16 term leaves of v (exact); nothing where the term is infinite or NaN.
__device__ __forceinline__ float rest(float v, float term) {
    return fabsf(term) < __builtin_huge_valf() ? v - term : 0.f;
}

// out[t, col .. col + 8) from the sums v of lane (g, c): y + v in bf16 (y itself without an adapter,
// bit for bit), or v in fp32.
template <bool PARTIAL>
__device__ __forceinline__ void put8(const LoraArgs& a, int64_t t, int col, const float (&v)[8], uint4 y, bool some) {
    if (PARTIAL) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(a.out) + t * a.ldo + col);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        if (some) {
            y.x = pack_bf16x2(bf16lo(y.x) + v[0], bf16hi(y.x) + v[1]);
            y.y = pack_bf16x2(bf16lo(y.y) + v[2], bf16hi(y.y) + v[3]);
            y.z = pack_bf16x2(bf16lo(y.z) + v[4], bf16hi(y.z) + v[5]);
            y.w = pack_bf16x2(bf16lo(y.w) + v[6], bf16hi(y.w) + v[7]);
        }
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + t * a.ldo + col) = y;
    }
}

// ------------------------------------------------------------------ up to 16 rows a request
// KK: 16-rank steps. Columns come in blocks of 32: MMA column tile j of a block holds columns
// 8 (n / 2) + 2 j + n % 2, so that lane (g, c) ends with the 8 consecutive columns 8 c .. 8 c + 7 of
// rows g and g + 8. B of the first PRE blocks of a warp is loaded before the exchange of h.
//
// GROUPED (one row per request): `per` clusters per adapter, which take the rows of all its requests
// 16 at a time; the rows without an adapter are dealt to all clusters. An adapter's weights are then
// read once per 16 rows, not once per request.
template <int KK, bool PARTIAL, bool GROUPED>
__global__ void __launch_bounds__(kLoraWarps * 32)
lora_small_kernel(const LoraArgs a, int num_reqs, int per) {
    constexpr int NT = 2 * KK, R16 = 16 * KK, TERMS = PARTIAL ? 3 : 2, PRE = KK == 1 ? 6 : KK == 2 ? 3 : 1;
    __shared__ __align__(16) float red[kLoraWarps * 16 * R16];  // a warp's sums; then h of the cluster
    __shared__ __align__(16) float part[16 * R16];              // this CTA's sums
    __shared__ int list[16], scan[32];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int C = static_cast<int>(cluster_nctarank()), rank_c = static_cast<int>(cluster_ctarank());
    const int id = static_cast<int>(blockIdx.x) / C;
    const bool report = rank_c == 0 && threadIdx.x == 0;

    // columns of this warp: blocks of 32, dealt in runs to the cluster's warps
    const int blocks = (a.N + 31) / 32, all = C * kLoraWarps, me = rank_c * kLoraWarps + warp;
    const int b_lo = static_cast<int>(static_cast<int64_t>(blocks) * me / all);
    const int b_hi = static_cast<int>(static_cast<int64_t>(blocks) * (me + 1) / all);
    uint2 bf[PRE][4][KK];
    int total = 0;  // rows of the adapter
    bool waiting = false;
    const int base0 = GROUPED ? id % per * 16 : 0;
    for (int base = base0; base == base0 || base < total; base += per * 16) {
        int adapter, rows;
        int64_t t[2];
        if (GROUPED) {
            adapter = id / per;
            total = 0;
            for (int r0 = 0; r0 < num_reqs; r0 += kLoraWarps * 32) {  // the requests of this adapter, in order
                const int r = r0 + threadIdx.x;
                const int own = r < num_reqs ? a.ids[r] : -1;
                if (own >= a.num_adapters && blockIdx.x == 0 && base == base0) record_error(a.err, MSGL_ERR_BOUNDS, 810);
                const int mine = own == adapter;
                int n;
                const int at = total + block_excl_scan(mine, scan, n) - base;
                if (mine && at >= 0 && at < 16) list[at] = r;
                total += n;
            }
            __syncthreads();
            rows = min(16, total - base);
            t[0] = g < rows ? list[g] : 0;
            t[1] = g + 8 < rows ? list[g + 8] : 0;
        } else {
            const LoraTile lt = lora_tile(a, id, 0, 16, report);
            adapter = lt.adapter;
            rows = lt.rows;
            t[0] = static_cast<int64_t>(lt.t0) + g;
            t[1] = t[0] + 8;
        }
        if (rows <= 0) break;  // the whole cluster
        const bool some = adapter >= 0;
        const bool live[2] = {g < rows, g + 8 < rows};
        const __nv_bfloat16* wb = a.b + static_cast<int64_t>(max(adapter, 0)) * a.N * a.R;
        const auto load_b = [&](int blk0) {
#pragma unroll
            for (int p = 0; p < PRE; ++p)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = (blk0 + p) * 32 + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
                    for (int kk = 0; kk < KK; ++kk) {
                        const int rank = 16 * kk + 4 * c;
                        bf[p][j][kk] = make_uint2(0, 0);
                        if (blk0 + p < b_hi && n < a.N && rank < a.R)
                            bf[p][j][kk] = *reinterpret_cast<const uint2*>(wb + static_cast<int64_t>(n) * a.R + rank);
                    }
                }
        };
        uint32_t ha[KK][TERMS][4];
        if (some) {
            load_b(b_lo);
            // ---- h = A x: this warp's range of K
            const int steps = (a.K + 31) / 32;
            const int k_lo = static_cast<int>(static_cast<int64_t>(steps) * me / all) * 32;
            const int k_hi = min(a.K, static_cast<int>(static_cast<int64_t>(steps) * (me + 1) / all) * 32);
            const __nv_bfloat16* x0 = a.x + t[0] * a.ldx;
            const __nv_bfloat16* x1 = a.x + t[1] * a.ldx;
            const __nv_bfloat16* wa = a.a + (static_cast<int64_t>(adapter) * a.R + g) * a.K;
            float acc[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
            const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll(KK <= 2 ? 4 : 1)
            for (int k0 = k_lo; k0 < k_hi; k0 += 32) {
                const int k = k0 + 8 * c;
                const bool in = k < k_hi;
                const uint4 u0 = in && live[0] ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
                const uint4 u1 = in && live[1] ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const uint4 v = in && 8 * j < a.R
                                        ? *reinterpret_cast<const uint4*>(wa + static_cast<int64_t>(8 * j) * a.K + k)
                                        : zero;
                    mma_bf16_16816(acc[j], u0.x, u1.x, u0.y, u1.y, v.x, v.y);
                    mma_bf16_16816(acc[j], u0.z, u1.z, u0.w, u1.w, v.z, v.w);
                }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float* p = red + (warp * 16 + g) * R16 + 8 * j + 2 * c;
                *reinterpret_cast<float2*>(p) = make_float2(acc[j][0], acc[j][1]);
                *reinterpret_cast<float2*>(p + 8 * R16) = make_float2(acc[j][2], acc[j][3]);
            }
            // the sums of the last 16 rows have been read by every CTA
            if (waiting) cluster_wait();
            __syncthreads();
            for (int i = threadIdx.x; i < rows * R16; i += kLoraWarps * 32) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < kLoraWarps; ++w) v += red[w * 16 * R16 + i];
                part[i] = v;
            }
            cluster_sync_all();
            const float scale = a.scales[adapter];
            for (int i = threadIdx.x; i < rows * R16; i += kLoraWarps * 32) {
                const uint32_t src = smem_u32(part + i);
                float v[8], sum = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = k < C ? ld_dsmem_f32(mapa_shared(src, k)) : 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) sum += v[k];  // in rank order
                red[i] = sum * scale;
            }
            cluster_arrive();  // waited for above or at the end
            waiting = true;
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (live[u] && 16 * kk + 4 * c < a.R)  // behind the rank: zero times x, NaN where that is infinite
                        f = *reinterpret_cast<const float4*>(red + (g + 8 * u) * R16 + 16 * kk + 4 * c);
                    float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                    for (int m = 0; m < TERMS; ++m) {
                        ha[kk][m][u] = pack_bf16x2(v[0], v[1]);
                        ha[kk][m][2 + u] = pack_bf16x2(v[2], v[3]);
                        v[0] = rest(v[0], bf16lo(ha[kk][m][u]));
                        v[1] = rest(v[1], bf16hi(ha[kk][m][u]));
                        v[2] = rest(v[2], bf16lo(ha[kk][m][2 + u]));
                        v[3] = rest(v[3], bf16hi(ha[kk][m][2 + u]));
                    }
                }
        }
        // ---- out = y + h B
        for (int blk0 = b_lo; blk0 < b_hi; blk0 += PRE) {
            if (some && blk0 > b_lo) load_b(blk0);
            uint4 yv[PRE][2];
            if (!PARTIAL) {
#pragma unroll
                for (int p = 0; p < PRE; ++p)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int col = (blk0 + p) * 32 + 8 * c;
                        yv[p][u] = blk0 + p < b_hi && col < a.N && live[u]
                                       ? *reinterpret_cast<const uint4*>(a.y + t[u] * a.ldy + col)
                                       : make_uint4(0, 0, 0, 0);
                    }
            }
#pragma unroll
            for (int p = 0; p < PRE; ++p) {
                if (blk0 + p >= b_hi) break;
                float acc[4][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
                if (some) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                            for (int m = TERMS - 1; m >= 0; --m)
                                mma_bf16_16816(acc[j], ha[kk][m][0], ha[kk][m][1], ha[kk][m][2], ha[kk][m][3],
                                               m ? finite2(bf[p][j][kk].x) : bf[p][j][kk].x,
                                               m ? finite2(bf[p][j][kk].y) : bf[p][j][kk].y);
                }
                const int col = (blk0 + p) * 32 + 8 * c;
                if (col >= a.N) continue;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (!live[u]) continue;
                    const float v[8] = {acc[0][2 * u], acc[0][2 * u + 1], acc[1][2 * u], acc[1][2 * u + 1],
                                        acc[2][2 * u], acc[2][2 * u + 1], acc[3][2 * u], acc[3][2 * u + 1]};
                    put8<PARTIAL>(a, t[u], col, v, PARTIAL ? make_uint4(0, 0, 0, 0) : yv[p][u], some);
                }
            }
        }
        if (!GROUPED) break;
        __syncthreads();  // list, red
    }
    if (GROUPED && (PARTIAL || a.out != a.y)) {  // this cluster's share of the rows without one
        for (int r = id; r < num_reqs; r += a.num_adapters * per) {
            const int own = a.ids[r];
            if (own >= 0 && own < a.num_adapters) continue;
            for (int col = (rank_c * kLoraWarps * 32 + threadIdx.x) * 8; col < a.N; col += C * kLoraWarps * 32 * 8) {
                const float none[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                const uint4 y = PARTIAL ? make_uint4(0, 0, 0, 0)
                                        : *reinterpret_cast<const uint4*>(a.y + static_cast<int64_t>(r) * a.ldy + col);
                put8<PARTIAL>(a, r, col, none, y, false);
            }
        }
    }
    if (waiting) cluster_wait();
}

// ------------------------------------------------------------------ chunks
constexpr int kTile = 64;     // rows a CTA
constexpr int kBK = 64;       // K columns a stage
constexpr int sh_stages(int kk) { return kk == 8 ? 4 : 5; }  // of 16 or 24 KB: two CTAs per SM
constexpr int kNSlice = 256;  // columns of an expand CTA

// h terms in the workspace: [term][T][R16] bf16, zero behind the rank (where the sums are zero times x,
// NaN where that is infinite).
__host__ __device__ constexpr int64_t h_terms(int64_t T, int r16, int term) { return term * T * r16; }

// A cluster of S CTAs (K ranges) per 64 rows; four warps of 16 rows times all ranks. x and A tiles
// of 64 columns (128-byte rows, 16-byte pieces swizzled by the row) go through a ring of cp.async
// stages; the S sums of a row are added through distributed shared memory, in rank order, scaled and
// written as bf16 terms.
template <int KK>
__global__ void __launch_bounds__(kLoraWarps * 32)
lora_shrink_kernel(const LoraArgs a, int terms) {
    constexpr int R16 = 16 * KK;
    constexpr int kStage = (kTile + R16) * kBK * 2, kShStages = sh_stages(KK);
    extern __shared__ __align__(128) uint8_t ring[];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int S = static_cast<int>(cluster_nctarank()), rank_c = static_cast<int>(cluster_ctarank());
    const int id = static_cast<int>(blockIdx.x) / S;
    const int tile = id % a.tiles, r = id / a.tiles;
    const LoraTile lt = lora_tile(a, r, tile, kTile, rank_c == 0 && tile == 0 && threadIdx.x == 0);
    if (lt.rows <= 0 || lt.adapter < 0) return;  // the whole cluster
    const int steps = (a.K + kBK - 1) / kBK;
    const int s_lo = static_cast<int>(static_cast<int64_t>(steps) * rank_c / S);
    const int s_n = static_cast<int>(static_cast<int64_t>(steps) * (rank_c + 1) / S) - s_lo;
    const __nv_bfloat16* wa = a.a + static_cast<int64_t>(lt.adapter) * a.R * a.K;
    const float scale = a.scales[lt.adapter];
    const auto issue = [&](int i) {
        const uint32_t dst = smem_u32(ring) + (i % kShStages) * kStage;
        const int k0 = (s_lo + i) * kBK;
#pragma unroll
        for (int p = threadIdx.x; p < (kTile + R16) * 8; p += kLoraWarps * 32) {
            const int row = p >> 3, k = k0 + (p & 7) * 8;
            const uint32_t d = dst + row * 128 + (((p & 7) ^ (row & 7)) << 4);
            if (row < kTile) {
                const bool in = row < lt.rows && k < a.K;
                cp_async16(d, a.x + (in ? static_cast<int64_t>(lt.t0 + row) * a.ldx + k : 0), in);
            } else {
                const bool in = row - kTile < a.R && k < a.K;
                cp_async16(d, wa + (in ? static_cast<int64_t>(row - kTile) * a.K + k : 0), in);
            }
        }
    };
    float acc[2 * KK][4];
#pragma unroll
    for (int j = 0; j < 2 * KK; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    for (int i = 0; i < kShStages - 1; ++i) {
        if (i < s_n) issue(i);
        cp_async_commit();
    }
    const int mi = lane >> 3, l7 = lane & 7;
    for (int i = 0; i < s_n; ++i) {
        cp_async_wait<kShStages - 2>();
        __syncthreads();
        if (i + kShStages - 1 < s_n) issue(i + kShStages - 1);
        cp_async_commit();
        const uint32_t xs = smem_u32(ring) + (i % kShStages) * kStage, as = xs + kTile * 128;
#pragma unroll
        for (int k = 0; k < kBK / 16; ++k) {
            const int xr = warp * 16 + (mi & 1) * 8 + l7;
            uint32_t x0, x1, x2, x3;
            ldsm_x4(xs + xr * 128 + (((2 * k + (mi >> 1)) ^ (xr & 7)) << 4), x0, x1, x2, x3);
#pragma unroll
            for (int j = 0; j < KK; ++j) {
                const int ar = 16 * j + (mi >> 1) * 8 + l7;
                uint32_t b0, b1, b2, b3;
                ldsm_x4(as + ar * 128 + (((2 * k + (mi & 1)) ^ (ar & 7)) << 4), b0, b1, b2, b3);
                mma_bf16_16816(acc[2 * j], x0, x1, x2, x3, b0, b1);
                mma_bf16_16816(acc[2 * j + 1], x0, x1, x2, x3, b2, b3);
            }
        }
    }
    cp_async_wait<0>();
    __syncthreads();
    float* sums = reinterpret_cast<float*>(ring);  // [64][R16]
#pragma unroll
    for (int j = 0; j < 2 * KK; ++j) {
        float* p = sums + (warp * 16 + g) * R16 + 8 * j + 2 * c;
        *reinterpret_cast<float2*>(p) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(p + 8 * R16) = make_float2(acc[j][2], acc[j][3]);
    }
    cluster_sync_all();
    for (int i = rank_c + S * static_cast<int>(threadIdx.x); i < lt.rows * R16 / 4; i += S * kLoraWarps * 32) {
        const uint32_t src = smem_u32(sums + 4 * i);
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = 0; k < S; ++k) {
            const float4 f = ld_dsmem_v4(mapa_shared(src, k));
            v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = 4 * i % R16 < a.R ? v[e] * scale : 0.f;
        __nv_bfloat16* dst = a.h + static_cast<int64_t>(lt.t0) * R16 + 4 * i;
        for (int m = 0; m < terms; ++m) {
            const uint2 u = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
            *reinterpret_cast<uint2*>(dst + h_terms(a.T, R16, m)) = u;
            v[0] = rest(v[0], bf16lo(u.x)); v[1] = rest(v[1], bf16hi(u.x));
            v[2] = rest(v[2], bf16lo(u.y)); v[3] = rest(v[3], bf16hi(u.y));
        }
    }
    cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

// One CTA per 64 rows and 256 columns; four warps of 32 rows x 128 columns, in blocks of 32 columns
// whose MMA column tiles interleave as in lora_small_kernel. B (rows of R16, its rows of a column
// tile next to each other) and the first block of y are loaded before the wait for the previous kernel:
// every kernel before `shrink` has completed once `shrink` runs. h comes behind it.
template <int KK, bool PARTIAL>
__global__ void __launch_bounds__(kLoraWarps * 32, KK == 8 ? 3 : 4)
lora_expand_kernel(const LoraArgs a, int n_slices) {
    constexpr int R16 = 16 * KK, PIECES = 2 * KK, TERMS = PARTIAL ? 3 : 2;
    constexpr int kSwz = KK == 1 ? 2 : KK == 2 ? 1 : 0, kMask = (PIECES < 8 ? PIECES : 8) - 1;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t bs = smem_u32(smem), hs = bs + kNSlice * R16 * 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    int64_t id = blockIdx.x;
    const int ns = static_cast<int>(id % n_slices);
    id /= n_slices;
    const int tile = static_cast<int>(id % a.tiles), r = static_cast<int>(id / a.tiles);
    const LoraTile lt = lora_tile(a, r, tile, kTile, false);
    if (lt.rows <= 0) {
        pdl_wait();  // no grid may end before its predecessor
        return;
    }
    const bool some = lt.adapter >= 0;
    const int n0 = ns * kNSlice;
    const auto swizzle = [](int row, int piece) {
        return static_cast<uint32_t>(row * R16 * 2 + ((piece ^ ((row >> kSwz) & kMask)) << 4));
    };
    if (some) {
        const __nv_bfloat16* wb = a.b + static_cast<int64_t>(lt.adapter) * a.N * a.R;
        for (int p = threadIdx.x; p < kNSlice * PIECES; p += kLoraWarps * 32) {
            const int n = p / PIECES, piece = p % PIECES;
            const int row = (n & ~31) + ((n & 7) >> 1) * 8 + ((n >> 3) & 3) * 2 + (n & 1);
            const bool in = n0 + n < a.N && piece * 8 < a.R;
            cp_async16(bs + swizzle(row, piece), wb + (in ? static_cast<int64_t>(n0 + n) * a.R + piece * 8 : 0), in);
        }
    }
    const int row0 = (warp & 1) * 32, blk0 = (warp >> 1) * 4;
    bool live[2][2];
    int64_t t[2][2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = row0 + mt * 16 + g + 8 * u;
            live[mt][u] = row < lt.rows;
            t[mt][u] = static_cast<int64_t>(lt.t0) + row;
        }
    uint4 yv[2][2][2];  // two blocks in flight
    const auto load_y = [&](int b) {
        const int col = n0 + (blk0 + b) * 32 + 8 * c;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                yv[b & 1][mt][u] = live[mt][u] && col < a.N
                                       ? *reinterpret_cast<const uint4*>(a.y + t[mt][u] * a.ldy + col)
                                       : make_uint4(0, 0, 0, 0);
    };
    if (!PARTIAL) load_y(0);
    pdl_wait();
    pdl_trigger();
    if (!PARTIAL && !some && a.out == a.y) return;  // in place: nothing to add
    if (some) {
#pragma unroll
        for (int m = 0; m < TERMS; ++m)
            for (int p = threadIdx.x; p < kTile * PIECES; p += kLoraWarps * 32) {
                const int row = p / PIECES, piece = p % PIECES;
                const bool in = row < lt.rows;
                cp_async16(hs + m * kTile * R16 * 2 + swizzle(row, piece),
                           a.h + h_terms(a.T, R16, m) + (in ? static_cast<int64_t>(lt.t0 + row) * R16 + piece * 8 : 0), in);
            }
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    const int mi = lane >> 3, l7 = lane & 7;
    constexpr bool kHold = !PARTIAL && KK <= 2;  // h in registers; of 64 ranks that leaves three CTAs an SM: 50 -> 52 us
    uint32_t hf[kHold ? KK : 1][TERMS][2][4];
    const auto load_h = [&](int kk, uint32_t (&f)[TERMS][2][4]) {
#pragma unroll
        for (int m = 0; m < TERMS; ++m)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const int row = row0 + mt * 16 + (mi & 1) * 8 + l7;
                ldsm_x4(hs + m * kTile * R16 * 2 + swizzle(row, 2 * kk + (mi >> 1)), f[m][mt][0], f[m][mt][1],
                        f[m][mt][2], f[m][mt][3]);
            }
    };
    if (kHold && some) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) load_h(kk, hf[kHold ? kk : 0]);
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        if (!PARTIAL && b < 3) load_y(b + 1);
        float acc[2][4][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[mt][j][0] = acc[mt][j][1] = acc[mt][j][2] = acc[mt][j][3] = 0.f;
        if (some) {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                uint32_t w[4][2];
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    const int row = (blk0 + b) * 32 + (j + (mi >> 1)) * 8 + l7;
                    ldsm_x4(bs + swizzle(row, 2 * kk + (mi & 1)), w[j][0], w[j][1], w[j + 1][0], w[j + 1][1]);
                }
                if (!kHold) load_h(kk, hf[0]);
                const auto& f = hf[kHold ? kk : 0];
                uint32_t wf[4][2];
#pragma unroll
                for (int j = 0; j < 4; ++j) wf[j][0] = finite2(w[j][0]), wf[j][1] = finite2(w[j][1]);
#pragma unroll
                for (int m = TERMS - 1; m >= 0; --m)
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            mma_bf16_16816(acc[mt][j], f[m][mt][0], f[m][mt][1], f[m][mt][2], f[m][mt][3],
                                           m ? wf[j][0] : w[j][0], m ? wf[j][1] : w[j][1]);
            }
        }
        const int col = n0 + (blk0 + b) * 32 + 8 * c;
        if (col >= a.N) continue;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (!live[mt][u]) continue;
                const float v[8] = {acc[mt][0][2 * u], acc[mt][0][2 * u + 1], acc[mt][1][2 * u], acc[mt][1][2 * u + 1],
                                    acc[mt][2][2 * u], acc[mt][2][2 * u + 1], acc[mt][3][2 * u], acc[mt][3][2 * u + 1]};
                put8<PARTIAL>(a, t[mt][u], col, v, PARTIAL ? make_uint4(0, 0, 0, 0) : yv[b & 1][mt][u], some);
            }
    }
}

int rank16(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

template <int KK, bool PARTIAL>
cudaError_t launch_chunks(const LoraArgs& a, int64_t row_tiles, int splits, cudaStream_t stream) {
    static std::atomic<int> optin[2][kMaxDevices];
    const size_t sh = size_t(sh_stages(KK)) * (kTile + 16 * KK) * kBK * 2;
    cudaError_t e = smem_optin(lora_shrink_kernel<KK>, sh, optin[0]);
    if (e != cudaSuccess) return e;
    const size_t ex = size_t(kNSlice + (PARTIAL ? 3 : 2) * kTile) * 16 * KK * 2;
    e = smem_optin(lora_expand_kernel<KK, PARTIAL>, ex, optin[1]);
    if (e != cudaSuccess) return e;
    e = launch_cluster(lora_shrink_kernel<KK>, row_tiles * splits, kLoraWarps * 32, splits, sh, stream, a, PARTIAL ? 3 : 2);
    if (e != cudaSuccess) return e;
    const int n_slices = (a.N + kNSlice - 1) / kNSlice;
    return launch_pdl(lora_expand_kernel<KK, PARTIAL>, dim3(static_cast<unsigned>(row_tiles * n_slices)),
                      dim3(kLoraWarps * 32), ex, stream, a, n_slices);
}

template <int KK>
cudaError_t launch_rank(const LoraArgs& a, int num_reqs, bool partial, cudaStream_t stream) {
    if (a.max_q_len <= 16) {
        // Clusters per adapter where that is fewer of them than one per request; CTAs of a cluster: up
        // to the portable size while about three per SM hold them.
        const bool grouped = !a.q_indptr && a.num_adapters > 0 && a.num_adapters < num_reqs;
        int64_t clusters = grouped ? a.num_adapters : num_reqs;
        int size = 8, per = 1;
        while (size > 2 && clusters * size > 3 * 148) size /= 2;
        if (grouped) {
            per = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(3 * 148 / (clusters * size), (num_reqs + 15) / 16)));
            clusters *= per;
        }
        const auto kern = partial ? (grouped ? lora_small_kernel<KK, true, true> : lora_small_kernel<KK, true, false>)
                                  : (grouped ? lora_small_kernel<KK, false, true> : lora_small_kernel<KK, false, false>);
        return launch_cluster(kern, clusters * size, kLoraWarps * 32, size, 0, stream, a, num_reqs, per);
    }
    // K ranges: about three CTAs per SM, ranges of at least 256 columns
    const int64_t row_tiles = int64_t(num_reqs) * a.tiles;
    int splits = 1;
    while (splits < 8 && row_tiles * splits * 2 <= 3 * 148 && a.K >= 512 * splits) splits *= 2;
    return partial ? launch_chunks<KK, true>(a, row_tiles, splits, stream)
                   : launch_chunks<KK, false>(a, row_tiles, splits, stream);
}

int launch_lora(LoraArgs a, int num_reqs, bool partial, void* workspace, size_t workspace_bytes,
                msgl_stream_t stream) {
    if (a.T < 0 || a.N <= 0 || a.K <= 0 || a.R <= 0 || a.num_adapters < 0 || num_reqs < 0 || a.max_q_len < 0)
        return set_error(MSGL_ERR_INVALID_ARG, "lora: bad sizes");
    if (a.K % 8 || a.N % 8 || a.R % 8 || a.R > kMaxRank)
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "lora: K, N and rank must be multiples of 8, rank <= 128");
    if (!a.q_indptr && (a.max_q_len != 1 || num_reqs != a.T))
        return set_error(MSGL_ERR_INVALID_ARG, "lora: one row per request without q_indptr");
    if (a.T == 0 || num_reqs == 0 || a.max_q_len == 0) return MSGL_OK;
    const int64_t ow = partial ? 4 : 8;  // elements per 16 bytes of out
    if (a.ldx < a.K || a.ldx % 8 || a.ldo < a.N || a.ldo % ow || (!partial && (a.ldy < a.N || a.ldy % 8)))
        return set_error(MSGL_ERR_INVALID_ARG, "lora: row strides must cover the row and keep it 16-byte aligned");
    if (!partial && a.out == a.y && a.ldo != a.ldy)
        return set_error(MSGL_ERR_INVALID_ARG, "lora: out in place of y needs y's row stride");
    if (!a.x || !a.ids || !a.out || (!partial && !a.y) || (a.num_adapters && (!a.a || !a.b || !a.scales)))
        return set_error(MSGL_ERR_INVALID_ARG, "lora: null pointer");
    if (!aligned16(a.x) || !aligned16(a.a) || !aligned16(a.b) || !aligned16(a.y) || !aligned16(a.out))
        return set_error(MSGL_ERR_INVALID_ARG, "lora: rows must be 16-byte aligned");
    if (!workspace || !aligned16(workspace) ||
        workspace_bytes < msgl_lora_workspace_size(a.T, a.K, a.R))
        return set_error(MSGL_ERR_WORKSPACE, "lora: workspace missing, unaligned or too small");
    a.err = device_error_word();
    if (!a.err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    a.max_q_len = std::min(a.max_q_len, a.T);  // no request can own more rows
    a.h = static_cast<__nv_bfloat16*>(workspace);
    a.tiles = (a.max_q_len + kTile - 1) / kTile;
    if (int64_t(num_reqs) * a.tiles * std::max(8, (a.N + kNSlice - 1) / kNSlice) > INT32_MAX)
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "lora: batch too large");
    const int r16 = rank16(a.R);
    const cudaError_t e = r16 == 16   ? launch_rank<1>(a, num_reqs, partial, stream)
                          : r16 == 32 ? launch_rank<2>(a, num_reqs, partial, stream)
                          : r16 == 64 ? launch_rank<4>(a, num_reqs, partial, stream)
                                      : launch_rank<8>(a, num_reqs, partial, stream);
    if (e != cudaSuccess) return set_error(MSGL_ERR_CUDA, cudaGetErrorString(e));
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

}  // namespace
}  // namespace msgl

using namespace msgl;

extern "C" {

size_t msgl_lora_workspace_size(int num_tokens, int K, int rank) {
    if (num_tokens <= 0 || K <= 0 || rank <= 0 || rank > kMaxRank) return 0;
    return size_t(3) * num_tokens * rank16(rank) * sizeof(__nv_bfloat16);
}

int msgl_lora_add(const void* x, int64_t ldx, const void* lora_a, const void* lora_b,
                  const float* scales, int num_adapters, const int* adapter_ids,
                  const int* q_indptr, int num_reqs, int max_q_len, const void* y, int64_t ldy,
                  void* out, int64_t ldo, int num_tokens, int N, int K, int rank, void* workspace,
                  size_t workspace_bytes, msgl_stream_t stream) {
    LoraArgs a = {};
    a.x = static_cast<const __nv_bfloat16*>(x);
    a.ldx = ldx;
    a.a = static_cast<const __nv_bfloat16*>(lora_a);
    a.b = static_cast<const __nv_bfloat16*>(lora_b);
    a.scales = scales;
    a.num_adapters = num_adapters;
    a.ids = adapter_ids;
    a.q_indptr = q_indptr;
    a.max_q_len = max_q_len;
    a.y = static_cast<const __nv_bfloat16*>(y);
    a.ldy = ldy;
    a.out = out;
    a.ldo = ldo;
    a.T = num_tokens;
    a.N = N;
    a.K = K;
    a.R = rank;
    return launch_lora(a, num_reqs, false, workspace, workspace_bytes, stream);
}

int msgl_lora_partial(const void* x, int64_t ldx, const void* lora_a, const void* lora_b,
                      const float* scales, int num_adapters, const int* adapter_ids,
                      const int* q_indptr, int num_reqs, int max_q_len, float* part, int64_t ldp,
                      int num_tokens, int N, int K, int rank, void* workspace,
                      size_t workspace_bytes, msgl_stream_t stream) {
    LoraArgs a = {};
    a.x = static_cast<const __nv_bfloat16*>(x);
    a.ldx = ldx;
    a.a = static_cast<const __nv_bfloat16*>(lora_a);
    a.b = static_cast<const __nv_bfloat16*>(lora_b);
    a.scales = scales;
    a.num_adapters = num_adapters;
    a.ids = adapter_ids;
    a.q_indptr = q_indptr;
    a.max_q_len = max_q_len;
    a.out = part;
    a.ldo = ldp;
    a.T = num_tokens;
    a.N = N;
    a.K = K;
    a.R = rank;
    return launch_lora(a, num_reqs, true, workspace, workspace_bytes, stream);
}

}  // extern "C"
