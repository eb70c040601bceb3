// lora.cu -- low-rank adapters of many requests at once beside a shared projection.
//
//  * msgl_lora_add      out[t] = y[t] + scale[a] * B[a] (A[a] x[t])      (bf16)
//  * msgl_lora_partial  part[t] = scale[a] * B[a] (A[a] x[t])            (fp32: one more split-K
//                       partial of the projection, summed by the kernel that follows it)
// with a = adapter_ids[r] of the request r that owns row t (none: the product is zero).
//
// Two launches. `shrink` computes h = A[a] x (rank values a row) as fp32 partials over K ranges;
// `expand` adds them, multiplies by B[a] and adds the result to y. Both are bound by what they
// stream (x and A; B, y and out), so operands go from global memory straight into MMA fragments
// as 8- or 16-byte pieces: the order of the products of a dot product is free, and the same piece
// of a lane is used on both operands. Token rows are the MMA's 16 rows; one token per request
// leaves 15 of them empty, which costs nothing while the weights are what is streamed.
//
// h is fp32: it enters the second product as a sum of bf16 terms (two terms, 2^-17 relative, for
// the bf16 result; three, 2^-25, for the fp32 partial), so it is not rounded to bf16.
#include <algorithm>

#include "common.cuh"

namespace msgl {
namespace {

constexpr int kLoraWarps = 4;
constexpr int kMaxSplits = 16;
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
    int splits, slice;  // K ranges of the shrink
    float* h;           // [splits][T][R]
    int tiles;          // row tiles per request
    int* err;
};

struct LoraTile {
    int adapter, t0, rows;  // first row of the tile and its row count
};

// Tile `tile` (of `per` rows) of request r. Rows outside [0, T) are never touched.
__device__ __forceinline__ LoraTile lora_tile(const LoraArgs& a, int r, int tile, int per, bool report) {
    LoraTile o;
    const int q0 = a.q_indptr ? a.q_indptr[r] : r;
    int qn = a.q_indptr ? a.q_indptr[r + 1] - q0 : 1;
    if (q0 < 0 || qn < 0 || qn > a.max_q_len || q0 + static_cast<int64_t>(qn) > a.T) {
        if (report) record_error(a.err, MSGL_ERR_BOUNDS, 811);
        qn = 0;
    }
    o.adapter = a.ids[r];
    if (o.adapter >= a.num_adapters) {
        if (report) record_error(a.err, MSGL_ERR_BOUNDS, 810);
        o.adapter = -1;
    }
    o.t0 = q0 + tile * per;
    o.rows = min(per, qn - tile * per);
    return o;
}

// NT: 8-rank tiles. SMALL: one 16-row tile per request, the four warps split the K range; else
// 64-row tiles, 16 rows a warp.
template <int NT, bool SMALL>
__global__ void __launch_bounds__(kLoraWarps * 32)
lora_shrink_kernel(const LoraArgs a) {
    __shared__ float red[SMALL ? kLoraWarps * 16 * NT * 8 : 1];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    int64_t id = blockIdx.x;
    const int s = static_cast<int>(id % a.splits);
    id /= a.splits;
    const int tile = static_cast<int>(id % a.tiles), r = static_cast<int>(id / a.tiles);
    const LoraTile lt = lora_tile(a, r, tile, SMALL ? 16 : 64, s == 0 && tile == 0 && threadIdx.x == 0);
    if (lt.rows <= 0 || lt.adapter < 0) return;
    const int row0 = SMALL ? 0 : warp * 16;
    int k_lo = s * a.slice, k_hi = min(a.K, k_lo + a.slice);
    if (SMALL) {
        const int part = a.slice / kLoraWarps;
        k_lo += warp * part;
        k_hi = min(k_hi, k_lo + part);
    }
    const bool live0 = row0 + g < lt.rows, live1 = row0 + g + 8 < lt.rows;
    const __nv_bfloat16* x0 = a.x + static_cast<int64_t>(lt.t0 + row0 + g) * a.ldx;
    const __nv_bfloat16* x1 = x0 + 8 * a.ldx;
    const __nv_bfloat16* wa = a.a + (static_cast<int64_t>(lt.adapter) * a.R + g) * a.K;
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    if (SMALL || row0 < lt.rows) {
#pragma unroll 4
        for (int k0 = k_lo; k0 < k_hi; k0 += 32) {
            const int k = k0 + 8 * c;
            const bool in = k < k_hi;
            const uint4 u0 = in && live0 ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
            const uint4 u1 = in && live1 ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const uint4 v = in && 8 * j < a.R
                                    ? *reinterpret_cast<const uint4*>(wa + static_cast<int64_t>(8 * j) * a.K + k)
                                    : zero;
                mma_bf16_16816(acc[j], u0.x, u1.x, u0.y, u1.y, v.x, v.y);
                mma_bf16_16816(acc[j], u0.z, u1.z, u0.w, u1.w, v.z, v.w);
            }
        }
    }
    float* h = a.h + (static_cast<int64_t>(s) * a.T + lt.t0) * a.R;
    if constexpr (!SMALL) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            if (8 * j >= a.R) break;
            float* dst = h + static_cast<int64_t>(row0 + g) * a.R + 8 * j + 2 * c;
            if (live0) *reinterpret_cast<float2*>(dst) = make_float2(acc[j][0], acc[j][1]);
            if (live1) *reinterpret_cast<float2*>(dst + 8 * a.R) = make_float2(acc[j][2], acc[j][3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float* p = red + (warp * 16 + g) * NT * 8 + 8 * j + 2 * c;
            p[0] = acc[j][0];
            p[1] = acc[j][1];
            p[8 * NT * 8] = acc[j][2];
            p[8 * NT * 8 + 1] = acc[j][3];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < lt.rows * NT * 8; i += kLoraWarps * 32) {
            const int row = i / (NT * 8), rank = i % (NT * 8);
            if (rank >= a.R) continue;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kLoraWarps; ++w) v += red[(w * 16 + row) * NT * 8 + rank];
            h[static_cast<int64_t>(row) * a.R + rank] = v;
        }
    }
}

// What a bf16 term leaves of v (exact); nothing where the term is infinite or NaN.
__device__ __forceinline__ float rest(float v, float term) {
    return fabsf(term) < __builtin_huge_valf() ? v - term : 0.f;
}

// KK: 16-rank steps. A warp's 16 rows times blocks of 32 output columns: MMA column tile j of a
// block holds columns 8 (n / 2) + 2 j + n % 2, so that lane (g, c) ends with the 8 consecutive
// columns 8 c .. 8 c + 7 of rows g and g + 8 (16-byte loads of y, 16-byte stores).
template <int KK, bool SMALL, bool PARTIAL>
__global__ void __launch_bounds__(kLoraWarps * 32)
lora_expand_kernel(const LoraArgs a, int n_slice, int n_slices) {
    constexpr int TERMS = PARTIAL ? 3 : 2;
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    int64_t id = blockIdx.x;
    const int ns = static_cast<int>(id % n_slices);
    id /= n_slices;
    const int tile = static_cast<int>(id % a.tiles), r = static_cast<int>(id / a.tiles);
    const LoraTile lt = lora_tile(a, r, tile, SMALL ? 16 : 64, false);
    const int row0 = SMALL ? 0 : warp * 16;
    if (lt.rows <= row0) return;
    int n_lo = ns * n_slice, n_hi = min(a.N, n_lo + n_slice);
    if (SMALL) {
        n_lo += warp * (n_slice / kLoraWarps);
        n_hi = min(n_hi, n_lo + n_slice / kLoraWarps);
    }
    const bool live[2] = {row0 + g < lt.rows, row0 + g + 8 < lt.rows};
    const int64_t t[2] = {lt.t0 + row0 + g, lt.t0 + row0 + g + 8};
    uint32_t ha[KK][TERMS][4];
    if (lt.adapter >= 0) {
        const float scale = a.scales[lt.adapter];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int rank = 16 * kk + 4 * c;
                float v[4] = {0.f, 0.f, 0.f, 0.f};
                if (live[u] && rank < a.R) {
                    const float* src = a.h + t[u] * a.R + rank;
                    for (int s = 0; s < a.splits; ++s) {
                        const float4 f = *reinterpret_cast<const float4*>(src + static_cast<int64_t>(s) * a.T * a.R);
                        v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] *= scale;
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
    const __nv_bfloat16* wb = a.b + static_cast<int64_t>(max(lt.adapter, 0)) * a.N * a.R;
    for (int n0 = n_lo; n0 < n_hi; n0 += 32) {
        const int col = n0 + 8 * c;
        const bool in = col < n_hi;
        uint4 yv[2];
        if (!PARTIAL) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                yv[u] = in && live[u] ? *reinterpret_cast<const uint4*>(a.y + t[u] * a.ldy + col)
                                      : make_uint4(0, 0, 0, 0);
        }
        float acc[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
        if (lt.adapter >= 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    const int rank = 16 * kk + 4 * c;
                    uint2 v = make_uint2(0, 0);
                    if (n < n_hi && rank < a.R)
                        v = *reinterpret_cast<const uint2*>(wb + static_cast<int64_t>(n) * a.R + rank);
#pragma unroll
                    for (int m = TERMS - 1; m >= 0; --m)
                        mma_bf16_16816(acc[j], ha[kk][m][0], ha[kk][m][1], ha[kk][m][2], ha[kk][m][3], v.x, v.y);
                }
            }
        }
        if (!in) continue;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (!live[u]) continue;
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[2 * j] = acc[j][2 * u];
                v[2 * j + 1] = acc[j][2 * u + 1];
            }
            if (PARTIAL) {
                float4* dst = reinterpret_cast<float4*>(static_cast<float*>(a.out) + t[u] * a.ldo + col);
                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                dst[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                uint4 o = yv[u];
                if (lt.adapter >= 0) {  // else y unchanged, bit for bit
                    o.x = pack_bf16x2(bf16lo(o.x) + v[0], bf16hi(o.x) + v[1]);
                    o.y = pack_bf16x2(bf16lo(o.y) + v[2], bf16hi(o.y) + v[3]);
                    o.z = pack_bf16x2(bf16lo(o.z) + v[4], bf16hi(o.z) + v[5]);
                    o.w = pack_bf16x2(bf16lo(o.w) + v[6], bf16hi(o.w) + v[7]);
                }
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + t[u] * a.ldo + col) = o;
            }
        }
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// K ranges that the workspace has room for: many for few rows, where one range per tile would
// leave most of the GPU without work.
int max_splits(int64_t T) { return T <= 1024 ? kMaxSplits : 8; }

template <int KK, bool PARTIAL>
auto expand_kernel(bool small) {
    return small ? lora_expand_kernel<KK, true, PARTIAL> : lora_expand_kernel<KK, false, PARTIAL>;
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
    if (!a.x || !a.ids || !a.out || (!partial && !a.y) || (a.num_adapters && (!a.a || !a.b || !a.scales)))
        return set_error(MSGL_ERR_INVALID_ARG, "lora: null pointer");
    if (!aligned16(a.x) || !aligned16(a.a) || !aligned16(a.b) || !aligned16(a.y) || !aligned16(a.out))
        return set_error(MSGL_ERR_INVALID_ARG, "lora: rows must be 16-byte aligned");
    if (!workspace || !aligned16(workspace) ||
        workspace_bytes < msgl_lora_workspace_size(a.T, a.K, a.R))
        return set_error(MSGL_ERR_WORKSPACE, "lora: workspace missing, unaligned or too small");
    a.err = device_error_word();
    if (!a.err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    a.h = static_cast<float*>(workspace);
    const bool small = a.max_q_len <= 16;
    a.tiles = small ? 1 : (a.max_q_len + 63) / 64;
    // about 4 CTAs per SM, ranges of at least 128 columns
    const int64_t rows = int64_t(num_reqs) * a.tiles;
    const int unit = small ? 128 : 32;
    int64_t s = std::min<int64_t>({(592 + rows - 1) / rows, (a.K + 127) / 128, max_splits(a.T)});
    a.slice = static_cast<int>(((a.K + s - 1) / s + unit - 1) / unit * unit);
    a.splits = (a.K + a.slice - 1) / a.slice;
    const int n_slice = small ? 512 : 256;
    const int n_slices = (a.N + n_slice - 1) / n_slice;
    if (rows * a.splits > INT32_MAX || rows * n_slices > INT32_MAX)
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "lora: batch too large");

    using Shrink = void (*)(LoraArgs);
    const int nt = a.R / 8;
    const Shrink shrink =
        nt <= 1 ? (small ? Shrink(lora_shrink_kernel<1, true>) : Shrink(lora_shrink_kernel<1, false>))
        : nt <= 2 ? (small ? Shrink(lora_shrink_kernel<2, true>) : Shrink(lora_shrink_kernel<2, false>))
        : nt <= 4 ? (small ? Shrink(lora_shrink_kernel<4, true>) : Shrink(lora_shrink_kernel<4, false>))
        : nt <= 8 ? (small ? Shrink(lora_shrink_kernel<8, true>) : Shrink(lora_shrink_kernel<8, false>))
                  : (small ? Shrink(lora_shrink_kernel<16, true>) : Shrink(lora_shrink_kernel<16, false>));
    launch_pdl(shrink, dim3(static_cast<unsigned>(rows * a.splits)), dim3(kLoraWarps * 32), 0, stream, a);
    MSGL_LAUNCH_CHECK();
    const int kk = (a.R + 15) / 16;
    const auto expand =
        kk <= 1 ? (partial ? expand_kernel<1, true>(small) : expand_kernel<1, false>(small))
        : kk <= 2 ? (partial ? expand_kernel<2, true>(small) : expand_kernel<2, false>(small))
        : kk <= 4 ? (partial ? expand_kernel<4, true>(small) : expand_kernel<4, false>(small))
                  : (partial ? expand_kernel<8, true>(small) : expand_kernel<8, false>(small));
    launch_pdl(expand, dim3(static_cast<unsigned>(rows * n_slices)), dim3(kLoraWarps * 32), 0, stream, a,
               n_slice, n_slices);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

}  // namespace
}  // namespace msgl

using namespace msgl;

extern "C" {

size_t msgl_lora_workspace_size(int num_tokens, int K, int rank) {
    if (num_tokens <= 0 || K <= 0 || rank <= 0 || rank > kMaxRank) return 0;
    return size_t(std::min<int64_t>(max_splits(num_tokens), (K + 127) / 128)) * num_tokens * rank * sizeof(float);
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
