// mrope.cu -- QK-norm + rotary positions of three axes + KV page store, one pass.
//
//  * msgl_qknorm_mrope_store_kv            bf16 QKV rows
//  * msgl_qknorm_mrope_store_kv_partials   the rows as fp32 split-K partials
//
// Per token and query / key head of 128: y = x / sqrt(mean(x^2) + eps) * w, then the rotate-half
// pair (d, d + 64) is turned by the table angle of position[axis(d)]: a token of an image or a
// video has one position per axis (0 time, 1 height, 2 width), and every rotary pair follows one
// of them. Values are copied. With equal positions on all axes this is the one-axis rotation of
// msgl_qknorm_rope_store_kv.
#include "common.cuh"

namespace msgl {
namespace {

constexpr int kHd = 128;
constexpr int kHalf = kHd / 2;
constexpr int kMropeWarps = 4;

struct MropeArgs {
    const __nv_bfloat16* qkv;
    const float* parts;
    int nparts;
    __nv_bfloat16 *q_out, *k_pool, *v_pool;
    int64_t num_slots;
    const int* positions;
    int64_t pos_stride;
    int s0, s1, s2, layout;
    const int* slots;
    const float* table;
    int max_position;
    const __nv_bfloat16 *qn, *kn;
    int num_tokens, hq, hkv;
    float eps;
    int* err;
};

__device__ __forceinline__ int axis_of_pair(int d, const MropeArgs& a) {
    if (a.layout == MSGL_MROPE_INTERLEAVED) {
        const int m = d % 3;
        return m == 1 && d < 3 * a.s1 ? 1 : m == 2 && d < 3 * a.s2 ? 2 : 0;
    }
    return d < a.s0 ? 0 : d < a.s0 + a.s1 ? 1 : 2;
}

// Eight lanes per head, four heads per warp: lane i of a head owns elements [8 i, 8 i + 8) of the
// first half and their rotate-half partners, so loads and stores are 16 bytes (32 for partials)
// and the sum of squares takes three shuffles. The token's 64 cosines and sines are gathered once
// per CTA into shared memory, one element per thread, behind the loads of the IT groups of heads that
// a warp takes. grid (tokens, head splits).
template <bool PARTS, int IT>
__global__ void __launch_bounds__(kMropeWarps * 32)
qknorm_mrope_store_kernel(const MropeArgs a) {
    __shared__ __align__(16) float cs[kHd];  // cos 0..63, sin 0..63
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int i = lane & 7;
    const int nh = a.hq + 2 * a.hkv;
    const int h0 = (blockIdx.y * IT * kMropeWarps + warp) * 4 + (lane >> 3);  // then every 16th head
    int pos = a.positions[axis_of_pair(threadIdx.x & (kHalf - 1), a) * a.pos_stride + t];
    const int64_t slot = a.slots[t];
    uint4 u[PARTS ? 1 : IT][2];
    if (!PARTS) {
#pragma unroll
        for (int n = 0; n < IT; ++n) {
            const int h = h0 + n * kMropeWarps * 4;
            const __nv_bfloat16* src = a.qkv + (static_cast<int64_t>(t) * nh + h) * kHd + 8 * i;
#pragma unroll
            for (int v = 0; v < 2; ++v)
                u[n][v] = h < nh ? *reinterpret_cast<const uint4*>(src + v * kHalf) : make_uint4(0, 0, 0, 0);
        }
    }
    if (static_cast<unsigned>(pos) >= static_cast<unsigned>(a.max_position)) {
        record_error(a.err, MSGL_ERR_BOUNDS, 102);
        pos = 0;
    }
    cs[threadIdx.x] = a.table[static_cast<int64_t>(pos) * kHd + threadIdx.x];
    if (slot >= a.num_slots && threadIdx.x == 0 && blockIdx.y == 0) record_error(a.err, MSGL_ERR_BOUNDS, 103);
    const bool store = slot >= 0 && slot < a.num_slots;
    if (!PARTS) __syncthreads();
#pragma unroll
    for (int n = 0; n < IT; ++n) {
        const int h = h0 + n * kMropeWarps * 4;
        const bool live = h < nh;
        float x[16];  // elements 8 i + e (e < 8) and 64 + 8 i + (e - 8)
        if (PARTS) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = 0.f;
            if (live) {
                const int64_t stride = static_cast<int64_t>(a.num_tokens) * nh * kHd;
                const float* src = a.parts + (static_cast<int64_t>(t) * nh + h) * kHd + 8 * i;
                int p = 0;
                for (; p < a.nparts; p += 3) {  // three parts' loads in flight, added in part order
                    float4 f[3][4];
#pragma unroll
                    for (int q = 0; q < 3; ++q)
#pragma unroll
                        for (int v = 0; v < 4; ++v)
                            f[q][v] = p + q < a.nparts ? *reinterpret_cast<const float4*>(src + (p + q) * stride + (v >> 1) * kHalf + (v & 1) * 4)
                                                       : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int q = 0; q < 3; ++q) {
                        if (p + q >= a.nparts) break;
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            x[4 * v] += f[q][v].x; x[4 * v + 1] += f[q][v].y;
                            x[4 * v + 2] += f[q][v].z; x[4 * v + 3] += f[q][v].w;
                        }
                    }
                }
            }
            if (n == 0) __syncthreads();
        } else {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const uint32_t w[4] = {u[n][v].x, u[n][v].y, u[n][v].z, u[n][v].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[8 * v + 2 * e] = bf16lo(w[e]);
                    x[8 * v + 2 * e + 1] = bf16hi(w[e]);
                }
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) ss += x[e] * x[e];
        ss += __shfl_xor_sync(0xffffffffu, ss, 1);
        ss += __shfl_xor_sync(0xffffffffu, ss, 2);
        ss += __shfl_xor_sync(0xffffffffu, ss, 4);
        __nv_bfloat16* dst = nullptr;
        if (h < a.hq + a.hkv) {
            const float inv = 1.0f / sqrtf(ss / kHd + a.eps);
            const __nv_bfloat16* w = (h < a.hq ? a.qn : a.kn) + 8 * i;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const uint4 uw = *reinterpret_cast<const uint4*>(w + v * kHalf);
                const uint32_t ww[4] = {uw.x, uw.y, uw.z, uw.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[8 * v + 2 * e] *= inv * bf16lo(ww[e]);
                    x[8 * v + 2 * e + 1] *= inv * bf16hi(ww[e]);
                }
            }
            float cv[8], sv[8];
            *reinterpret_cast<float4*>(cv) = *reinterpret_cast<const float4*>(cs + 8 * i);
            *reinterpret_cast<float4*>(cv + 4) = *reinterpret_cast<const float4*>(cs + 8 * i + 4);
            *reinterpret_cast<float4*>(sv) = *reinterpret_cast<const float4*>(cs + kHalf + 8 * i);
            *reinterpret_cast<float4*>(sv + 4) = *reinterpret_cast<const float4*>(cs + kHalf + 8 * i + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float lo = x[e], hi = x[8 + e];
                x[e] = lo * cv[e] - hi * sv[e];
                x[8 + e] = lo * sv[e] + hi * cv[e];
            }
            if (h < a.hq) dst = a.q_out + (static_cast<int64_t>(t) * a.hq + h) * kHd;
            else if (store) dst = a.k_pool + (slot * a.hkv + (h - a.hq)) * kHd;
        } else if (live && store) {
            dst = a.v_pool + (slot * a.hkv + (h - a.hq - a.hkv)) * kHd;
        }
        if (!dst) continue;
#pragma unroll
        for (int v = 0; v < 2; ++v)
            *reinterpret_cast<uint4*>(dst + v * kHalf + 8 * i) =
                make_uint4(pack_bf16x2(x[8 * v], x[8 * v + 1]), pack_bf16x2(x[8 * v + 2], x[8 * v + 3]),
                           pack_bf16x2(x[8 * v + 4], x[8 * v + 5]), pack_bf16x2(x[8 * v + 6], x[8 * v + 7]));
    }
}

int launch_mrope(MropeArgs a, const int* sections, int layout, int head_dim, msgl_stream_t stream) {
    if (head_dim != kHd) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "qknorm_mrope: head_dim != 128");
    if (a.num_tokens < 0 || a.hq <= 0 || a.hkv <= 0 || a.max_position <= 0 || a.num_slots < 0 || !sections)
        return set_error(MSGL_ERR_INVALID_ARG, "qknorm_mrope: bad sizes");
    const int s0 = sections[0], s1 = sections[1], s2 = sections[2];
    if (s0 < 0 || s1 < 0 || s2 < 0 || s0 > kHalf || s1 > kHalf || s2 > kHalf || s0 + s1 + s2 != kHalf)
        return set_error(MSGL_ERR_INVALID_ARG, "qknorm_mrope: sections must be >= 0 and sum to head_dim / 2");
    if (layout != MSGL_MROPE_SECTIONS && layout != MSGL_MROPE_INTERLEAVED)
        return set_error(MSGL_ERR_INVALID_ARG, "qknorm_mrope: unknown layout");
    if (layout == MSGL_MROPE_INTERLEAVED && (s1 > kHalf / 3 || s2 > kHalf / 3))
        return set_error(MSGL_ERR_INVALID_ARG, "qknorm_mrope: interleaved height / width sections are at most 21 pairs");
    if (a.num_tokens == 0) return MSGL_OK;
    if (a.pos_stride != 0 && a.pos_stride < a.num_tokens)
        return set_error(MSGL_ERR_INVALID_ARG, "qknorm_mrope: position_stride must be 0 or >= num_tokens");
    if ((!a.qkv && !a.parts) || !a.q_out || !a.k_pool || !a.v_pool || !a.positions || !a.slots ||
        !a.table || !a.qn || !a.kn)
        return set_error(MSGL_ERR_INVALID_ARG, "qknorm_mrope: null pointer");
    if (!aligned16(a.qkv) || !aligned16(a.parts) || !aligned16(a.q_out) || !aligned16(a.k_pool) ||
        !aligned16(a.v_pool) || !aligned16(a.qn) || !aligned16(a.kn))
        return set_error(MSGL_ERR_INVALID_ARG, "qknorm_mrope: rows must be 16-byte aligned");
    a.s0 = s0; a.s1 = s1; a.s2 = s2; a.layout = layout;
    a.err = device_error_word();
    if (!a.err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    const int nh = a.hq + 2 * a.hkv;
    // Many tokens: three groups of heads a warp, so that a thread has 96 bytes in flight and the
    // table is gathered once for 48 heads; few: one, for more CTAs.
    const int it = !a.parts && a.num_tokens >= 8 * 148 ? 3 : 1;
    const int splits = (nh + 4 * kMropeWarps * it - 1) / (4 * kMropeWarps * it);
    if (splits > 65535) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "qknorm_mrope: too many heads");
    launch_pdl(a.parts ? qknorm_mrope_store_kernel<true, 1>
                       : it == 3 ? qknorm_mrope_store_kernel<false, 3> : qknorm_mrope_store_kernel<false, 1>,
               dim3(a.num_tokens, splits), dim3(kMropeWarps * 32), 0, stream, a);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

}  // namespace
}  // namespace msgl

using namespace msgl;

extern "C" {

int msgl_qknorm_mrope_store_kv(const void* qkv, void* q_out, void* k_pool, void* v_pool,
                               int64_t num_slots, const int* positions, int64_t position_stride,
                               const int* sections, int layout, const int* slot_mapping,
                               const float* cos_sin_cache, int max_position, const void* q_norm_w,
                               const void* k_norm_w, int num_tokens, int num_q_heads,
                               int num_kv_heads, int head_dim, float eps, msgl_stream_t stream) {
    MropeArgs a = {};
    a.qkv = static_cast<const __nv_bfloat16*>(qkv);
    a.q_out = static_cast<__nv_bfloat16*>(q_out);
    a.k_pool = static_cast<__nv_bfloat16*>(k_pool);
    a.v_pool = static_cast<__nv_bfloat16*>(v_pool);
    a.num_slots = num_slots;
    a.positions = positions;
    a.pos_stride = position_stride;
    a.slots = slot_mapping;
    a.table = cos_sin_cache;
    a.max_position = max_position;
    a.qn = static_cast<const __nv_bfloat16*>(q_norm_w);
    a.kn = static_cast<const __nv_bfloat16*>(k_norm_w);
    a.num_tokens = num_tokens;
    a.hq = num_q_heads;
    a.hkv = num_kv_heads;
    a.eps = eps;
    return launch_mrope(a, sections, layout, head_dim, stream);
}

int msgl_qknorm_mrope_store_kv_partials(const float* parts, int nparts, void* q_out, void* k_pool,
                                        void* v_pool, int64_t num_slots, const int* positions,
                                        int64_t position_stride, const int* sections, int layout,
                                        const int* slot_mapping, const float* cos_sin_cache,
                                        int max_position, const void* q_norm_w,
                                        const void* k_norm_w, int num_tokens, int num_q_heads,
                                        int num_kv_heads, int head_dim, float eps,
                                        msgl_stream_t stream) {
    if (!parts || nparts < 1 || nparts > 64)
        return set_error(MSGL_ERR_INVALID_ARG, "qknorm_mrope_partials: parts / nparts in [1, 64]");
    MropeArgs a = {};
    a.parts = parts;
    a.nparts = nparts;
    a.q_out = static_cast<__nv_bfloat16*>(q_out);
    a.k_pool = static_cast<__nv_bfloat16*>(k_pool);
    a.v_pool = static_cast<__nv_bfloat16*>(v_pool);
    a.num_slots = num_slots;
    a.positions = positions;
    a.pos_stride = position_stride;
    a.slots = slot_mapping;
    a.table = cos_sin_cache;
    a.max_position = max_position;
    a.qn = static_cast<const __nv_bfloat16*>(q_norm_w);
    a.kn = static_cast<const __nv_bfloat16*>(k_norm_w);
    a.num_tokens = num_tokens;
    a.hq = num_q_heads;
    a.hkv = num_kv_heads;
    a.eps = eps;
    return launch_mrope(a, sections, layout, head_dim, stream);
}

}  // extern "C"
