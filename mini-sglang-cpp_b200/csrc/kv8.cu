// kv8.cu -- append to the 8-bit key / value pool, and attention of single tokens and drafted rows over it.
//
//  * msgl_qknorm_rope_store_kv8 (+ _partials)  QK-norm + rotation + quantised append
//  * msgl_paged_attention_kv8                  attention (more than 16 rows x heads: kv8_tiles.cu)
//
// Format and conversions: kv8.cuh.
#include <algorithm>

#include "kv8.cuh"

namespace msgl {
namespace {

constexpr int kPage = kKv8Page;
constexpr int kHd = kKv8Head;
constexpr int kHalf = kHd / 2;
constexpr float kNegInf = -__builtin_huge_valf();

// ------------------------------------------------------------------ append
// Two warps per touched page, kv head and kind (keys, values): they bring the page's 16 x 128 values together
// in registers (earlier tokens from their codes, new ones from the projection, zeros behind the context's
// end), take the largest magnitude, and write codes and exponent. So the scale is that of the values
// which the page holds now (a rejected draft does not keep it up), and old codes are only rounded again
// where they become subnormal: e4m3 times a power of two is e4m3. NaN and infinities are stored as NaN
// and do not count for the scale, so they stay where they are. HBM bound.
// Lane 8 c + i: dimensions 8 i .. 8 i + 7 of one or both halves (keys: rotate-half partners) of the tokens 2 c, 2 c + 1
// and / or 8 + 2 c, 9 + 2 c: rows are read in pieces of 128 bytes, value units written in 16. Keys are split over the
// warps by tokens, values by dimensions; with one warp and 64 values a lane the kernel needed 162 registers and 8.5k
// tokens took 79 us, so 50 (24 of them the append, 29 the query heads by themselves; 53 with near_middle below).
// Query heads: eight lanes a head, as in the bf16 append.
constexpr int kStoreWarps = 4;

struct StoreArgs {
    const __nv_bfloat16* qkv;
    const float* parts;
    int nparts;
    __nv_bfloat16* q_out;
    uint8_t *kv8, *scales;
    int64_t num_pages;
    const int *positions, *page_table;
    int max_pages;
    const int *seq_lens, *q_indptr;
    int num_reqs, max_q_len;
    const float* table;
    int max_position;
    const __nv_bfloat16 *qn, *kn;
    int num_tokens, hq, hkv;
    float eps;
    int page_tasks;    // pages a request may touch
    int kv_blocks;     // blocks of the append; the others take query heads
    int q_groups;      // of 16 query heads, of a token
    int* err;
};

// 16 values of a head row: elements 8 i + e (e < 8) and 64 + 8 i + (e - 8), bf16 (their 32 bytes first, so that several
// rows' loads are in flight) or summed in part order.
__device__ __forceinline__ void load_raw(const StoreArgs& a, int64_t row, int head, int i, uint4 (&u)[2]) {
    const __nv_bfloat16* src = a.qkv + (row * (a.hq + 2 * a.hkv) + head) * kHd + 8 * i;
    u[0] = *reinterpret_cast<const uint4*>(src);
    u[1] = *reinterpret_cast<const uint4*>(src + kHalf);
}
__device__ __forceinline__ void raw_values(const uint4 (&u)[2], float (&x)[16]) {
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const uint32_t w[4] = {u[v].x, u[v].y, u[v].z, u[v].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[8 * v + 2 * e] = bf16lo(w[e]);
            x[8 * v + 2 * e + 1] = bf16hi(w[e]);
        }
    }
}
__device__ __forceinline__ void sum_parts(const StoreArgs& a, int64_t row, int head, int i, float (&x)[16]) {
    const int nh = a.hq + 2 * a.hkv;
    const int64_t stride = static_cast<int64_t>(a.num_tokens) * nh * kHd;
    const float* at = a.parts + (row * nh + head) * kHd + 8 * i;
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.f;
    for (int p = 0; p < a.nparts; p += 3) {  // three parts' loads in flight, added in part order
        float4 f[3][4];
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
            for (int v = 0; v < 4; ++v)
                f[q][v] = p + q < a.nparts ? *reinterpret_cast<const float4*>(at + (p + q) * stride + (v >> 1) * kHalf + (v & 1) * 4)
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

// x = x / sqrt(mean(x^2) + eps) * w, then the rotate-half pairs (8 i + e, 64 + 8 i + e) turned by the angle of
// table row `turn`. The eight lanes of a head call it together.
__device__ __forceinline__ void norm_turn(float (&x)[16], const __nv_bfloat16* w, const float* turn, int i, float eps) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) ss += x[e] * x[e];
    ss += __shfl_xor_sync(0xffffffffu, ss, 1);
    ss += __shfl_xor_sync(0xffffffffu, ss, 2);
    ss += __shfl_xor_sync(0xffffffffu, ss, 4);
    float inv = 1.0f / sqrtf(ss / kHd + eps);
    if (__any_sync(0xffffffffu, ss > 3.4e38f)) {  // squares beyond fp32: the sum once more, of x 2^-70
        float s2 = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float y = x[e] * 0x1p-70f;
            s2 += y * y;
        }
        s2 += __shfl_xor_sync(0xffffffffu, s2, 1);
        s2 += __shfl_xor_sync(0xffffffffu, s2, 2);
        s2 += __shfl_xor_sync(0xffffffffu, s2, 4);
        if (ss > 3.4e38f) inv = 0x1p-70f / sqrtf(s2 / kHd);
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const uint4 u = *reinterpret_cast<const uint4*>(w + 8 * i + v * kHalf);
        const uint32_t ww[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[8 * v + 2 * e] *= inv * bf16lo(ww[e]);
            x[8 * v + 2 * e + 1] *= inv * bf16hi(ww[e]);
        }
    }
    float c[8], s[8];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        *reinterpret_cast<float4*>(c + 4 * v) = *reinterpret_cast<const float4*>(turn + 8 * i + 4 * v);
        *reinterpret_cast<float4*>(s + 4 * v) = *reinterpret_cast<const float4*>(turn + kHalf + 8 * i + 4 * v);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float lo = x[e], hi = x[8 + e];
        x[e] = lo * c[e] - hi * s[e];
        x[8 + e] = lo * s[e] + hi * c[e];
    }
}

// A value as h + l, and exact sums and products of fp32 values as such.
struct Two {
    float h, l;
};
__device__ __forceinline__ Two two_sum(float a, float b) {
    const float s = __fadd_rn(a, b), t = __fsub_rn(s, a);
    return {s, __fadd_rn(__fsub_rn(a, __fsub_rn(s, t)), __fsub_rn(b, t))};
}
__device__ __forceinline__ Two two_product(float a, float b) {
    const float p = __fmul_rn(a, b);
    return {p, fmaf(a, b, -p)};
}

// h + l rounded to the odd neighbour unless it is exact: rounding that to fewer bits is then right.
__device__ __forceinline__ float odd_sum(float h, float l) {
    const Two s = two_sum(h, l);
    const uint32_t u = __float_as_uint(s.h);
    if (!(fabsf(s.l) > 0.f) || (u & 1)) return s.h;
    return __uint_as_float((s.l > 0.f) == (s.h > 0.f) ? u + 1 : u - 1);
}

// norm_turn of a key, rounded once at the end.
__device__ __forceinline__ void norm_turn_exactly(float (&x)[16], const __nv_bfloat16* w, const float* turn, int i, float eps) {
    Two part[4];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const Two p = two_product(x[e], x[e]), t = two_sum(e < 4 ? 0.f : part[e & 3].h, p.h);
        part[e & 3] = {t.h, (e < 4 ? 0.f : part[e & 3].l) + (t.l + p.l)};
    }
    const Two s0 = two_sum(part[0].h, part[1].h), s1 = two_sum(part[2].h, part[3].h), all = two_sum(s0.h, s1.h);
    Two ss = {all.h, (part[0].l + part[1].l) + (part[2].l + part[3].l) + (s0.l + s1.l) + all.l};
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const float h = __shfl_xor_sync(0xffffffffu, ss.h, o), l = __shfl_xor_sync(0xffffffffu, ss.l, o);
        const Two t = two_sum(ss.h, h);
        ss = {t.h, ss.l + l + t.l};
    }
    // 1 / sqrt(mean + eps): the fp32 value, and a step of Newton's method for the rest
    const Two m = two_sum(ss.h / kHd, eps), v = two_sum(m.h, m.l + ss.l / kHd);
    Two inv = {1.0f / sqrtf(v.h), 0.f};
    const Two square = two_product(inv.h, inv.h);
    inv.l = 0.5f * inv.h * (fmaf(-v.h, square.h, 1.f) - fmaf(v.h, square.l, v.l * square.h));
    if (__any_sync(0xffffffffu, ss.h > 3.4e38f)) {  // squares beyond fp32: the sum once more, of x 2^-70
        float s2 = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float y = x[e] * 0x1p-70f;
            s2 += y * y;
        }
        s2 += __shfl_xor_sync(0xffffffffu, s2, 1);
        s2 += __shfl_xor_sync(0xffffffffu, s2, 2);
        s2 += __shfl_xor_sync(0xffffffffu, s2, 4);
        if (ss.h > 3.4e38f) inv = {0x1p-70f / sqrtf(s2 / kHd), 0.f};
    }
    auto normed = [&](float y, float weight) {
        Two g = two_product(inv.h, weight);
        g.l = fmaf(inv.l, weight, g.l);
        Two z = two_product(y, g.h);
        z.l = fmaf(y, g.l, z.l);
        return z;
    };
#pragma unroll
    for (int v4 = 0; v4 < 2; ++v4) {
        const float4 c4 = *reinterpret_cast<const float4*>(turn + 8 * i + 4 * v4), s4 = *reinterpret_cast<const float4*>(turn + kHalf + 8 * i + 4 * v4);
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
        const uint2 w0 = *reinterpret_cast<const uint2*>(w + 8 * i + 4 * v4), w1 = *reinterpret_cast<const uint2*>(w + kHalf + 8 * i + 4 * v4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t a = e < 2 ? w0.x : w0.y, b = e < 2 ? w1.x : w1.y;
            const Two lo = normed(x[4 * v4 + e], e & 1 ? bf16hi(a) : bf16lo(a)), hi = normed(x[8 + 4 * v4 + e], e & 1 ? bf16hi(b) : bf16lo(b));
            auto turned = [&](const Two& y, float f, const Two& z, float g) {  // y f + z g
                const Two p = two_product(y.h, f), q = two_product(z.h, g), t = two_sum(p.h, q.h);
                return odd_sum(t.h, t.l + (p.l + q.l) + fmaf(y.l, f, z.l * g));
            };
            x[4 * v4 + e] = turned(lo, c[e], hi, -s[e]);
            x[8 + 4 * v4 + e] = turned(lo, s[e], hi, c[e]);
        }
    }
}

// Where each step is rounded to fp32, a value that is within some 2^-23 of the middle of two codes may end on the wrong side:
// one of 10^6. Tokens with a value that close (6 of its units; the bits behind the code tell) are computed again, exactly
// but for one rounding, which is 1% of the warps' tokens: 8.5k tokens 4% more time, 240 rows behind 6 partials 6%.
// (All of them so: 20% and 60%.) What is left, one of 10^7, are codes below 2^-6, whose middles lie elsewhere.
__device__ __forceinline__ bool near_middle(float code) { return ((__float_as_uint(code) - 0x80000u + 6u) & 0xfffffu) <= 12u; }

// 4 N values of a head row as sums of partials, to the odd neighbour: N float4 at at + step * v, three parts' loads in flight.
template <int N>
__device__ __forceinline__ void sum_exactly(const float* at, const int (&step)[N], int64_t stride, int nparts, float* x) {
    float l[4 * N];
#pragma unroll
    for (int e = 0; e < 4 * N; ++e) x[e] = l[e] = 0.f;
    for (int p = 0; p < nparts; p += 3) {
        float4 f[3][N];
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
            for (int v = 0; v < N; ++v)
                f[q][v] = p + q < nparts ? *reinterpret_cast<const float4*>(at + (p + q) * stride + step[v]) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
            for (int v = 0; v < N; ++v) {
                const float y[4] = {f[q][v].x, f[q][v].y, f[q][v].z, f[q][v].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float z = __fsub_rn(y[e], l[4 * v + e]), t = __fadd_rn(x[4 * v + e], z);  // Kahan
                    l[4 * v + e] = __fsub_rn(__fsub_rn(t, x[4 * v + e]), z);
                    x[4 * v + e] = t;
                }
            }
    }
#pragma unroll
    for (int e = 0; e < 4 * N; ++e) x[e] = odd_sum(x[e], -l[e]);
}
template <bool PARTS>
__device__ __noinline__ void key_exactly(const void* src, int64_t stride, int nparts, const __nv_bfloat16* w, const float* turn, int i, float eps, float* y) {
    float x[16];
    if (PARTS) {
        const int step[4] = {0, 4, kHalf, kHalf + 4};
        sum_exactly<4>(static_cast<const float*>(src), step, stride, nparts, x);
    } else {
        const __nv_bfloat16* raw = static_cast<const __nv_bfloat16*>(src);
        const uint4 u[2] = {*reinterpret_cast<const uint4*>(raw), *reinterpret_cast<const uint4*>(raw + kHalf)};
        raw_values(u, x);
    }
    norm_turn_exactly(x, w, turn, i, eps);
#pragma unroll
    for (int e = 0; e < 16; ++e) y[e] = fabsf(x[e]) < __builtin_huge_valf() ? x[e] : __int_as_float(0x7fffffff);
}
__device__ __noinline__ void values_exactly(const float* src, int64_t stride, int nparts, float* y) {
    float x[8];
    const int step[2] = {0, 4};
    sum_exactly<2>(src, step, stride, nparts, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = fabsf(x[e]) < __builtin_huge_valf() ? x[e] : __int_as_float(0x7fffffff);
}

__device__ __forceinline__ const float* turn_row(const StoreArgs& a, int64_t row) {
    int pos = a.positions[row];
    if (static_cast<unsigned>(pos) >= static_cast<unsigned>(a.max_position)) {
        record_error(a.err, MSGL_ERR_BOUNDS, 912);
        pos = 0;
    }
    return a.table + static_cast<int64_t>(pos) * kHd;
}

// The page of a task: its place in the pool, and which of its tokens are held already (t < old), new, or behind the
// context's end (pos >= L).
struct PageTask {
    int64_t block;  // page and head
    int kind, h, page, old, begin, L, q0, n;

    __device__ __forceinline__ bool live(int t) const { return t >= old && page * kPage + t < L; }
    // row of a new token; of the others the request's last one, so that all lanes work on something
    __device__ __forceinline__ int64_t row(int t) const { return q0 + (live(t) ? page * kPage + t - begin : n - 1); }
};

__device__ __forceinline__ bool find_page(const StoreArgs& a, int task, bool report, PageTask& p) {
    p.kind = task & 1;  // 0 keys, 1 values
    task >>= 1;
    p.h = task % a.hkv;
    task /= a.hkv;
    const int r = task / a.page_tasks, nth = task % a.page_tasks;
    p.L = a.seq_lens[r];
    p.q0 = a.q_indptr ? a.q_indptr[r] : r;
    p.n = a.q_indptr ? a.q_indptr[r + 1] - p.q0 : 1;
    const bool first = report && nth == 0 && p.h == 0 && p.kind == 0;
    if (p.L < 0 || p.L > a.max_pages * static_cast<int64_t>(kPage) || p.n < 0 || p.n > p.L) {
        if (first && p.n != 0) record_error(a.err, MSGL_ERR_BOUNDS, 910);
        return false;
    }
    if (p.n == 0) return false;
    if (p.n > a.max_q_len || p.q0 < 0 || p.q0 > a.num_tokens - p.n) {
        if (first) record_error(a.err, MSGL_ERR_BOUNDS, 911);
        return false;
    }
    p.begin = p.L - p.n;
    p.page = p.begin / kPage + nth;
    if (p.page * kPage >= p.L) return false;
    const int phys = a.page_table[static_cast<int64_t>(r) * a.max_pages + p.page];
    if (phys < 0 || phys >= a.num_pages) {
        if (report) record_error(a.err, MSGL_ERR_BOUNDS, 913);
        return false;
    }
    p.block = static_cast<int64_t>(phys) * a.hkv + p.h;
    p.old = p.begin - p.page * kPage;
    return true;
}

// The exponent of the page's values, of which the two warps of a pair hold 32 a lane each; NaN and infinities become
// NaN and do not count. (A maximum within fp32's rounding of 448 2^e may take the exponent next to the definition's, one page of
// 10^6: e4m3 of either scale is the same but for subnormals.)
__device__ __forceinline__ int page_exponent(float (&x)[32], float* maxima, int warp, int lane) {
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        if (fabsf(x[e]) < __builtin_huge_valf()) amax = fmaxf(amax, fabsf(x[e]));
        else x[e] = __int_as_float(0x7fffffff);
    }
    amax = warp_max(amax);
    if (lane == 0) maxima[warp] = amax;
    __syncwarp();
    asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp >> 1)) : "memory");
    return kv8_exponent(fmaxf(maxima[warp & ~1], maxima[warp | 1]));
}

// Keys: this warp's tokens are t0 + 2 c and t0 + 2 c + 1, t0 = 0 or 8.
template <bool PARTS>
__device__ __forceinline__ void append_keys(const StoreArgs& a, const PageTask& p, float* maxima, int warp, int lane) {
    uint8_t* codes = a.kv8 + p.block * kKv8Bytes;
    const int c = lane >> 3, i = lane & 7, t0 = (warp & 1) * 8 + 2 * c;
    float x[32];  // token t0 + e: [16 e, 16 e + 16)
    uint4 raw[2][2];
    bool some[2];  // some lane's token is a new one
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        some[e] = __any_sync(0xffffffffu, p.live(t0 + e));
        if (some[e] && !PARTS) load_raw(a, p.row(t0 + e), a.hq + p.h, i, raw[e]);
    }
    if (p.old > 0) {
        const float s = kv8_power(a.scales[2 * p.block]);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const uint2 u = *reinterpret_cast<const uint2*>(codes + v * 1024 + (t0 + e) * 64 + 8 * i);
                const uint32_t w[2] = {u.x, u.y};
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const float2 f = __half22float2(__nv_cvt_fp8x2_to_halfraw2(w[b >> 1] >> ((b & 1) * 16) & 0xffff, __NV_E4M3));
                    x[16 * e + 8 * v + 2 * b] = f.x * s;
                    x[16 * e + 8 * v + 2 * b + 1] = f.y * s;
                }
            }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int t = t0 + e;
        if (some[e]) {
            float y[16];
            const int64_t row = p.row(t);
            if (PARTS) sum_parts(a, row, a.hq + p.h, i, y);
            else raw_values(raw[e], y);
            norm_turn(y, a.kn, turn_row(a, row), i, a.eps);
#pragma unroll
            for (int d = 0; d < 16; ++d) x[16 * e + d] = p.live(t) ? y[d] : t < p.old ? x[16 * e + d] : 0.f;
        } else if (t >= p.old) {
#pragma unroll
            for (int d = 0; d < 16; ++d) x[16 * e + d] = 0.f;
        }
    }
    const int stored = page_exponent(x, maxima, warp, lane);
    const float inv = kv8_inverse(stored);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        bool near = false;
#pragma unroll
        for (int d = 0; d < 16; ++d) near |= near_middle(x[16 * e + d] * inv);
        if (some[e] && __any_sync(0xffffffffu, near)) {
            const int nh = a.hq + 2 * a.hkv;
            const int64_t row = p.row(t0 + e), at = (row * nh + a.hq + p.h) * kHd + 8 * i;
            float y[16];
            key_exactly<PARTS>(PARTS ? static_cast<const void*>(a.parts + at) : a.qkv + at, static_cast<int64_t>(a.num_tokens) * nh * kHd, a.nparts, a.kn,
                               turn_row(a, row), i, a.eps, y);
#pragma unroll
            for (int d = 0; d < 16; ++d)
                if (p.live(t0 + e)) x[16 * e + d] = y[d];
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            uint32_t w[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) w[b] = e4m3_codes2(x[16 * e + 8 * v + 2 * b] * inv, x[16 * e + 8 * v + 2 * b + 1] * inv);
            *reinterpret_cast<uint2*>(codes + v * 1024 + (t0 + e) * 64 + 8 * i) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
        }
    if ((warp & 1) == 0 && lane == 0) a.scales[2 * p.block] = static_cast<uint8_t>(stored);
}

// Values: this warp's dimensions are half + 8 i .. + 7, half = 0 or 64; of the tokens 2 c, 2 c + 1, 8 + 2 c, 9 + 2 c.
template <bool PARTS>
__device__ __forceinline__ void append_values(const StoreArgs& a, const PageTask& p, float* maxima, int warp, int lane) {
    const int c = lane >> 3, i = lane & 7, half = (warp & 1) * kHalf;
    uint8_t* codes = a.kv8 + p.block * kKv8Bytes + kKv8Values + (half / 4 + 2 * i) * 64 + c * 16;  // a unit, and one 64 further
    const int head = a.hq + a.hkv + p.h, nh = a.hq + 2 * a.hkv;
    float x[32];  // token e, dimension d: 8 e + d
    uint4 raw[4], held[2];
    bool some[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int t = token_at(4 * c + e);
        some[e] = __any_sync(0xffffffffu, p.live(t));
        if (some[e] && !PARTS) raw[e] = *reinterpret_cast<const uint4*>(a.qkv + (p.row(t) * nh + head) * kHd + half + 8 * i);
    }
    float s = 0.f;
    if (p.old > 0) {
        s = kv8_power(a.scales[2 * p.block + 1]);
#pragma unroll
        for (int v = 0; v < 2; ++v) held[v] = *reinterpret_cast<const uint4*>(codes + v * 64);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int t = token_at(4 * c + e);
        float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (some[e]) {
            if (PARTS) {
                const int64_t stride = static_cast<int64_t>(a.num_tokens) * nh * kHd;
                const float* at = a.parts + (p.row(t) * nh + head) * kHd + half + 8 * i;
#pragma unroll 3
                for (int q = 0; q < a.nparts; ++q)
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const float4 f = *reinterpret_cast<const float4*>(at + q * stride + 4 * v);
                        y[4 * v] += f.x; y[4 * v + 1] += f.y; y[4 * v + 2] += f.z; y[4 * v + 3] += f.w;
                    }
            } else {
                const uint32_t w[4] = {raw[e].x, raw[e].y, raw[e].z, raw[e].w};
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    y[2 * d] = bf16lo(w[d]);
                    y[2 * d + 1] = bf16hi(w[d]);
                }
            }
        }
#pragma unroll
        for (int d = 0; d < 8; ++d) x[8 * e + d] = p.live(t) ? y[d] : 0.f;
        if (p.old > 0 && t < p.old) {
#pragma unroll
            for (int d = 0; d < 8; ++d) {  // unit d / 4, its dimension d % 4: word d % 4, byte e
                const uint4& u = held[d >> 2];
                const uint32_t w = (d & 3) == 0 ? u.x : (d & 3) == 1 ? u.y : (d & 3) == 2 ? u.z : u.w;
                x[8 * e + d] = __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<uint8_t>(w >> (8 * e)), __NV_E4M3))) * s;
            }
        }
    }
    const int stored = page_exponent(x, maxima, warp, lane);
    const float inv = kv8_inverse(stored);
    if (PARTS)  // (the others are bf16 as they stand)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int t = token_at(4 * c + e);
            bool near = false;
#pragma unroll
            for (int d = 0; d < 8; ++d) near |= near_middle(x[8 * e + d] * inv);
            if (near && p.live(t)) {
                float y[8];
                values_exactly(a.parts + (p.row(t) * nh + head) * kHd + half + 8 * i, static_cast<int64_t>(a.num_tokens) * nh * kHd, a.nparts, y);
#pragma unroll
                for (int d = 0; d < 8; ++d) x[8 * e + d] = y[d];
            }
        }
    __syncwarp();
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        uint32_t w[4];
#pragma unroll
        for (int d = 0; d < 4; ++d)
            w[d] = e4m3_codes2(x[4 * v + d] * inv, x[8 + 4 * v + d] * inv) |
                   e4m3_codes2(x[16 + 4 * v + d] * inv, x[24 + 4 * v + d] * inv) << 16;
        *reinterpret_cast<uint4*>(codes + v * 64) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if ((warp & 1) == 0 && lane == 0) a.scales[2 * p.block + 1] = static_cast<uint8_t>(stored);
}

template <bool PARTS, int IT>
__global__ void __launch_bounds__(kStoreWarps * 32, PARTS ? 4 : 8)
qknorm_rope_store_kv8_kernel(const StoreArgs a) {
    pdl_wait();
    pdl_trigger();
    __shared__ float maxima[kStoreWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (static_cast<int>(blockIdx.x) < a.kv_blocks) {
        const int task = blockIdx.x * (kStoreWarps / 2) + (warp >> 1);
        PageTask p;
        if (task >= a.num_reqs * a.page_tasks * a.hkv * 2 || !find_page(a, task, lane == 0 && (warp & 1) == 0, p)) return;
        if (p.kind == 0) append_keys<PARTS>(a, p, maxima, warp, lane);
        else append_values<PARTS>(a, p, maxima, warp, lane);
        return;
    }
    // query heads: a warp takes four of 16 heads of a token, IT such groups in a row with their loads in flight together
    const int i = lane & 7;
    const int64_t first = a.q_indptr ? a.q_indptr[0] : 0, last = a.q_indptr ? a.q_indptr[a.num_reqs] : a.num_tokens;
    const int64_t g0 = static_cast<int64_t>(blockIdx.x - a.kv_blocks) * IT;
    uint4 raw[PARTS ? 1 : IT][2];
    const float* turn[IT];
    int64_t token[IT];
    int head[IT];
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        token[k] = (g0 + k) / a.q_groups;
        head[k] = static_cast<int>((g0 + k) % a.q_groups) * 16 + warp * 4 + (lane >> 3);
        if (token[k] < first || token[k] >= last || token[k] >= a.num_tokens) token[k] = -1;  // no request's row
        if (token[k] < 0) continue;
        if (!PARTS) load_raw(a, token[k], min(head[k], a.hq - 1), i, raw[PARTS ? 0 : k]);
        turn[k] = turn_row(a, token[k]);
    }
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        if (token[k] < 0) continue;
        float x[16];
        if (PARTS) sum_parts(a, token[k], min(head[k], a.hq - 1), i, x);
        else raw_values(raw[PARTS ? 0 : k], x);
        norm_turn(x, a.qn, turn[k], i, a.eps);
        if (head[k] < a.hq) {
#pragma unroll
            for (int v = 0; v < 2; ++v)
                *reinterpret_cast<uint4*>(a.q_out + (token[k] * a.hq + head[k]) * kHd + v * kHalf + 8 * i) =
                    make_uint4(pack_bf16x2(x[8 * v], x[8 * v + 1]), pack_bf16x2(x[8 * v + 2], x[8 * v + 3]),
                               pack_bf16x2(x[8 * v + 4], x[8 * v + 5]), pack_bf16x2(x[8 * v + 6], x[8 * v + 7]));
        }
        __syncwarp();
    }
}

int launch_store(StoreArgs a, int head_dim, int page_size, msgl_stream_t stream) {
    if (head_dim != kHd) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "store_kv8: head_dim must be 128");
    if (page_size != kPage) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "store_kv8: page_size must be 16");
    if (a.num_tokens < 0 || a.num_reqs < 0 || a.max_q_len < 0 || a.hq <= 0 || a.hkv <= 0 || a.max_position <= 0 ||
        a.num_pages <= 0 || a.max_pages <= 0 || a.max_pages > INT32_MAX / kPage)
        return set_error(MSGL_ERR_INVALID_ARG, "store_kv8: bad sizes");
    if (!a.q_indptr && (a.max_q_len != 1 || a.num_tokens != a.num_reqs))
        return set_error(MSGL_ERR_INVALID_ARG, "store_kv8: one row per request without q_indptr");
    if (a.num_tokens == 0 || a.num_reqs == 0 || a.max_q_len == 0) return MSGL_OK;
    if ((!a.qkv && !a.parts) || !a.q_out || !a.kv8 || !a.scales || !a.positions || !a.page_table || !a.seq_lens ||
        !a.table || !a.qn || !a.kn)
        return set_error(MSGL_ERR_INVALID_ARG, "store_kv8: null pointer");
    if (!aligned16(a.qkv) || !aligned16(a.parts) || !aligned16(a.q_out) || !aligned16(a.kv8) || !aligned16(a.qn) ||
        !aligned16(a.kn) || !aligned16(a.table))
        return set_error(MSGL_ERR_INVALID_ARG, "store_kv8: rows must be 16-byte aligned");
    const int64_t rows = std::min(a.max_q_len, a.num_tokens);
    a.page_tasks = static_cast<int>((rows + kPage - 2) / kPage + 1);
    // Groups of query heads a warp: four, so that its loads cover their latency (8.2k tokens 50 us, with one 54);
    // of partials one, whose sums have loads enough.
    const int it = a.parts ? 1 : 4;
    a.q_groups = (a.hq + 15) / 16;
    const int64_t tasks = static_cast<int64_t>(a.num_reqs) * a.page_tasks * a.hkv * 2;
    const int64_t kv = (tasks + kStoreWarps / 2 - 1) / (kStoreWarps / 2);
    const int64_t grid = kv + (static_cast<int64_t>(a.num_tokens) * a.q_groups + it - 1) / it;
    if (tasks > INT32_MAX / 2 || grid > INT32_MAX)
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "store_kv8: too many rows, requests or heads");
    a.kv_blocks = static_cast<int>(kv);
    a.err = device_error_word();
    if (!a.err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    launch_pdl(a.parts ? qknorm_rope_store_kv8_kernel<true, 1> : qknorm_rope_store_kv8_kernel<false, 4>,
               dim3(static_cast<unsigned>(grid)), dim3(kStoreWarps * 32), 0, stream, a);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

// ------------------------------------------------------------------ attention of few rows
// The rows of a kv head (query row x head of its group, at most 8 NT of them) against its pages. MMAs
// m16n8k16 in f16: S = Q K^T with the rows as M and the 16 keys of a page as two N tiles, then
// O^T += V^T P^T with 16 dimensions as M, 8 rows as N and the page's keys as K, where S's accumulators are
// P^T's fragments as they stand. Codes are exact in f16; q is scaled by a power of two per row (kv8.cuh); a page's scales enter the exponent,
//   s = (q . k) 2^(q + k exponents) scale log2(e) + (exponent of v),  p = 2^(s - m + 11) in f16 (kv8.cuh),
// so that O needs no scaling by page, and l adds p 2^-(11 + exponent of v). HBM bound: 4 KB a page and head,
// 24 or 32 MMAs, 64 conversions.
//
// In a CTA the pages of an item go around the warps, each with a ring of 4 KB stages that a warp of its own
// fills by bulk copies, across items. Where an item is shared by CTAs they leave partial sums in the workspace.
constexpr int kWarps = 7;                        // that attend (eight warps in all: 128 registers a thread at two CTAs an SM)
constexpr int kBatch = 32 / kWarps * kWarps;     // pages whose ids are read together
constexpr int kAttThreads = kWarps * 32;        // that attend; one warp more copies
constexpr int kPitch = kHd + 4;  // floats of a row in the joining buffer
constexpr int kItemCost = 12;    // of an item, in pages: 128 requests of 200 to 3800 tokens 108 us without, 102 with 8 or 12

template <int NT>
struct RowsShape {
    static constexpr int kCtas = NT == 1 ? 2 : 1;  // per SM
    static constexpr int kRing = NT == 1 ? 2 : 4;  // stages of a warp
    static constexpr int kRows = NT * 8;
    static constexpr size_t kJoin = static_cast<size_t>(kWarps) * kRows * (kPitch + 2) * 4;
    static constexpr size_t kSmem = static_cast<size_t>(kRing) * kWarps * kKv8Bytes + kJoin;
};

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT>
struct RowState {
    uint32_t q[8][NT == 1 ? 2 : 4];  // Q fragments: k step, a0 a2 (a1 a3)
    float qs[NT];                    // 2^(q exponent) scale log2(e)
    int lim[NT];                     // last visible key of rows g (and 8 + g); -1: no such row
    float m[NT], l[NT];
    float o[8][NT][4];
};

// NaN values at keys that only some rows see: those rows' sums become NaN. nan[v]: bytes of the lane's value
// words (4 dimensions x 4 tokens) that hold NaN, 0x80 each.
template <int NT>
__device__ __forceinline__ void spread_nan(RowState<NT>& st, const uint32_t (&nan)[16], int key0, int lane) {
    const int c = lane & 3;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        uint32_t tok = 0;  // tokens of the page
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (nan[v] & (0x80u << (8 * e))) tok |= 1u << ((e >> 1) * 8 + 2 * c + (e & 1));
        tok |= __shfl_xor_sync(0xffffffffu, tok, 1);
        tok |= __shfl_xor_sync(0xffffffffu, tok, 2);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int lim = __shfl_sync(0xffffffffu, st.lim[t], (2 * c + b) * 4);  // of row 8 t + 2 c + b
                const int seen = min(16, lim - key0 + 1);
                const uint32_t vis = seen <= 0 ? 0u : (1u << seen) - 1u;
                // tile (v / 4, (v % 4) / 2): dimension rows g (even v) and 8 + g (odd v)
                if (tok & vis) st.o[v >> 1][t][(v & 1) * 2 + b] = __int_as_float(0x7fffffff);
            }
    }
}

// One page: EDGE where some live row does not see all of its keys.
template <int NT, bool EDGE>
__device__ __forceinline__ void attend_page8(const uint8_t* page, uint32_t scale2, RowState<NT>& st, int key0, int min_lim,
                                             int lane) {
    const int g = lane >> 2, c = lane & 3;
    float s[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint4 u[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) u[t] = *reinterpret_cast<const uint4*>(page + half * 1024 + (t * 8 + g) * 64 + c * 16);
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                uint32_t b0, b1;
                e4m3x4_to_half(w == 0 ? u[t].x : w == 1 ? u[t].y : w == 2 ? u[t].z : u[t].w, b0, b1);
                const uint32_t* q = st.q[half * 4 + w];
                mma_f16_16816(s[t], q[0], NT == 1 ? 0u : q[NT == 1 ? 0 : 2], q[1], NT == 1 ? 0u : q[NT == 1 ? 0 : 3], b0, b1);
            }
    }
    const float kscale = kv8_power(scale2 & 0xff);
    const int vstored = kv8_value_exponent(scale2);
    const float vexp = static_cast<float>(vstored - 127), vinv = kv8_inverse(vstored) * kKv8Unlift;
    float p[NT][4];
    bool moved = false;
    float alpha[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float f = st.qs[t] * kscale;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = fmaf(s[e >> 1][2 * t + (e & 1)], f, vexp);
            p[t][e] = EDGE && key0 + (e >> 1) * 8 + 2 * c + (e & 1) > st.lim[t] ? kNegInf : x;
        }
        float mx = fmaxf(fmaxf(p[t][0], p[t][1]), fmaxf(p[t][2], p[t][3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const bool move = kv8_grows(mx, st.m[t]);
        const float next = move ? fmaxf(mx, st.m[t]) : st.m[t];
        alpha[t] = 1.f;
        if (move && next != kNegInf) {
            alpha[t] = exp2f(st.m[t] - next);
            moved = true;
        }
        st.m[t] = next;
        const float base = kv8_base(next);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            p[t][e] = exp2f(p[t][e] - base);
            sum += p[t][e];
        }
        st.l[t] = fmaf(sum, vinv, st.l[t] * alpha[t]);
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float a0 = __shfl_sync(0xffffffffu, alpha[t], (2 * c) * 4);
            const float a1 = __shfl_sync(0xffffffffu, alpha[t], (2 * c + 1) * 4);
#pragma unroll
            for (int v = 0; v < 8; ++v) {
                st.o[v][t][0] *= a0;
                st.o[v][t][1] *= a1;
                st.o[v][t][2] *= a0;
                st.o[v][t][3] *= a1;
            }
        }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        pb[t][0] = pack_half2(p[t][0], p[t][1]);
        pb[t][1] = pack_half2(p[t][2], p[t][3]);
    }
    uint32_t hidden = 0;  // 0x80 in the bytes of tokens that some live row does not see
    if (EDGE)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (key0 + (e >> 1) * 8 + 2 * c + (e & 1) > min_lim) hidden |= 0x80u << (8 * e);
    uint32_t nan[EDGE ? 16 : 1], any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint4 u = *reinterpret_cast<const uint4*>(page + kKv8Values + ((g + 8 * i) * 4 + c) * 16);
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (EDGE) {
                const uint32_t bad = nan_codes(w[j]) & hidden;
                nan[EDGE ? 4 * i + j : 0] = bad;
                any |= bad;
                w[j] &= ~((bad >> 7) * 0xffu);
            }
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
            uint32_t a0, a1, a2, a3;
            e4m3x4_to_half(w[2 * jj], a0, a2);
            e4m3x4_to_half(w[2 * jj + 1], a1, a3);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_f16_16816(st.o[2 * i + jj][t], a0, a1, a2, a3, pb[t][0], pb[t][1]);
        }
    }
    if (EDGE)
        if (__any_sync(0xffffffffu, any != 0)) spread_nan<NT>(st, reinterpret_cast<uint32_t(&)[16]>(nan), key0, lane);
}

// Q rows of an item into fragments. Row m: query row m / group, head m % group.
template <int NT>
__device__ __forceinline__ void load_rows(const Kv8AttnArgs& a, const Kv8Item& it, RowState<NT>& st, int lane) {
    const int g = lane >> 2, c = lane & 3, group = a.hq / a.hkv;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int m = t * 8 + g;
        const bool live = m < it.rows * group;
        const int i = it.row0 + (live ? m / group : 0);
        st.lim[t] = live ? it.L - it.n + i : -1;
        const __nv_bfloat16* src = a.q + (static_cast<int64_t>(it.q0 + i) * a.hq + it.h * group + (live ? m % group : 0)) * kHd;
        uint4 u[4];
#pragma unroll
        for (int v = 0; v < 4; ++v)
            u[v] = live ? *reinterpret_cast<const uint4*>(src + (v >> 1) * kHalf + 16 * c + (v & 1) * 8) : make_uint4(0, 0, 0, 0);
        float amax = 0.f;
        bool bad = false;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const uint32_t w[4] = {u[v].x, u[v].y, u[v].z, u[v].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = fmaxf(fabsf(bf16lo(w[e])), fabsf(bf16hi(w[e])));
                amax = fmaxf(amax, x);
                bad |= finite2(w[e]) != w[e];
            }
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const uint32_t bads = __ballot_sync(0xffffffffu, bad) >> (4 * g) & 0xfu;
        const int stored = kv8_query_exponent(amax);
        const float inv = kv8_inverse(stored);
        // a row with an infinity or a NaN has no defined logit: NaN throughout
        st.qs[t] = bads ? __int_as_float(0x7fffffff) : kv8_power(stored) * a.sl2e;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const uint32_t w[4] = {u[v].x, u[v].y, u[v].z, u[v].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // word 2 (v % 2) + e / 2 of the 16 bytes of codes, its bytes 2 (e % 2)
                const uint32_t f = bads ? 0u : pack_half2(bf16lo(w[e]) * inv, bf16hi(w[e]) * inv);
                st.q[(v >> 1) * 4 + (v & 1) * 2 + (e >> 1)][(NT == 1 ? 0 : 2 * t) + (e & 1)] = f;
            }
        }
        st.m[t] = kNegInf;
        st.l[t] = 0.f;
    }
#pragma unroll
    for (int v = 0; v < 8; ++v)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[v][t][e] = 0.f;
}

// The attending warps.
__device__ __forceinline__ void attending_barrier() {
    __syncwarp();
    asm volatile("bar.sync 1, %0;" ::"n"(kAttThreads) : "memory");
}

template <int NT>
__global__ void __launch_bounds__(kAttThreads + 32, RowsShape<NT>::kCtas)
attend_rows_kernel(const Kv8AttnArgs a) {
    using S = RowsShape<NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    float* join = reinterpret_cast<float*>(smem + S::kRing * kWarps * kKv8Bytes);  // [warp][row][kPitch]
    float* join_ml = join + kWarps * S::kRows * kPitch;                            // [warp][row]{m, l}
    __shared__ uint64_t full[S::kRing * kWarps], empty[S::kRing * kWarps];
    __shared__ uint32_t stage_scales[S::kRing * kWarps];
    __shared__ Kv8Scan<kAttThreads + 32> scan;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.hq / a.hkv;
    if (tid == 0) {
        for (int i = 0; i < S::kRing * kWarps; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        fence_barrier_init();
    }
    pdl_wait();
    pdl_trigger();
    const int per_block = S::kRows / group;  // query rows of a block
    Kv8Walk<kPage, kItemCost> use;
    if (!kv8_part(a, per_block, scan, use)) return;

    if (warp == kWarps) {
        // ---------------- copies: lane l takes pages l, kBatch + l, ... of an item's part, for warp l % kWarps
        int filled = 0;  // pages that this warp got before this item
        bool ok = true;
        do {
            const int p0 = use.u0(), p1 = use.u1();
            const int* table = a.page_table + static_cast<int64_t>(use.it.r) * a.max_pages;
            const int w = lane % kWarps;
            int next = lane < kBatch && p0 + lane < p1 ? table[p0 + lane] : 0;
            for (int base = p0; base < p1; base += kBatch) {
                const int p = lane < kBatch ? base + lane : p1;
                int id = next;
                next = p + kBatch < p1 ? table[p + kBatch] : 0;
                if (id < 0 || id >= a.num_pages) {
                    record_error(a.err, MSGL_ERR_BOUNDS, 902);
                    id = 0;
                }
                const int64_t block = static_cast<int64_t>(id) * a.hkv + use.it.h;
                const uint32_t sc = p < p1 ? *reinterpret_cast<const uint16_t*>(a.scales + block * 2) : 0u;
                const int n = filled + (p - p0) / kWarps, st = w * S::kRing + n % S::kRing;
#pragma unroll
                for (int round = 0; round < kBatch / kWarps; ++round) {
                    if (lane / kWarps == round && p < p1) {
                        if (n >= S::kRing) ok = ok && mbar_wait(&empty[st], (n / S::kRing - 1) & 1, a.err, 903);
                        if (ok) {
                            stage_scales[st] = sc;
                            mbar_arrive_expect_tx(&full[st], kKv8Bytes);
                            bulk_load(smem + st * kKv8Bytes, a.kv8 + block * kKv8Bytes, kKv8Bytes, &full[st]);
                        }
                    }
                    __syncwarp();
                }
            }
            filled += (p1 - p0 - w + kWarps - 1) / kWarps;
        } while (__all_sync(0xffffffffu, ok) && use.next(a, per_block));
        // after a wait that ran out: no copy is left on its way into the block's shared memory
        if (lane < kWarps)
            for (int i = max(0, filled - S::kRing); i < filled; ++i) mbar_wait(&full[lane * S::kRing + i % S::kRing], (i / S::kRing) & 1, a.err, 904);
        return;
    }

    RowState<NT> st;
    int used = 0;
    bool ok = true;
    do {
        load_rows<NT>(a, use.it, st, lane);
        const int min_lim = use.it.L - use.it.n + use.it.row0;  // last key of the block's first query row
        const int p1 = use.u1();
        for (int p = use.u0() + warp; p < p1; p += kWarps) {
            const int sg = warp * S::kRing + used % S::kRing;
            ok = ok && mbar_wait(&full[sg], (used / S::kRing) & 1, a.err, 904);
            const uint8_t* page = smem + sg * kKv8Bytes;
            if (__all_sync(0xffffffffu, ok)) {
                const uint32_t scale2 = stage_scales[sg];
                if (p * kPage + kPage - 1 > min_lim) attend_page8<NT, true>(page, scale2, st, p * kPage, min_lim, lane);
                else attend_page8<NT, false>(page, scale2, st, p * kPage, min_lim, lane);
            }
            fence_proxy_async();  // the page's reads ahead of the copy that overwrites it
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[sg]);
            ++used;
        }
        // ---------------- join the warps: unnormalised sums and (m, l) of each through shared memory
        const int g = lane >> 2, c = lane & 3;
        attending_barrier();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float l = st.l[t];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (c == 0) {
                join_ml[(warp * S::kRows + t * 8 + g) * 2] = st.m[t];
                join_ml[(warp * S::kRows + t * 8 + g) * 2 + 1] = l;
            }
#pragma unroll
            for (int v = 0; v < 8; ++v)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    join[(warp * S::kRows + t * 8 + 2 * c + (e & 1)) * kPitch + 4 * (g + 8 * (v >> 1)) + 2 * (v & 1) + (e >> 1)] = st.o[v][t][e];
        }
        attending_barrier();
        const int a0 = use.cta0(), a1 = use.cta1();
        // a CTA takes part in at most one item that it did not begin and one that it does not end
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (static_cast<int>(blockIdx.x) == a0);
        for (int i = tid; i < use.it.rows * group * (kHd / 4); i += kAttThreads) {
            const int m = i / (kHd / 4), d = i % (kHd / 4) * 4;
            float M = kNegInf;
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, join_ml[(w * S::kRows + m) * 2]);
            float l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = 0; w < kWarps; ++w) {
                const float ms = join_ml[(w * S::kRows + m) * 2];
                // a warp without a visible key has l = 0 (or NaN where a NaN was seen)
                const float f = ms == kNegInf ? 1.f : exp2_ftz(ms - M);
                const float4 x = *reinterpret_cast<const float4*>(join + (w * S::kRows + m) * kPitch + d);
                l += join_ml[(w * S::kRows + m) * 2 + 1] * f;
                o.x += x.x * f; o.y += x.y * f; o.z += x.z * f; o.w += x.w * f;
            }
            if (a0 == a1) {
                const float inv = l == 0.f ? 0.f : kKv8Unlift / l;
                *reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(use.it.q0 + use.it.row0 + m / group) * a.hq + use.it.h * group + m % group) * kHd + d) =
                    make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
            } else {
                *reinterpret_cast<float4*>(a.ws_o + (slot * S::kRows + m) * kHd + d) = o;
                if (d == 0) {
                    a.ws_ml[(slot * S::kRows + m) * 2] = M;
                    a.ws_ml[(slot * S::kRows + m) * 2 + 1] = l;
                }
            }
        }
    } while (use.next(a, per_block));
}

// ------------------------------------------------------------------ joining
// Partial sums of the items that CTAs share, in the CTAs' order. Block (b, y): the item that CTA b goes on with, if
// the CTA before it is the first; eight parts' loads in flight. A kernel of its own: where the last CTA of an item to
// arrive joined it, one request at 4k took 20.5 us for 18.0 and 256 rows at 8k 133 for 75.
// COLUMNS false (up to 16 rows, row after row): a lane per four dimensions, rows 4 y .. 4 y + 3, two warps a row or
// four where there are only two, each with its share of the parts, which add up through shared memory (one request
// at 4k is 37 parts of two rows: a warp per row took 3.6 us more; blocks of two rows cost 64 requests 1.2 us, as most
// items have few parts). COLUMNS true (four dimensions of all rows after each other): a lane per row, of 32 y ..
// 32 y + 31, four such columns a warp; with row after row 256 rows' stores took 18 us a part.
constexpr int kJoinWarps = 8;
constexpr int kJoinRows = 4;  // COLUMNS false

// Unnormalised sums over parts, relative to the maximum M.
struct JoinSum {
    float M, l;
    float4 o;
    __device__ __forceinline__ void scale(float f) {
        l *= f;
        o.x *= f; o.y *= f; o.z *= f; o.w *= f;
    }
    __device__ __forceinline__ void add(float f, float l1, const float4& x) {
        l += l1 * f;
        o.x += x.x * f; o.y += x.y * f; o.z += x.z * f; o.w += x.w * f;
    }
};

template <bool COLUMNS>
__global__ void __launch_bounds__(kJoinWarps * 32)
join_shared_kernel(const Kv8AttnArgs a, int slot_rows) {
    __shared__ JoinSum split_sums[COLUMNS ? 1 : kJoinWarps][32];
    pdl_wait();
    pdl_trigger();
    const Kv8Shared s = a.ws_shared[blockIdx.x + 1];
    if (s.last < s.first || s.first != static_cast<int>(blockIdx.x)) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = a.hq / a.hkv;
    const int row0 = blockIdx.y * (COLUMNS ? 32 : kJoinRows);
    if (row0 >= s.rows) return;
    const int at_once = s.rows - row0 > kJoinRows / 2 ? kJoinRows : kJoinRows / 2, step = COLUMNS ? 1 : kJoinWarps / at_once;
    const int split = COLUMNS ? 0 : warp / at_once;
    for (int turn = 0; turn < (COLUMNS ? kHd / 4 / kJoinWarps : 1); ++turn) {
        const int m = row0 + (COLUMNS ? lane : warp % at_once);
        const int column = COLUMNS ? turn * kJoinWarps + warp : lane;  // four dimensions
        if (COLUMNS && m >= s.rows) continue;
        const bool live = m < s.rows;
        const int64_t at = COLUMNS ? static_cast<int64_t>(column) * slot_rows + m : static_cast<int64_t>(m) * (kHd / 4) + column;
        JoinSum sum = {kNegInf, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
        for (int b0 = s.first + split; live && b0 <= s.last; b0 += 8 * step) {
            float2 ml[8];
            float4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int b = b0 + i * step;
                const int64_t slot = 2 * static_cast<int64_t>(b) + (b == s.first);
                ml[i] = b <= s.last ? __ldcg(reinterpret_cast<const float2*>(a.ws_ml) + slot * slot_rows + m) : make_float2(kNegInf, 0.f);
                x[i] = b <= s.last ? __ldcg(reinterpret_cast<const float4*>(a.ws_o) + slot * slot_rows * (kHd / 4) + at) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            float next = sum.M;
#pragma unroll
            for (int i = 0; i < 8; ++i) next = fmaxf(next, ml[i].x);
            sum.scale(sum.M == kNegInf ? 1.f : exp2_ftz(sum.M - next));
            sum.M = next;
            // a part without a visible key has l = 0 (or NaN where a NaN was seen)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum.add(ml[i].x == kNegInf ? 1.f : exp2_ftz(ml[i].x - next), ml[i].y, x[i]);
        }
        if (!COLUMNS) {
            split_sums[COLUMNS ? 0 : warp][lane] = sum;
            __syncthreads();
            if (split > 0) return;
            for (int i = 1; i < step; ++i) {
                const JoinSum& y = split_sums[COLUMNS ? 0 : i * at_once + warp][lane];
                const float next = fmaxf(sum.M, y.M);
                sum.scale(sum.M == kNegInf ? 1.f : exp2_ftz(sum.M - next));
                sum.add(y.M == kNegInf ? 1.f : exp2_ftz(y.M - next), y.l, y.o);
                sum.M = next;
            }
        }
        if (!live) continue;
        const float inv = sum.l == 0.f ? 0.f : kKv8Unlift / sum.l;
        *reinterpret_cast<uint2*>(a.out + ((s.q_row + m / group) * a.hq + s.h * group + m % group) * kHd + column * 4) =
            make_uint2(pack_bf16x2(sum.o.x * inv, sum.o.y * inv), pack_bf16x2(sum.o.z * inv, sum.o.w * inv));
    }
}

// ------------------------------------------------------------------ host side
// The form by the rows of a block: the query rows of a request x the heads of a group, as long as one block holds them all
// and so reads the keys once (32 requests over 4096 tokens, 32 / 8 heads: 8 rows 54 us, 16 rows 66, 20 rows, the
// first on tcgen05, 102 as up to 64; larger ones in kv8_tiles.cu).
// Workspace: what each CTA goes on with, then the partial sums of two items a CTA.
struct RowsPlan {
    int rows;  // of a block: MMA rows
    int grid;
    size_t off_o, off_ml, bytes;
};

RowsPlan plan_rows(int max_q_len, int hq, int hkv) {
    RowsPlan p{};
    const int64_t rows = static_cast<int64_t>(max_q_len) * (hq / hkv);
    p.rows = rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
    p.grid = 148 * (p.rows == 8 ? 2 : 1);
    p.off_o = (p.grid * sizeof(Kv8Shared) + 255) / 256 * 256;
    p.off_ml = p.off_o + static_cast<size_t>(p.grid) * 2 * p.rows * kHd * 4;
    p.bytes = p.off_ml + static_cast<size_t>(p.grid) * 2 * p.rows * 8;
    return p;
}

template <int NT>
int launch_rows(const Kv8AttnArgs& a, int grid, msgl_stream_t stream) {
    using S = RowsShape<NT>;
    static std::atomic<int> optin[kMaxDevices];
    const cudaError_t e = smem_optin(attend_rows_kernel<NT>, S::kSmem, optin);
    if (e != cudaSuccess) return set_error(MSGL_ERR_CUDA, cudaGetErrorString(e));
    launch_pdl(attend_rows_kernel<NT>, dim3(grid), dim3(kAttThreads + 32), S::kSmem, stream, a);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

int check_attend(int num_reqs, int total_q, int max_q_len, int max_seq_len, int hq, int hkv, int head_dim, int page_size) {
    if (head_dim != kHd) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "attention_kv8: head_dim must be 128");
    if (page_size != kPage) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "attention_kv8: page_size must be 16");
    if (num_reqs < 0 || total_q < 0 || max_q_len < 0 || max_seq_len < 0 || hq <= 0 || hkv <= 0 || hq % hkv)
        return set_error(MSGL_ERR_INVALID_ARG, "attention_kv8: bad sizes or Hq % Hkv != 0");
    const int group = hq / hkv;
    if (group > 8 || (group & (group - 1)))
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "attention_kv8: Hq / Hkv must be 1, 2, 4 or 8");
    if (num_reqs > 65535 || hkv > 1024 || total_q > 1 << 24)
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "attention_kv8: too many requests, heads or rows");
    return MSGL_OK;
}

}  // namespace
}  // namespace msgl

using namespace msgl;

extern "C" {

int msgl_qknorm_rope_store_kv8(const void* qkv, void* q_out, void* kv8, void* scales, int64_t num_pages,
                               const int* positions, const int* page_table, int max_pages, const int* seq_lens,
                               const int* q_indptr, int num_reqs, int max_q_len, const float* cos_sin_cache,
                               int max_position, const void* q_norm_w, const void* k_norm_w, int num_tokens,
                               int num_q_heads, int num_kv_heads, int head_dim, int page_size, float eps,
                               msgl_stream_t stream) {
    StoreArgs a = {};
    a.qkv = static_cast<const __nv_bfloat16*>(qkv);
    a.q_out = static_cast<__nv_bfloat16*>(q_out);
    a.kv8 = static_cast<uint8_t*>(kv8);
    a.scales = static_cast<uint8_t*>(scales);
    a.num_pages = num_pages;
    a.positions = positions;
    a.page_table = page_table;
    a.max_pages = max_pages;
    a.seq_lens = seq_lens;
    a.q_indptr = q_indptr;
    a.num_reqs = num_reqs;
    a.max_q_len = max_q_len;
    a.table = cos_sin_cache;
    a.max_position = max_position;
    a.qn = static_cast<const __nv_bfloat16*>(q_norm_w);
    a.kn = static_cast<const __nv_bfloat16*>(k_norm_w);
    a.num_tokens = num_tokens;
    a.hq = num_q_heads;
    a.hkv = num_kv_heads;
    a.eps = eps;
    return launch_store(a, head_dim, page_size, stream);
}

int msgl_qknorm_rope_store_kv8_partials(const float* parts, int nparts, void* q_out, void* kv8, void* scales,
                                        int64_t num_pages, const int* positions, const int* page_table,
                                        int max_pages, const int* seq_lens, const int* q_indptr, int num_reqs,
                                        int max_q_len, const float* cos_sin_cache, int max_position,
                                        const void* q_norm_w, const void* k_norm_w, int num_tokens,
                                        int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                                        float eps, msgl_stream_t stream) {
    if (!parts || nparts < 1 || nparts > 64)
        return set_error(MSGL_ERR_INVALID_ARG, "store_kv8_partials: parts / nparts in [1, 64]");
    StoreArgs a = {};
    a.parts = parts;
    a.nparts = nparts;
    a.q_out = static_cast<__nv_bfloat16*>(q_out);
    a.kv8 = static_cast<uint8_t*>(kv8);
    a.scales = static_cast<uint8_t*>(scales);
    a.num_pages = num_pages;
    a.positions = positions;
    a.page_table = page_table;
    a.max_pages = max_pages;
    a.seq_lens = seq_lens;
    a.q_indptr = q_indptr;
    a.num_reqs = num_reqs;
    a.max_q_len = max_q_len;
    a.table = cos_sin_cache;
    a.max_position = max_position;
    a.qn = static_cast<const __nv_bfloat16*>(q_norm_w);
    a.kn = static_cast<const __nv_bfloat16*>(k_norm_w);
    a.num_tokens = num_tokens;
    a.hq = num_q_heads;
    a.hkv = num_kv_heads;
    a.eps = eps;
    return launch_store(a, head_dim, page_size, stream);
}

size_t msgl_paged_attention_kv8_workspace_size(int max_q_len, int num_q_heads, int num_kv_heads) {
    if (max_q_len <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
        num_q_heads / num_kv_heads > 8)
        return 0;
    // the largest of the forms that this call or a smaller one may take
    const int group = num_q_heads / num_kv_heads;
    size_t most = plan_rows(max_q_len, num_q_heads, num_kv_heads).bytes;
    for (int rows : {8, 16, 64, 128})
        most = std::max(most, plan_rows(std::min(max_q_len, rows / group), num_q_heads, num_kv_heads).bytes);
    return most;
}

int msgl_paged_attention_kv8(const void* q, const void* kv8, const void* scales, int64_t num_pages,
                             const int* page_table, int max_pages, const int* seq_lens, const int* q_indptr,
                             int num_reqs, int total_q, int max_q_len, int max_seq_len, int num_q_heads,
                             int num_kv_heads, int head_dim, int page_size, float scale, void* out,
                             void* workspace, size_t workspace_bytes, msgl_stream_t stream) {
    int rc = check_attend(num_reqs, total_q, max_q_len, max_seq_len, num_q_heads, num_kv_heads, head_dim, page_size);
    if (rc) return rc;
    if (num_pages <= 0 || num_pages > INT32_MAX || max_pages <= 0 || max_seq_len > static_cast<int64_t>(max_pages) * kPage)
        return set_error(MSGL_ERR_INVALID_ARG, "attention_kv8: bad pool or page-table width");
    if (!q_indptr && (max_q_len != 1 || total_q != num_reqs))
        return set_error(MSGL_ERR_INVALID_ARG, "attention_kv8: one row per request without q_indptr");
    if (num_reqs == 0 || total_q == 0 || max_q_len == 0) return MSGL_OK;
    if (!q || !kv8 || !scales || !page_table || !seq_lens || !out)
        return set_error(MSGL_ERR_INVALID_ARG, "attention_kv8: null pointer");
    if (!aligned16(q) || !aligned16(kv8) || !aligned16(out) || (reinterpret_cast<uintptr_t>(scales) & 1))
        return set_error(MSGL_ERR_INVALID_ARG, "attention_kv8: q, kv8 and out must be 16-byte aligned, scales 2-byte");
    Kv8AttnArgs a = {};
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.kv8 = static_cast<const uint8_t*>(kv8);
    a.scales = static_cast<const uint8_t*>(scales);
    a.num_pages = num_pages;
    a.page_table = page_table;
    a.max_pages = max_pages;
    a.max_len = max_seq_len;
    a.seq_lens = seq_lens;
    a.q_indptr = q_indptr;
    a.num_reqs = num_reqs;
    a.total_q = total_q;
    a.max_q_len = std::min(max_q_len, total_q);
    a.hq = num_q_heads;
    a.hkv = num_kv_heads;
    a.sl2e = scale * 1.4426950408889634f;
    a.out = static_cast<__nv_bfloat16*>(out);
    const RowsPlan p = plan_rows(a.max_q_len, num_q_heads, num_kv_heads);
    if (!workspace || workspace_bytes < p.bytes || !aligned16(workspace))
        return set_error(MSGL_ERR_WORKSPACE, "attention_kv8: workspace missing, too small or not 16-byte aligned");
    a.err = device_error_word();
    if (!a.err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    a.ws_shared = reinterpret_cast<Kv8Shared*>(ws);
    a.ws_o = reinterpret_cast<float*>(ws + p.off_o);
    a.ws_ml = reinterpret_cast<float*>(ws + p.off_ml);
    a.min_units = p.rows <= 16 ? kWarps : 4;  // a page for each warp, or 256 keys
    rc = p.rows == 8 ? launch_rows<1>(a, p.grid, stream) : p.rows == 16 ? launch_rows<2>(a, p.grid, stream)
                                                          : launch_attend_tiles(a, p.rows, p.grid, stream);
    if (rc) return rc;
    const bool columns = p.rows > 16;
    launch_pdl(columns ? join_shared_kernel<true> : join_shared_kernel<false>, dim3(p.grid - 1, columns ? p.rows / 32 : p.rows / kJoinRows),
               dim3(kJoinWarps * 32), 0, stream, a, p.rows);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

}  // extern "C"
