// verify.cu -- probabilities of logits, and the verification of drafted tokens against them.
//
//  * msgl_token_probs    p = softmax(logits / temperature) per row, one-hot where greedy
//  * msgl_verify_drafts  speculative sampling (Leviathan, Kalman, Matias, "Fast inference from
//                        transformers via speculative decoding", ICML 2023): draft i with target
//                        probability p and draft probability q is accepted iff u q < p; the token behind
//                        the accepted ones is drawn from max(p - q, 0) of the first rejected draft's rows,
//                        or from the target's last row. With given uniform numbers nothing is random.
//
// Comparisons and running sums that decide a token are in 64 bits: of 150k borders in [0, 1), fp32 sums
// put one in thirty uniform numbers on the wrong side, 64-bit sums one in 10^9.
#include <algorithm>

#include "common.cuh"

namespace msgl {
namespace {

constexpr int kProbThreads = 512;
constexpr int kProbPart = 20480;  // values of a row that a CTA holds, at most (80 KB)
constexpr int kMaxCluster = 16;
constexpr float kNegInf = -__builtin_huge_valf();

__device__ __forceinline__ double ld_dsmem_f64(uint32_t addr) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
    return v;
}

// Larger float -> larger key, NaN above all; then the smaller index.
__device__ __forceinline__ unsigned long long argmax_key(float v, uint32_t i) {
    const uint32_t u = v != v ? 0x7fffffffu : __float_as_uint(v);
    const uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return (static_cast<unsigned long long>(k) << 32) | (0xffffffffu - i);
}

// ------------------------------------------------------------------ probabilities
// A row is read once and written once: a cluster's CTAs hold it in shared memory, each takes the maximum and the sum
// of its own part, and one exchange through distributed shared memory joins them:
// p = exp(x - m_thread) * (exp(m_thread - m) / sum). HBM bound; up to three CTAs an SM, so that one's loads run while
// the others reduce, exchange and store. 320 rows of 151936: 88 us, 4.4 TB/s. The parts in registers: 97 us with two
// CTAs an SM, 137 with one; clusters that walk the rows with the next row's loads in flight (one CTA an SM, and 15
// clusters of 8 are all that the GPU holds then) 122; clusters of 16: 165.
template <int VEC>
__device__ __forceinline__ void copy_async(float* dst, const float* src) {
    if (VEC == 4) cp_async16(smem_u32(dst), src, true);
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
template <int VEC>
__device__ __forceinline__ void read_part(const float* src, float (&v)[VEC]) {
    if (VEC == 4) {
        const float4 f = *reinterpret_cast<const float4*>(src);
        v[0] = f.x; v[1 % VEC] = f.y; v[2 % VEC] = f.z; v[3 % VEC] = f.w;
    } else {
        v[0] = *src;
    }
}
// Maximum m and sum s = sum exp2((x - m) c) of a warp's 32 such pairs, in every lane.
__device__ __forceinline__ void join_pairs(float& m, float& s, float c) {
    const float all = warp_max(m);
    s = warp_sum(m == kNegInf ? s : s * exp2_ftz((m - all) * c));
    m = all;
}

template <int VEC>
__device__ __forceinline__ void write_part(float* dst, const float (&v)[VEC]) {
    if (VEC == 4) *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1 % VEC], v[2 % VEC], v[3 % VEC]);
    else *dst = v[0];
}

template <int VEC>
__global__ void __launch_bounds__(kProbThreads, 3)
token_probs_kernel(const float* logits, int64_t ldx, const float* __restrict__ temperature, float* probs,
                   int64_t ldp, int vocab, int part) {
    extern __shared__ __align__(16) float here[];
    __shared__ float2 red[kProbThreads / 32];
    __shared__ float2 mine;  // the CTA's maximum and sum, read by the cluster
    __shared__ unsigned long long red_key[kProbThreads / 32], mine_key;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = cluster_ctarank(), size = cluster_nctarank();
    const int begin = rank * part, count = min(vocab, begin + part) - begin;  // a multiple of VEC but for the row's end
    pdl_wait();
    pdl_trigger();
    const int64_t row = cluster_id_x();
    const float* x = logits + row * ldx + begin;
    float* p = probs + row * ldp + begin;
    // all loads in flight together; a thread works on what it loaded
    for (int i = tid * VEC; i < count; i += kProbThreads * VEC) copy_async<VEC>(here + i, x + i);
    cp_async_commit();
    const float T = temperature ? temperature[row] : 1.f;
    cp_async_wait<0>();
    if (T <= 0.f) {  // the whole cluster
        unsigned long long best = 0;
        for (int k = tid * VEC; k < count; k += kProbThreads * VEC)
            for (int i = k; i < k + VEC; ++i) {
                const unsigned long long key = argmax_key(here[i], begin + i);
                best = key > best ? key : best;
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long y = __shfl_xor_sync(0xffffffffu, best, o);
            best = y > best ? y : best;
        }
        if (lane == 0) red_key[warp] = best;
        __syncthreads();
        for (int w = 0; w < kProbThreads / 32; ++w) best = red_key[w] > best ? red_key[w] : best;
        if (tid == 0) mine_key = best;
        cluster_sync_all();
        for (int q = 0; q < size; ++q) {
            const unsigned long long y = __double_as_longlong(ld_dsmem_f64(mapa_shared(smem_u32(&mine_key), q)));
            best = y > best ? y : best;
        }
        cluster_arrive();
        const int top = static_cast<int>(0xffffffffu - static_cast<uint32_t>(best)) - begin;
        for (int k = tid * VEC; k < count; k += kProbThreads * VEC)
            for (int i = k; i < k + VEC; ++i) p[i] = i == top ? 1.f : 0.f;
        cluster_wait();  // no CTA leaves while its shared memory may be read
        return;
    }
    const float factor = 1.4426950408889634f / T, c = factor > 3.0e38f ? 3.0e38f : factor;  // (NaN stays)
    // Each thread against its own maximum: one reduction of (maximum, sum) pairs, and exponentials ahead of it.
    float own = kNegInf;
#pragma unroll 4
    for (int i = tid * VEC; i < count; i += kProbThreads * VEC) {
        float v[VEC];
        read_part<VEC>(here + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) own = fmaxf(own, v[e]);
    }
    const float base = own == kNegInf ? 0.f : own;  // values without a finite one add nothing (NaN still does)
    float s0 = 0.f, s1 = 0.f;
#pragma unroll 4
    for (int i = tid * VEC; i < count; i += kProbThreads * VEC) {
        float v[VEC];
        read_part<VEC>(here + i, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            v[e] = exp2_ftz((v[e] - base) * c);
            (e & 1 ? s1 : s0) += v[e];
        }
        write_part<VEC>(here + i, v);
    }
    float m = own, s = s0 + s1;
    join_pairs(m, s, c);
    if (lane == 0) red[warp] = make_float2(m, s);
    __syncthreads();
    m = lane < kProbThreads / 32 ? red[lane].x : kNegInf;
    s = lane < kProbThreads / 32 ? red[lane].y : 0.f;
    join_pairs(m, s, c);
    if (tid == 0) mine = make_float2(m, s);
    cluster_sync_all();
    m = kNegInf;  // lane q: CTA q's maximum and sum
    s = 0.f;
    if (lane < size) {
        m = ld_dsmem_f32(mapa_shared(smem_u32(&mine.x), lane));
        s = ld_dsmem_f32(mapa_shared(smem_u32(&mine.y), lane));
    }
    cluster_arrive();  // this CTA's peers are read; waited for at the end
    join_pairs(m, s, c);
    // a row without any logit above -inf: S = 0, zeros (S is NaN where a logit is NaN or +inf)
    const float f = s == 0.f ? 0.f : (own == kNegInf ? 1.f : exp2_ftz((own - m) * c)) / s;
#pragma unroll 4
    for (int i = tid * VEC; i < count; i += kProbThreads * VEC) {
        float v[VEC];
        read_part<VEC>(here + i, v);
        if (VEC == 4) __stcs(reinterpret_cast<float4*>(p + i), make_float4(v[0] * f, v[1 % VEC] * f, v[2 % VEC] * f, v[3 % VEC] * f));
        else __stcs(p + i, v[0] * f);
    }
    cluster_wait();  // no CTA leaves while its shared memory may be read
}

// ------------------------------------------------------------------ verification
// One cluster per request. Every CTA finds the first rejected draft (two loads a draft) and takes one
// range of the vocabulary of that draft's rows; its warps take consecutive parts of the range and sum
// their weights. One exchange of the CTAs' sums gives every CTA the total and what lies before it; the
// warp whose part holds u * total walks that part again, 128 values at a time. HBM bound for many
// requests, a chain of four latencies (drafts, rows, exchange, walk) for one.
constexpr int kVerThreads = 512;
constexpr int kVerWarps = kVerThreads / 32;

struct VerifyArgs {
    const float* p;
    int64_t ldp;
    const float* q;  // null: draft i has probability 1 for its token
    int64_t ldq;
    const int *drafts, *indptr;
    const float *u, *u_last;
    int num_drafts, max_drafts, vocab, part;
    int *accepted, *tokens;
    int* err;
};

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Weight of a token: p - q where positive (NaN: none).
__device__ __forceinline__ double rest_of(float p, float q) {
    const double w = static_cast<double>(p) - static_cast<double>(q);
    return w > 0.0 ? w : 0.0;
}

template <int VEC>
__device__ __forceinline__ void load_values(const float* row, int i, int end, float (&v)[4]) {
    if (VEC == 4) {
        const float4 f = i < end ? __ldg(reinterpret_cast<const float4*>(row + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = i + e < end ? __ldg(row + i + e) : 0.f;
    }
}

template <int VEC>
__global__ void __launch_bounds__(kVerThreads)
verify_drafts_kernel(const VerifyArgs a) {
    __shared__ double parts[kVerWarps];
    __shared__ __align__(8) double mine[2];  // sum of this CTA's weights, in either turn
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = cluster_ctarank(), size = cluster_nctarank();
    pdl_wait();
    pdl_trigger();
    const int r = cluster_id_x();
    const int d0 = a.indptr[r], k = a.indptr[r + 1] - d0;
    int* out = a.tokens + static_cast<int64_t>(r) * (a.max_drafts + 1);
    if (d0 < 0 || k < 0 || k > a.max_drafts || d0 > a.num_drafts - k) {  // the same for the whole cluster
        if (rank == 0) {
            for (int i = tid; i <= a.max_drafts; i += kVerThreads) out[i] = -1;
            if (tid == 0) {
                a.accepted[r] = 0;
                record_error(a.err, MSGL_ERR_BOUNDS, 920);
            }
        }
        return;
    }
    const float* p0 = a.p + (static_cast<int64_t>(d0) + r) * a.ldp;
    // the first rejected draft, by every warp for itself
    int n = k;
    for (int b = 0; b < k && n == k; b += 32) {
        const int i = b + lane;
        bool rejected = false;
        if (i < k) {
            const int x = a.drafts[d0 + i];
            rejected = true;
            if (x >= 0 && x < a.vocab) {
                const float px = __ldg(p0 + i * a.ldp + x);
                const float qx = a.q ? __ldg(a.q + (static_cast<int64_t>(d0) + i) * a.ldq + x) : 1.f;
                rejected = !(static_cast<double>(a.u[d0 + i]) * static_cast<double>(qx) < static_cast<double>(px));
            } else if (rank == 0 && warp == 0) {
                record_error(a.err, MSGL_ERR_BOUNDS, 921);
            }
        }
        const uint32_t any = __ballot_sync(0xffffffffu, rejected);
        if (any) n = b + __ffs(any) - 1;
    }
    const float* prow = p0 + n * a.ldp;
    const float* qrow = n < k && a.q ? a.q + (static_cast<int64_t>(d0) + n) * a.ldq : nullptr;
    const int point = n < k && !a.q ? a.drafts[d0 + n] : -1;  // weight of this token: p - 1 <= 0
    // this warp's part of the CTA's range
    const int begin = min(a.vocab, rank * a.part), end = min(a.vocab, begin + a.part);
    const int share = (a.part / 128 + kVerWarps - 1) / kVerWarps * 128;
    const int w0 = min(end, begin + warp * share), w1 = min(end, w0 + share);
    // sum of the weights of [w0, w1), the warp's; FALL: of the target's row alone
    auto weigh = [&](bool fall) {
        double sum = 0.0;
#pragma unroll 4
        for (int i = w0 + lane * 4; i < w1; i += 128) {
            float pv[4], qv[4] = {0.f, 0.f, 0.f, 0.f};
            load_values<VEC>(prow, i, w1, pv);
            if (qrow && !fall) load_values<VEC>(qrow, i, w1, qv);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (i + e == point && !fall) qv[e] = 1.f;
                sum += rest_of(pv[e], qv[e]);
            }
        }
        return warp_sum64(sum);
    };
    double total = 0.0, before = 0.0, here = 0.0;
    int last_part = -1;  // last CTA with any weight
    bool fall = false;
    for (int turn = 0; turn < 2; ++turn) {  // where p <= q everywhere (rounding), once more over the target's own row
        fall = turn == 1;
        const double sum = weigh(fall);
        if (lane == 0) parts[warp] = sum;
        __syncthreads();
        if (tid == 0) {
            double s = 0.0;
            for (int w = 0; w < kVerWarps; ++w) s += parts[w];
            mine[turn] = s;
        }
        cluster_sync_all();
        total = 0.0;
        for (int c = 0; c < size; ++c) {
            const double s = ld_dsmem_f64(mapa_shared(smem_u32(&mine[turn]), c));
            if (c == rank) {
                before = total;
                here = s;
            }
            total += s;
            if (s > 0.0) last_part = c;
        }
        if (total > 0.0 || (!qrow && point < 0)) break;
    }
    cluster_arrive();
    const bool fine = total > 0.0 && total < __longlong_as_double(0x7ff0000000000000ll);
    double goal = static_cast<double>(a.u_last[r]) * total;
    if (!(goal >= 0.0)) goal = 0.0;
    if (rank == 0) {
        for (int i = tid; i <= a.max_drafts; i += kVerThreads)
            if (i != n || !fine) out[i] = i < n ? a.drafts[d0 + i] : -1;
        if (tid == 0) {
            a.accepted[r] = n;
            if (!fine) record_error(a.err, MSGL_ERR_BOUNDS, 922);
        }
    }
    // The first place whose running sum passes the goal lies in this CTA (in the last one with any
    // weight where u is 1 or more).
    const bool holds = here > 0.0 && before <= goal && (goal < before + here || rank == last_part);
    if (fine && holds) {
        double sum = before;
        int pick = -1, last = -1;
        for (int w = 0; w < kVerWarps; ++w) {
            if (parts[w] > 0.0) last = w;
            if (pick < 0 && goal < sum + parts[w]) pick = w;
            if (pick < 0) sum += parts[w];
        }
        if (pick < 0) {  // the sums over warps and over CTAs round differently
            pick = last;
            sum -= parts[last];
        }
        if (warp == pick) {
            int found = -1, weighty = -1;  // weighty: the last token with any weight
            for (int b = w0; b < w1 && found < 0; b += 128) {
                const int i = b + lane * 4;
                float pv[4], qv[4] = {0.f, 0.f, 0.f, 0.f};
                load_values<VEC>(prow, i, w1, pv);
                if (qrow && !fall) load_values<VEC>(qrow, i, w1, qv);
                double wv[4], own = 0.0;
                int mine_last = -1;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (i + e == point && !fall) qv[e] = 1.f;
                    wv[e] = rest_of(pv[e], qv[e]);
                    own += wv[e];
                    if (wv[e] > 0.0) mine_last = i + e;
                }
                double upto = own;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += y;
                }
                weighty = max(weighty, __reduce_max_sync(0xffffffffu, mine_last));
                const uint32_t passed = __ballot_sync(0xffffffffu, own > 0.0 && goal < sum + upto);
                if (passed) {
                    const int lead = __ffs(passed) - 1;
                    int at = -1;
                    double c = sum + upto - own;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        c += wv[e];
                        if (at < 0 && wv[e] > 0.0 && goal < c) at = i + e;
                    }
                    if (at < 0) at = mine_last;
                    found = __shfl_sync(0xffffffffu, at, lead);
                }
                sum += __shfl_sync(0xffffffffu, upto, 31);
            }
            if (lane == 0) out[n] = found >= 0 ? found : weighty;
        }
    }
    cluster_wait();
}

// CTAs of a row or request: a power of two, enough for `fit`, doubled while the GPU has room; 16 only where all of them
// run at once: they find places more slowly (16 rows of probabilities 10.3 us as clusters of 8, 13.0 of 16; but 4 rows 10.0
// and 7.2, one request's verification 11.5 and 7.5).
int cluster_size(int64_t rows, int fit) {
    int c = 1;
    while (c < fit) c *= 2;
    while (c < kMaxCluster && rows * c < 148 && (c < 8 || rows * 16 <= 148)) c *= 2;
    return c;
}

template <typename... K>
cudaError_t allow_large_clusters(void (*kernel)(K...), std::atomic<int> (&done)[kMaxDevices]) {
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const auto set = [&](int want) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, want);
    };
    if (dev < 0 || dev >= kMaxDevices) return set(1);
    return raise_limit(done[dev], 1, set);
}

}  // namespace
}  // namespace msgl

using namespace msgl;

extern "C" {

int msgl_token_probs(const float* logits, int64_t ldx, int num_rows, int vocab, const float* temperature,
                     float* probs, int64_t ldp, msgl_stream_t stream) {
    if (num_rows < 0 || vocab <= 0 || ldx < vocab || ldp < vocab)
        return set_error(MSGL_ERR_INVALID_ARG, "token_probs: bad sizes");
    constexpr int kPer = kProbPart;
    if (vocab > kPer * kMaxCluster)
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "token_probs: vocab above 327680");
    if (num_rows > INT32_MAX / kMaxCluster) return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "token_probs: too many rows");
    if (num_rows == 0) return MSGL_OK;
    if (!logits || !probs) return set_error(MSGL_ERR_INVALID_ARG, "token_probs: null pointer");
    if (logits == probs && ldx != ldp) return set_error(MSGL_ERR_INVALID_ARG, "token_probs: in place with another stride");
    const bool vec = vocab % 4 == 0 && ldx % 4 == 0 && ldp % 4 == 0 && aligned16(logits) && aligned16(probs);
    const int size = cluster_size(num_rows, (vocab + kPer - 1) / kPer);
    const int part = ((vocab + size - 1) / size + 3) / 4 * 4;
    const auto kernel = vec ? token_probs_kernel<4> : token_probs_kernel<1>;
    static std::atomic<int> large[2][kMaxDevices], room[2][kMaxDevices];
    cudaError_t e = smem_optin(kernel, kPer * sizeof(float), room[vec]);
    if (e == cudaSuccess && size > 8) e = allow_large_clusters(kernel, large[vec]);
    if (e != cudaSuccess) return set_error(MSGL_ERR_CUDA, cudaGetErrorString(e));
    launch_cluster(kernel, static_cast<int64_t>(num_rows) * size, kProbThreads, size, part * sizeof(float), stream, logits, ldx,
                   temperature, probs, ldp, vocab, part);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

int msgl_verify_drafts(const float* target_probs, int64_t ldp, const float* draft_probs, int64_t ldq,
                       const int* draft_tokens, const int* draft_indptr, const float* uniforms,
                       const float* last_uniforms, int num_reqs, int num_drafts, int max_drafts, int vocab,
                       int* accepted, int* tokens, msgl_stream_t stream) {
    if (num_reqs < 0 || num_drafts < 0 || max_drafts < 0 || vocab <= 0 || ldp < vocab || (draft_probs && ldq < vocab))
        return set_error(MSGL_ERR_INVALID_ARG, "verify_drafts: bad sizes");
    if (vocab > 1 << 30 || num_reqs > INT32_MAX / kMaxCluster || max_drafts > 1 << 20)
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "verify_drafts: too many requests, drafts or tokens");
    if (num_reqs == 0) return MSGL_OK;
    if (!target_probs || !draft_indptr || !last_uniforms || !accepted || !tokens ||
        (num_drafts > 0 && (!draft_tokens || !uniforms)))
        return set_error(MSGL_ERR_INVALID_ARG, "verify_drafts: null pointer");
    const bool vec = vocab % 4 == 0 && ldp % 4 == 0 && aligned16(target_probs) &&
                     (!draft_probs || (ldq % 4 == 0 && aligned16(draft_probs)));
    // four at least, for an even load of many requests: 256 81 us, with one each 107, with eight 99
    const int size = cluster_size(num_reqs, 4);
    const int part = ((vocab + size - 1) / size + 127) / 128 * 128;
    static std::atomic<int> large4[kMaxDevices], large1[kMaxDevices];
    const cudaError_t e = size <= 8 ? cudaSuccess
                          : vec ? allow_large_clusters(verify_drafts_kernel<4>, large4)
                                : allow_large_clusters(verify_drafts_kernel<1>, large1);
    if (e != cudaSuccess) return set_error(MSGL_ERR_CUDA, cudaGetErrorString(e));
    const VerifyArgs a = {target_probs, ldp, draft_probs, ldq, draft_tokens, draft_indptr, uniforms, last_uniforms,
                          num_drafts, max_drafts, vocab, part, accepted, tokens, device_error_word()};
    if (!a.err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    launch_cluster(vec ? verify_drafts_kernel<4> : verify_drafts_kernel<1>, static_cast<int64_t>(num_reqs) * size,
                   kVerThreads, size, 0, stream, a);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

}  // extern "C"
