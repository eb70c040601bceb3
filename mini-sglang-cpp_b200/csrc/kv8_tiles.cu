// kv8_tiles.cu -- attention of many rows (chunks, drafted rows) over the 8-bit key / value pool, on tcgen05.
//
// Persistent: each CTA takes an equal part of the steps (64 keys) of all items (block of query rows x kv head;
// rows = query rows x the group's heads); of items shared by CTAs they leave partial sums. Codes are converted to
// f16 (exactly) into the operands' canonical tiles, q is scaled to f16 by a power of two per row (kv8.cuh). A page's scales enter the exponent: s = (q . k) 2^(q + k exponents) scale log2(e) + (exponent of v),
// p = 2^(s - m + 11) in f16 (kv8.cuh), so that O needs no scaling by page, and l adds p 2^-(11 + exponent of v).
//
// Two streams of up to 128 MMA rows each:
//   FEW = false  blocks of 256 rows: the streams are its halves, and both take every step;
//   FEW = true   blocks of up to 128 rows: both streams hold them and take every other step, joined at the
//                item's end, so that one's softmax runs while the other's MMAs do.
// Warps (those of 64 rows in brackets):
//   0-3, 4-7   [0, 1, 6, 7] softmax of stream 0 / 1: a thread per row. S from tensor memory, p as f16 pairs over the
//              first half of S, l and m in registers; O in tensor memory is rescaled only where the maximum grew by
//              more than 4;
//   8, 9       [2, 3 of stream 0, 8, 9 of stream 1] conversion of a step's keys to [64][128],
//   10, 11     [4, 5; 10, 11] of its values to [128][64], both K-major (the keys of a page in the order in which the
//              pool stores their values);
//   12, 13     one lane each issues a stream's MMAs: PV(i), then S(i + 2). S has two buffers of 64 columns, so that
//              the next S is there before the softmax of a step ends; while one stream waits for a hand-over
//              (100 to 400 clocks each) the other's MMAs run;
//   14         page ids and scales, a bulk copy of 4 KB a page into a ring of two steps [two of each stream] (loads by
//              the converting warps held them up for half of their time).
// Tensor memory: two S buffers a stream and O: 2 x (128 + 128) columns.
//
// Bound: chunks by the softmax, whose two warps a scheduler take 1560 clocks a step (1024 of them exponentials) of
// 2500, ahead of the MMAs' 1024; few rows by the chain from a step's copy over its conversion to its softmax, 1500
// clocks a step where HBM would allow 700. Measured: two chunks of 2048 rows over 6k to 8k tokens, 32 / 8 heads, 417 to 424
// us (905 to 920 TFLOP/s); 24 requests x 6 rows over 5k to 20k tokens, 32 / 4 heads, 107 us (3.0 TB/s).
#include <algorithm>

#include "kv8.cuh"

namespace msgl {
namespace {

constexpr int kPage = kKv8Page;
constexpr int kHd = kKv8Head;
constexpr int kStep = 64;                      // keys
constexpr int kPages = kStep / kPage;          // of a step
constexpr int kRows = 128;                     // of a stream
constexpr int kKTile = 2 * kStep * 128;        // [2 halves of the dimensions][64 keys][64 f16]
constexpr int kVTile = kHd * 128;              // [128 dimensions][64 keys f16]
constexpr int kItems = 16;  // items whose NaN are kept; the copies are ahead by fewer than ten (of one step each)
constexpr int kThreads = 512;

// The forms by the rows of a block. 256: the streams are its halves, and both take every step. 128, 64: both streams
// hold the block and take every other step, joined at the item's end, so that one's softmax runs while the
// other's MMAs do. With 64 rows half of the softmax warps would have none: they convert, a team for each stream (one
// team of eight warps took as long for a step as four for their own: 24 requests x 48 rows 18% less time with
// eight in place of four, 10% less again as two teams). 32 requests over 4096 tokens: 64 rows 104 us, 68 (as 128) 126,
// 128 rows 135, 132 (as 256) 169, 256 rows 182.
template <int ROWS>
struct Form {
    static constexpr bool kFew = ROWS <= 128;
    static constexpr int kSoftmaxWarps = ROWS == 64 ? 2 : 4;    // of a stream
    static constexpr int kConvertWarps = 2;                     // of keys, and as many of values
    static constexpr int kTeams = ROWS == 64 ? 2 : 1;           // of them: one, or one for each stream
    static constexpr int kStages = 4;                           // of keys and of values
    static constexpr int kRaw = ROWS == 64 ? 4 : 2;             // steps of codes
    // Steps whose scales are kept: more than the copies are ahead of a softmax (by the slots of codes, the stages and two).
    static constexpr int kInfo = ROWS == 64 ? 16 : 8;
    static constexpr int kQHalf = (ROWS == 64 ? 64 : kRows) * 128;  // 64 dimensions of a tile of Q: [rows][64 f16]
    static constexpr int kQTiles = ROWS == 64 ? 1 : 2;
    static constexpr int kQ = 2 * kQTiles * kQHalf;
    static constexpr size_t kSmem = 1024 + kQ + kStages * (kKTile + kVTile) + kRaw * kPages * kKv8Bytes;
    static constexpr int kJoinDims = kQ / 4 / ROWS < kHd ? kQ / 4 / ROWS : kHd;  // of stream 1's sums that the place of Q holds
    // Stages of keys and values. Few rows: two for each stream, so that a stream meets every phase of its barriers (one
    // that skipped a phase would take the one before for it); else all for both. n: steps taken before.
    __device__ static int stage(int t, int n) { return kFew ? 2 * t + n % 2 : n % kStages; }
    __device__ static int use(int n) { return kFew ? n / 2 : n / kStages; }
    // Slots of codes: of each team its own, for the same reason.
    __device__ static int slot(int t, int n) { return kTeams == 2 ? 2 * t + n % 2 : n % 2; }
};
constexpr float kNegInf = -__builtin_huge_valf();

__host__ __device__ constexpr uint32_t idesc_f16(int M, int N) {  // A, B f16 K-major, D fp32
    return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ bool elect_lane() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ void named_barrier(int id, int threads) {
    __syncwarp();
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Waits of a whole warp: even lanes for the use-th completion of a, odd ones for that of b. A vote orders no memory:
// the warp barrier behind it is what lets each lane see what the other half waited for.
__device__ __forceinline__ bool wait_two(uint64_t* a, int use_a, uint64_t* b, int use_b, int* err, int site) {
    const bool odd = threadIdx.x & 1;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(odd ? b : a, (odd ? use_b : use_a) & 1, err, site));
    __syncwarp();
    return ok;
}
__device__ __forceinline__ bool wait_one(uint64_t* a, int use, int* err, int site) {
    return __all_sync(0xffffffffu, mbar_wait(a, use & 1, err, site));
}

// Scales of a page: keys' factor, values' exponent and inverse factor (of 2^-11 p).
struct PageScale {
    float k, v_exp, v_inv, pad;
};

template <int ROWS>
struct Shared {
    uint64_t raw_full[Form<ROWS>::kRaw], raw_empty[Form<ROWS>::kRaw], k_full[4], k_empty[4], v_full[4], v_empty[4];
    uint64_t q_full[2], s_full[2][2], p_full[2][2], o_done[2][2];  // stream, parity of its steps
    PageScale info[Form<ROWS>::kInfo][kPages];
    int nan_seen[kItems];  // by item in turn: a value hidden from some of its rows was NaN
    uint32_t tmem;
    union {
        Kv8Scan<kThreads> scan;  // before the walk
        float2 ml[Form<ROWS>::kFew ? ROWS : 1];  // stream 1's (m, l)
    };
};

// Two fp32 values in a register pair.
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
    return v;
}
__device__ __forceinline__ uint64_t pair(float v) { return pair(__float_as_uint(v), __float_as_uint(v)); }
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// One step of a row: 64 S columns into pairs of p. EDGE: keys behind `lim` do not count. The factor of a page
// is positive, so the page's largest logit comes from its largest product, and a masked one stays -inf: where the scales'
// product underflows (a row of zeros over keys of zeros, scale 0) it is the smallest normal number in its place, which
// makes logits of at most 2^-109 of the products.
template <bool EDGE>
__device__ __forceinline__ void softmax_step(uint32_t (&s)[64], uint32_t (&out)[32], const PageScale* info, float qs, int key0,
                                             int lim, float& m, float& l, float& alpha) {
    float f[kPages], v_exp[kPages], v_inv[kPages], mx[kPages];
#pragma unroll
    for (int p = 0; p < kPages; ++p) {
        const float4 sc = *reinterpret_cast<const float4*>(&info[p]);
        f[p] = fmaxf(qs * sc.x, 0x1p-126f);
        v_exp[p] = sc.y;
        v_inv[p] = sc.z;
        float x[kPage];
#pragma unroll
        for (int i = 0; i < kPage; ++i) {
            if (EDGE && key0 + p * kPage + token_at(i) > lim) s[p * kPage + i] = 0xff800000u;
            x[i] = __uint_as_float(s[p * kPage + i]);
        }
        const float a = max3(x[0], x[1], x[2]), b = max3(x[3], x[4], x[5]), c = max3(x[6], x[7], x[8]);
        const float d = max3(x[9], x[10], x[11]), e = max3(x[12], x[13], x[14]);
        mx[p] = __fmaf_ru(fmaxf(max3(a, b, c), max3(d, e, x[15])), f[p], v_exp[p]);
    }
    const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
    const float next = kv8_grows(top, m) ? fmaxf(m, top) : m;
    const float base = kv8_base(next);
    alpha = next == m ? 1.f : exp2_ftz(m - next);
    // Of each turn: the sums and f16 of the page before, this page's exponentials, the next one's exponents. The warp barrier
    // keeps the turns apart for the compiler (chunks 2% less).
    float sum = 0.f;
    uint64_t z[8], e[8];
#pragma unroll
    for (int k = -1; k <= kPages; ++k) {
        if (k >= 1) {  // the page before
            const int p = k - 1;
            uint64_t part[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float a, b;
                part[i & 1] = add2(part[i & 1], e[i]);
                unpair(e[i], a, b);
                out[p * 8 + i] = pack_half2(a, b);
            }
            float a, b;
            unpair(add2(part[0], part[1]), a, b);
            sum = fmaf(a + b, v_inv[p], sum);
        }
        if (k >= 0 && k < kPages) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float x, y;
                unpair(z[i], x, y);
                x = exp2_ftz(x);
                y = exp2_ftz(y);
                e[i] = pair(__float_as_uint(x), __float_as_uint(y));
            }
        }
        if (k + 1 < kPages) {
            const int p = k + 1;
            const uint64_t f2 = pair(f[p]), v2 = pair(__fsub_rd(v_exp[p], base));
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = fma2(pair(s[p * 16 + 2 * i], s[p * 16 + 2 * i + 1]), f2, v2);
        }
        __syncwarp();
    }
    l = fmaf(l, alpha, sum);
    m = next;
}

// Waits for the loads that write r: no use of r moves ahead of it.
template <int N>
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[N]) {
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < N; ++e) asm volatile("" : "+r"(r[e]));
}

// 32 consecutive columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    __syncwarp();
    uint32_t lo[16], hi[16];
    tmem_ld16(taddr, lo);
    tmem_ld16(taddr + 16, hi);
    tmem_loaded(lo);
    tmem_loaded(hi);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        r[e] = lo[e];
        r[16 + e] = hi[e];
    }
}

// Of an item, in steps (Q loaded, the pipeline filled and emptied, sums stored): four prompts of 2048 328 us with 3, 234 with
// 6, 222 with 10.
constexpr int kItemCost = 10;
using Walk = Kv8Walk<kStep, kItemCost>;

// A CTA's steps of an item: [u0, u1) of its units. Of them, a stream's own ones are first, first + stride, ...
template <bool FEW>
struct Share {
    int u0, u1;
    __device__ __forceinline__ explicit Share(const Walk& w) : u0(w.u0()), u1(w.u1()) {}
    // number of stream t's steps
    __device__ __forceinline__ int own(const Kv8Item& it, int per_stream, int t) const {
        if (FEW) return (u1 - u0 + 1 - t) / 2;
        return max(0, min(u1, kv8_units<kStep>(it.L, it.n, it.row0 + t * per_stream, min(per_stream, it.rows - t * per_stream))) - u0);
    }
    __device__ __forceinline__ int step(int t, int i) const { return FEW ? u0 + t + 2 * i : u0 + i; }
};

template <int ROWS>
__global__ void __launch_bounds__(kThreads, 1)
attend_tiles_kernel(const Kv8AttnArgs a) {
    using F = Form<ROWS>;
    constexpr bool FEW = F::kFew;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Shared<ROWS> sh;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sK = smem;                             // [kStages]
    uint8_t* sQ = sK + F::kStages * kKTile;         // a tile per stream, or one; FEW: stream 1's sums between two items
    uint8_t* sV = sQ + F::kQ;                       // [kStages]
    uint8_t* sRaw = sV + F::kStages * kVTile;       // [kRaw][kPages]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.hq / a.hkv, per_block = ROWS / group, per_stream = FEW ? per_block : per_block / 2;
    if (tid == 0) {
        for (int i = 0; i < F::kRaw; ++i) {
            mbar_init(&sh.raw_full[i], 1);
            mbar_init(&sh.raw_empty[i], 2 * F::kConvertWarps);
        }
        for (int i = 0; i < F::kStages; ++i) {
            mbar_init(&sh.k_full[i], F::kConvertWarps);
            mbar_init(&sh.k_empty[i], FEW ? 1 : 2);
            mbar_init(&sh.v_full[i], F::kConvertWarps);
            mbar_init(&sh.v_empty[i], FEW ? 1 : 2);
        }
        for (int i = 0; i < kItems; ++i) sh.nan_seen[i] = 0;
        for (int t = 0; t < 2; ++t) {
            mbar_init(&sh.q_full[t], F::kSoftmaxWarps);
            for (int b = 0; b < 2; ++b) {
                mbar_init(&sh.s_full[t][b], 1);
                mbar_init(&sh.p_full[t][b], F::kSoftmaxWarps);
                mbar_init(&sh.o_done[t][b], 1);
            }
        }
        fence_barrier_init();
    }
    pdl_wait();
    pdl_trigger();
    Walk walk;
    if (!kv8_part(a, per_block, sh.scan, walk)) return;
    if (warp == 12) {
        tmem_alloc(&sh.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    // Every role walks the CTA's items by itself: `count` steps of the items before this one, the `item`-th item.
    int count = 0, item = 0;
    bool ok = true;

    constexpr int kSoftmaxThreads = 2 * F::kSoftmaxWarps * 32;
    if (warp < 8 && (ROWS > 64 || warp < 2 || warp > 5)) {
        // ---------------- softmax of stream t: a thread per row
        const int t = warp >> 2, row = (warp & (F::kSoftmaxWarps - 1)) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + t * 128 + lanes, tO = tmem + 256 + t * 128 + lanes;
        int done = 0;  // steps of this stream
        while (true) {
            const Share<FEW> share(walk);
            const Kv8Item& it = walk.it;
            const int i_row = it.row0 + (FEW ? 0 : t * per_stream) + row / group;
            const bool live = i_row < it.row0 + it.rows;
            const int lim = live ? it.L - it.n + i_row : -1;
            const int first_lim = it.L - it.n + it.row0;                                   // last key of the block's first row
            const int stream_first = first_lim + (FEW ? 0 : t * per_stream);               // of the stream's
            const int64_t at = (static_cast<int64_t>(it.q0 + (live ? i_row : 0)) * a.hq + it.h * group + row % group) * kHd;
            const int own = share.own(it, per_stream, t);
            float qs = 0.f, m = kNegInf, l = 0.f;
            if (own > 0 && ok) {
                const uint4* src = reinterpret_cast<const uint4*>(a.q + at);
                float amax = 0.f;
                bool bad = false;
                uint4 u[16];
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    u[v] = live ? src[v] : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {u[v].x, u[v].y, u[v].z, u[v].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        amax = fmaxf(amax, fmaxf(fabsf(bf16lo(w[e])), fabsf(bf16hi(w[e]))));
                        bad |= finite2(w[e]) != w[e];
                    }
                }
                const int stored = kv8_query_exponent(amax);
                const float inv = a.sl2e < 0.f ? -kv8_inverse(stored) : kv8_inverse(stored);
                // a row (or a scale) with an infinity or a NaN has no defined logit: NaN throughout, by its sum of weights
                bad |= !(fabsf(a.sl2e) < __builtin_huge_valf());
                qs = bad ? 0.f : kv8_power(stored) * fabsf(a.sl2e);
                if (bad && lim >= 0) l = __int_as_float(0x7fffffff);  // (a row before the context's first token sees nothing: zeros)
                uint8_t* dst = sQ + (F::kQTiles == 1 ? 0 : t * 2 * F::kQHalf) + row * 128;
#pragma unroll
                for (int v = 0; v < (F::kQTiles == 1 && t == 1 ? 0 : 16); ++v) {
                    const uint32_t w[4] = {u[v].x, u[v].y, u[v].z, u[v].w};
                    uint32_t f[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[e] = bad ? 0u : pack_half2(bf16lo(w[e]) * inv, bf16hi(w[e]) * inv);
                    *reinterpret_cast<uint4*>(dst + (v >> 3) * F::kQHalf + (((v & 7) ^ (row & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0 && F::kQTiles == 2) mbar_arrive(&sh.q_full[t]);
                // One tile for both. Stream 1 is told of items in which it has steps: of the others nothing would hold back the next
                // item's arrival until its MMA warp has met this phase, and a phase that passes unseen is taken for the one before.
                if (lane == 0 && F::kQTiles == 1 && t == 0) {
                    mbar_arrive(&sh.q_full[0]);
                    if (share.own(it, per_stream, 1) > 0) mbar_arrive(&sh.q_full[1]);
                }
            }
            for (int i = 0; i < own && ok; ++i, ++done) {
                const int b = done & 1, u = share.step(t, i), c = count + u - share.u0;
                ok = wait_one(&sh.s_full[t][b], done >> 1, a.err, 906);
                if (!ok) break;
                tc_fence_after();
                uint32_t s[64], pairs[32];
                tmem_ld64(tS + b * 64, s);
                tmem_loaded(s);
                const PageScale* info = sh.info[c % F::kInfo];
                float alpha;
                if ((u + 1) * kStep - 1 > stream_first) softmax_step<true>(s, pairs, info, qs, u * kStep, lim, m, l, alpha);
                else softmax_step<false>(s, pairs, info, qs, u * kStep, lim, m, l, alpha);
                tmem_st32(tS + b * 64, pairs);
                if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                    // O *= alpha once the step before has landed, and before this one is issued
                    ok = wait_one(&sh.o_done[t][b ^ 1], (done - 1) >> 1, a.err, 907);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int part = 0; part < 4; ++part) {
                        uint32_t o[32];
                        tmem_ld32(tO + part * 32, o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st32(tO + part * 32, o);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[t][b]);
            }
            if (own > 0 && ok) ok = wait_one(&sh.o_done[t][(done - 1) & 1], (done - 1) >> 1, a.err, 907);
            tc_fence_after();
            const bool nan_seen = *reinterpret_cast<volatile int*>(&sh.nan_seen[item % kItems]) != 0;
            // the row's sums, 32 dimensions at a time
            auto sums = [&](int part, uint32_t (&o)[32]) {
                if (own > 0 && ok) {
                    tmem_ld32(tO + part * 32, o);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                }
                if (nan_seen) {  // NaN values between the block's first row and this one: their dimensions are NaN
                    uint32_t gone = 0;
                    for (int k = max(first_lim + 1, share.u0 * kStep); k <= min(lim, share.u1 * kStep - 1); ++k) {
                        int page = a.page_table[static_cast<int64_t>(it.r) * a.max_pages + k / kPage];
                        if (page < 0 || page >= a.num_pages) page = 0;
                        const int tk = k % kPage;
                        const uint8_t* v = a.kv8 + (static_cast<int64_t>(page) * a.hkv + it.h) * kKv8Bytes + kKv8Values + part * 512 +
                                           tk % 8 / 2 * 16 + tk / 8 * 2 + tk % 2;
#pragma unroll 1
                        for (int d = 0; d < 32; ++d)
                            if ((v[d / 4 * 64 + d % 4 * 4] & 0x7f) == 0x7f) gone |= 1u << d;
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (gone >> e & 1) o[e] = 0x7fffffffu;
                }
            };
            float scale0 = 1.f, scale1 = 0.f;  // FEW: factors of the streams' sums
            float* other = reinterpret_cast<float*>(sQ);  // FEW: stream 1's sums [dimension][row]
            const bool joins = FEW && share.own(it, per_stream, 1) > 0;
            const int a0 = walk.cta0(), a1 = walk.cta1();
            // a CTA takes part in at most one item that it did not begin and one that it does not end
            const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (static_cast<int>(blockIdx.x) == a0);
            const int slot_row = FEW ? row : t * kRows + row;
            auto store = [&](int part) {
                uint32_t o[32];
                sums(part, o);
                const float inv = a0 != a1 ? 1.f : l == 0.f ? 0.f : kKv8Unlift / l;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    float x = __uint_as_float(o[e]);
                    if (joins) x = x * scale0 + other[(part * 32 + e) % F::kJoinDims * ROWS + row] * scale1;
                    o[e] = __float_as_uint(x * inv);
                }
                if (live && a0 != a1) {
                    // [group of four dimensions][row]: a warp's stores are next to each other
                    float4* dst = reinterpret_cast<float4*>(a.ws_o + slot * ROWS * kHd) + part * 8 * ROWS + slot_row;
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        dst[c * ROWS] = make_float4(__uint_as_float(o[4 * c]), __uint_as_float(o[4 * c + 1]), __uint_as_float(o[4 * c + 2]),
                                                    __uint_as_float(o[4 * c + 3]));
                } else if (live) {
                    uint4* dst = reinterpret_cast<uint4*>(a.out + at + part * 32);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(__uint_as_float(o[8 * c + 2 * e]), __uint_as_float(o[8 * c + 2 * e + 1]));
                        dst[c] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            };
            if (FEW) {
                constexpr int kParts = F::kJoinDims / 32;  // at a time
                named_barrier(1, kSoftmaxThreads);  // both streams are done with Q
                if (t == 1) sh.ml[row] = make_float2(m, l);
#pragma unroll 1
                for (int part0 = 0; part0 < 4; part0 += kParts) {
                    if (t == 1 && own > 0) {
#pragma unroll 1
                        for (int part = part0; part < part0 + kParts; ++part) {
                            uint32_t o[32];
                            sums(part, o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) other[((part - part0) * 32 + e) * ROWS + row] = __uint_as_float(o[e]);
                        }
                    }
                    named_barrier(1, kSoftmaxThreads);
                    if (t == 0) {
                        if (part0 == 0) {
                            if (joins) {
                                const float2 x = sh.ml[row];
                                const float M = fmaxf(m, x.x);
                                scale0 = m == kNegInf ? 1.f : exp2_ftz(m - M);
                                scale1 = x.x == kNegInf ? 1.f : exp2_ftz(x.x - M);
                                l = l * scale0 + x.y * scale1;
                                m = M;
                            }
                            if (a0 != a1 && live) *reinterpret_cast<float2*>(a.ws_ml + (slot * ROWS + slot_row) * 2) = make_float2(m, l);
                        }
#pragma unroll 1
                        for (int part = part0; part < part0 + kParts; ++part) store(part);
                    }
                    named_barrier(1, kSoftmaxThreads);  // stream 1's sums were read: the next ones or Q may come
                }
            } else {
                if (a0 != a1 && live) *reinterpret_cast<float2*>(a.ws_ml + (slot * ROWS + slot_row) * 2) = make_float2(m, l);
#pragma unroll 1
                for (int part = 0; part < 4; ++part) store(part);
            }
            tc_fence_before();
            count += share.u1 - share.u0;
            ++item;
            if (!walk.next(a, per_block)) break;
        }
    } else if (warp < 12) {
        // ---------------- each step into f16 tiles: keys by one team of warps, values by the other
        // 64 rows: stream 0's are warps 2 .. 5, stream 1's 8 .. 11; else the latter for both
        const int cw = warp < 8 ? warp - 2 : warp - 8, ct = (cw & 1) * 32 + lane, mine = warp < 8 ? 0 : 1;
        const bool keys = cw < 2;
        // keys: token, 16 dimensions of each half; the row is the token's place
        const int k_tok = ct >> 2, k_c = ct & 3, k_place = k_tok % 8 / 2 * 4 + k_tok / 8 * 2 + k_tok % 2;
        // values: 8 keys of a page (half v_b), groups of four dimensions v_dq and v_dq + 8, pages v_page and v_page + 2:
        // eight lanes store to eight different 16-byte columns, and load with two to a bank
        const int v_b = lane & 1, v_page = lane >> 2 & 1, v_dq = (lane >> 1 & 1) | (lane >> 3) << 1 | (cw & 1) << 4;
        constexpr int kUnits = 4;
        int count = 0, taken[2] = {0, 0};
        while (ok) {
            const Share<FEW> share(walk);
            const Kv8Item& it = walk.it;
            const int first_lim = it.L - it.n + it.row0, last_lim = first_lim + it.rows - 1;
            for (int u = share.u0 + (F::kTeams == 2 ? mine : 0); u < share.u1 && ok; u += F::kTeams) {
                const int t = FEW ? (u - share.u0) & 1 : 0, n = F::kTeams == 2 ? taken[t] : count + u - share.u0;
                const int raw = F::slot(t, n), st = F::stage(t, taken[t]), use = F::use(taken[t]);
                ++taken[t];
                uint64_t* empty = keys ? &sh.k_empty[st] : &sh.v_empty[st];
                // With a team for each stream the codes are read as soon as they are there, ahead of their tile (their slots then come
                // back earlier: 24 requests x 6 drafted rows 4% less). One team has not the registers (chunks 2% more).
                constexpr bool kAhead = F::kTeams == 2;
                const bool both = !kAhead && use > 0;
                ok = wait_two(&sh.raw_full[raw], n / 2, both ? empty : &sh.raw_full[raw], both ? use - 1 : n / 2, a.err, 908);
                if (!ok) break;
                const uint8_t* src = sRaw + raw * kPages * kKv8Bytes;
                // The fence before a slot is given back puts its reads ahead of the copy that overwrites it: without, that copy
                // overtook loads on their way (giving it back after the conversion instead: chunks a quarter more).
                if (keys) {
                    const uint8_t* ks = src + k_tok * 64 + k_c * 16;
                    uint8_t* kd = sK + st * kKTile + k_place * 128;
                    const int to[2] = {((2 * k_c) ^ (k_place & 7)) << 4, ((2 * k_c + 1) ^ (k_place & 7)) << 4};
                    auto codes = [&](int i, int x) { return *reinterpret_cast<const uint4*>(ks + i * kKv8Bytes + x * 1024); };
                    auto convert = [&](int i, int x, const uint4& v) {
                        uint32_t f[8];
                        e4m3x4_to_half(v.x, f[0], f[1]);
                        e4m3x4_to_half(v.y, f[2], f[3]);
                        e4m3x4_to_half(v.z, f[4], f[5]);
                        e4m3x4_to_half(v.w, f[6], f[7]);
                        uint8_t* dst = kd + x * (kKTile / 2) + i * (kPage * 128);
                        *reinterpret_cast<uint4*>(dst + to[0]) = make_uint4(f[0], f[1], f[2], f[3]);
                        *reinterpret_cast<uint4*>(dst + to[1]) = make_uint4(f[4], f[5], f[6], f[7]);
                    };
                    // 128 rows: all codes first, so that their slot comes back early (8% less, where two steps are all that is on
                    // its way); else two pages at a time, less code at once (24 x 6 rows 3% less).
                    if constexpr (ROWS == 128) {
                        uint4 w[kPages][2];
#pragma unroll
                        for (int i = 0; i < kPages; ++i)
#pragma unroll
                            for (int x = 0; x < 2; ++x) w[i][x] = codes(i, x);
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.raw_empty[raw]);
#pragma unroll
                        for (int i = 0; i < kPages; ++i)
#pragma unroll
                            for (int x = 0; x < 2; ++x) convert(i, x, w[i][x]);
                    } else {
                        if (kAhead && use > 0) ok = wait_one(empty, use - 1, a.err, 908);
                        if (!ok) break;
#pragma unroll 2
                        for (int i = 0; i < kPages; ++i)
#pragma unroll
                            for (int x = 0; x < 2; ++x) convert(i, x, codes(i, x));
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (ROWS != 128 && lane == 0) mbar_arrive(&sh.raw_empty[raw]);
                    if (lane == 0) mbar_arrive(&sh.k_full[st]);
                    continue;
                }
                uint4 w[kUnits][2];  // pages v_page + 2 (i / 2), groups v_dq + 8 (i % 2)
#pragma unroll
                for (int i = 0; i < kUnits; ++i)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        w[i][x] = *reinterpret_cast<const uint4*>(src + (v_page + 2 * (i / 2)) * kKv8Bytes + kKv8Values + (v_dq + 8 * (i % 2)) * 64 + v_b * 32 + x * 16);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.raw_empty[raw]);
                if ((u + 1) * kStep - 1 > first_lim) {  // some row does not see all of the step
                    bool any = false;
#pragma unroll
                    for (int i = 0; i < kUnits; ++i)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int key = u * kStep + (v_page + 2 * (i / 2)) * kPage;
                            uint32_t hidden = 0, seen = 0;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int k = key + (e >> 1) * 8 + (2 * v_b + x) * 2 + (e & 1);
                                if (k > first_lim) hidden |= 0x80u << (8 * e);
                                if (k <= last_lim) seen |= 0x80u << (8 * e);
                            }
                            uint32_t y[4] = {w[i][x].x, w[i][x].y, w[i][x].z, w[i][x].w};
#pragma unroll
                            for (int d = 0; d < 4; ++d) {
                                const uint32_t bad = nan_codes(y[d]) & hidden;
                                any |= (bad & seen) != 0;
                                y[d] &= ~((bad >> 7) * 0xffu);
                            }
                            w[i][x] = make_uint4(y[0], y[1], y[2], y[3]);
                        }
                    if (any) *reinterpret_cast<volatile int*>(&sh.nan_seen[item % kItems]) = 1;
                    __threadfence_block();
                }
                if (kAhead && use > 0) ok = wait_one(empty, use - 1, a.err, 908);
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < kUnits; ++i) {
                    const uint32_t w0[4] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w};
                    const uint32_t w1[4] = {w[i][1].x, w[i][1].y, w[i][1].z, w[i][1].w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int dim = (v_dq + 8 * (i % 2)) * 4 + x;
                        uint32_t f[4];
                        e4m3x4_to_half(w0[x], f[0], f[1]);
                        e4m3x4_to_half(w1[x], f[2], f[3]);
                        *reinterpret_cast<uint4*>(sV + st * kVTile + dim * 128 + (((2 * (v_page + 2 * (i / 2)) + v_b) ^ (dim & 7)) << 4)) =
                            make_uint4(f[0], f[1], f[2], f[3]);
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.v_full[st]);
            }
            count += share.u1 - share.u0;
            ++item;
            if (!walk.next(a, per_block)) break;
        }
    } else if (warp < 14) {
        // ---------------- MMAs of stream t: the warp waits together, one lane issues (descriptors stay uniform)
        constexpr uint32_t id_s = idesc_f16(kRows, kStep), id_o = idesc_f16(kRows, kHd);
        const int t = warp - 12;
        const bool lead = elect_lane();
        // 64 rows: MMA rows 64 t and on are theirs, the others' sums nobody reads (whatever lies there in shared memory)
        const uint64_t dQ = umma_desc_sw128(smem_u32(F::kQTiles == 1 ? sQ - t * F::kQHalf : sQ + t * 2 * F::kQHalf)), dK = umma_desc_sw128(smem_u32(sK)), dV = umma_desc_sw128(smem_u32(sV));
        const uint32_t tS = tmem + t * 128, tO = tmem + 256 + t * 128;
        int s_count = 0, p_count = 0, loaded = 0;  // S and PV issued so far, items in which the stream had any
        while (ok) {
            const Share<FEW> share(walk);
            const int own = share.own(walk.it, per_stream, t);
            auto issue_s = [&](int i) {  // S of the i-th own step into its buffer, which p of two steps before has left
                if (i >= own || !ok) return;
                const int n = FEW ? s_count : count + i, st = F::stage(t, n), use = F::use(n), b = s_count & 1;
                if (i == 0) ok = wait_one(&sh.q_full[t], loaded, a.err, 905);
                ok = ok && wait_two(&sh.k_full[st], use, s_count < 2 ? &sh.k_full[st] : &sh.o_done[t][b],
                                    s_count < 2 ? use : (s_count - 2) >> 1, a.err, 908);
                if (!ok) return;
                tc_fence_after();
                if (lead) {
                    const uint64_t k = dK + (st * kKTile >> 4);
#pragma unroll
                    for (int x = 0; x < 8; ++x)  // 16 dimensions: 32 bytes; the second 64 lie in the other half tile
                        umma_bf16(tS + b * 64, dQ + (((x >> 2) * F::kQHalf + (x & 3) * 32) >> 4),
                                  k + (((x >> 2) * (kKTile / 2) + (x & 3) * 32) >> 4), id_s, x > 0 ? 1u : 0u);
                    umma_commit(&sh.s_full[t][b]);
                    umma_commit(&sh.k_empty[st]);
                }
                __syncwarp();
                ++s_count;
            };
            issue_s(0);
            issue_s(1);
            for (int i = 0; i < own && ok; ++i) {
                const int n = FEW ? p_count : count + i, st = F::stage(t, n), b = p_count & 1;
                ok = wait_two(&sh.v_full[st], F::use(n), &sh.p_full[t][b], p_count >> 1, a.err, 909);
                if (!ok) break;
                tc_fence_after();
                if (lead) {
                    const uint64_t v = dV + (st * kVTile >> 4);
#pragma unroll
                    for (int x = 0; x < 4; ++x)  // 16 keys: 8 columns of p
                        umma_bf16_ta(tO, tS + b * 64 + x * 8, v + (x * 32 >> 4), id_o, (i > 0 || x > 0) ? 1u : 0u);
                    umma_commit(&sh.o_done[t][b]);
                    umma_commit(&sh.v_empty[st]);
                }
                __syncwarp();
                ++p_count;
                issue_s(i + 2);
            }
            // steps that only the other stream sees: their stages are free as far as this one goes
            if (!FEW)
                for (int u = share.u0 + own; u < share.u1 && ok; ++u) {
                    const int c = count + u - share.u0, st = F::stage(0, c);
                    ok = wait_two(&sh.k_full[st], F::use(c), &sh.v_full[st], F::use(c), a.err, 908);
                    if (ok && lead) {
                        mbar_arrive(&sh.k_empty[st]);
                        mbar_arrive(&sh.v_empty[st]);
                    }
                    __syncwarp();
                }
            count += share.u1 - share.u0;
            if (own > 0) ++loaded;
            if (!walk.next(a, per_block)) break;
        }
    } else if (warp == 14) {
        // ---------------- codes and scales of each step
        int c = 0, filled[2] = {0, 0};  // steps; of a team
        while (ok) {
            const Share<FEW> share(walk);
            const Kv8Item& it = walk.it;
            const int seen = (it.L - it.n + it.row0 + it.rows - 1) / kPage + 1;  // pages that any row sees
            const int* table = a.page_table + static_cast<int64_t>(it.r) * a.max_pages;
            const int pages = min(seen, share.u1 * kPages);
            // eight steps at a time: lane 4 s + p has page p of the s-th, the next eight's ids on their way
            int next = share.u0 * kPages + lane < pages ? table[share.u0 * kPages + lane] : 0;
            if (lane == 0) sh.nan_seen[item % kItems] = 0;  // last of an item that is done
            for (int u0 = share.u0; u0 < share.u1 && ok; u0 += 8) {
                const int page = u0 * kPages + lane;
                int id = next;
                next = page + 32 < pages ? table[page + 32] : 0;
                if (id < 0 || id >= a.num_pages) {
                    record_error(a.err, MSGL_ERR_BOUNDS, 902);
                    id = 0;
                }
                const int64_t block = static_cast<int64_t>(id) * a.hkv + it.h;
                const uint32_t sc = page < pages ? *reinterpret_cast<const uint16_t*>(a.scales + block * 2) : 0x7f7fu;
                const int v_stored = kv8_value_exponent(sc);
                const PageScale scale = {kv8_power(sc & 0xff), static_cast<float>(v_stored - 127), kv8_inverse(v_stored) * kKv8Unlift, 0.f};
                const uint8_t* codes = a.kv8 + block * kKv8Bytes;
                for (int s = 0; s < 8 && u0 + s < share.u1; ++s, ++c) {
                    const int t = F::kTeams == 2 ? (u0 + s - share.u0) & 1 : 0, n = filled[t], raw = F::slot(t, n);
                    if (n >= 2) ok = ok && wait_one(&sh.raw_empty[raw], n / 2 - 1, a.err, 908);
                    if (!ok) break;
                    ++filled[t];
                    // the scales go ahead of the barrier that the conversion, the MMAs and so the softmax wait for
                    if (lane >> 2 == s) sh.info[c % F::kInfo][lane & 3] = scale;
                    __syncwarp();
                    // the bytes are expected before any of them comes
                    if (lane == 0) mbar_arrive_expect_tx(&sh.raw_full[raw], min(kPages, pages - (u0 + s) * kPages) * kKv8Bytes);
                    __syncwarp();
                    if (lane >> 2 == s && page < pages) bulk_load(sRaw + (raw * kPages + (lane & 3)) * kKv8Bytes, codes, kKv8Bytes, &sh.raw_full[raw]);
                }
            }
            ++item;
            if (!walk.next(a, per_block)) break;
        }
        // after a wait that ran out: no copy is left on its way into the block's shared memory
        for (int t = 0; t < F::kTeams; ++t)
            for (int n = max(0, filled[t] - 2); n < filled[t]; ++n) wait_one(&sh.raw_full[F::slot(t, n)], n / 2, a.err, 908);
    }
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int ROWS>
int launch(const Kv8AttnArgs& a, int grid, msgl_stream_t stream) {
    static std::atomic<int> optin[kMaxDevices];
    const cudaError_t e = smem_optin(attend_tiles_kernel<ROWS>, Form<ROWS>::kSmem, optin);
    if (e != cudaSuccess) return set_error(MSGL_ERR_CUDA, cudaGetErrorString(e));
    launch_pdl(attend_tiles_kernel<ROWS>, dim3(grid), dim3(kThreads), Form<ROWS>::kSmem, stream, a);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

}  // namespace

int launch_attend_tiles(const Kv8AttnArgs& a, int rows, int grid, msgl_stream_t stream) {
    return rows <= 64 ? launch<64>(a, grid, stream) : rows <= 128 ? launch<128>(a, grid, stream) : launch<256>(a, grid, stream);
}

}  // namespace msgl
