// kv8.cuh -- the 8-bit key / value pool: format, exponents and conversions shared by its kernels.
//
// kv8 [num_pages, Hkv, 4096] bytes of e4m3 codes and scales [num_pages, Hkv, 2] stored exponents (keys,
// values): value = code * 2^(scale - 127). Of a page and kv head,
//   keys    byte  (d / 64) * 1024 + t * 64 + d % 64                     of token t, dimension d;
//   values  byte  2048 + (d / 4) * 64 + (t % 8) / 2 * 16 + (d % 4) * 4 + (t / 8) * 2 + t % 2.
// That is the order in which an m16n8k16 MMA wants its fragments: lane 4 g + c takes 16 bytes of key g
// (or 8 + g) at dimension 16 c of a half, and 4 dimensions x the tokens 2 c, 2 c + 1, 8 + 2 c, 9 + 2 c of the
// values, so a warp reads 512 consecutive bytes at a time, from global or shared memory, and neither
// ldmatrix nor a swizzle is needed. A page and head is one copy of 4 KB.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "kv8_args.h"

namespace msgl {
// Attention of more than 16 rows x heads of a group (kv8_tiles.cu). Items that CTAs share are left as partial sums:
// CTA b's in slot 2 b where it goes on with an item, in slot 2 b + 1 where it leaves one to the next.
// rows: of a block, 64, 128 or 256.
int launch_attend_tiles(const Kv8AttnArgs& a, int rows, int grid, msgl_stream_t stream);

constexpr int kKv8Page = 16;
constexpr int kKv8Head = 128;
constexpr int kKv8Bytes = 4096;   // of a page and kv head
constexpr int kKv8Values = 2048;  // where the values begin
// Smallest stored exponent, 2^-96: the weights' sum of the attention, which counts a page in units of
// its values' scale, stays within fp32 then.
constexpr int kKv8Floor = 31;

// Stored exponent of the smallest power of two s with amax <= 448 s (448: the largest e4m3 value).
__device__ __forceinline__ int kv8_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    return max(kKv8Floor, static_cast<int>(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u));
}
__device__ __forceinline__ float kv8_power(int stored) { return __uint_as_float(static_cast<uint32_t>(stored) << 23); }
// 2^-(stored - 127), stored in [1, 253]
__device__ __forceinline__ float kv8_inverse(int stored) { return __uint_as_float(static_cast<uint32_t>(254 - stored) << 23); }
// The values' stored exponent of a page's two scale bytes, as the attention takes it. The append stores none below the
// floor; a page that was only cleared (codes of 0, scale bytes of 0) counts as zeros at the floor: with 2^-127 its keys' weights
// would not fit the sum.
__device__ __forceinline__ int kv8_value_exponent(uint32_t scale2) { return max(kKv8Floor, static_cast<int>(scale2 >> 8 & 0xff)); }

// Token of a page at place i of its values' order.
__host__ __device__ constexpr int token_at(int i) { return (i % 4 / 2) * 8 + (i / 4) * 2 + i % 2; }

// Two e4m3 codes (the low 16 bits) as two halves, exactly.
__device__ __forceinline__ uint32_t e4m3_to_half2(uint32_t codes) {
    uint32_t h;
    asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(h) : "r"(codes));
    return h;
}
// Four codes of a word: halves of bytes 0, 1 and of bytes 2, 3.
__device__ __forceinline__ void e4m3x4_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}
// Codes of x0 (low byte) and x1, rounded to nearest even; |x| <= 448 or NaN.
__device__ __forceinline__ uint32_t e4m3_codes2(float x0, float x1) {
    return __nv_cvt_float2_to_fp8x2(make_float2(x0, x1), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Queries of the attention, in f16: a row over 2^(this - 127), which puts its largest element into [2^14, 2^15) (up to 65280
// next to bf16's largest, less below 2^-112): f16 holds it exactly down to 2^-31 of that, and to 2^-39 behind. (Into [1, 2): to
// 2^-17 and 2^-25, which shows where the largest element meets zeros.) Sums of products with codes stay below 2^32.
__device__ __forceinline__ int kv8_query_exponent(float amax) { return max(1, min(239, static_cast<int>(__float_as_uint(amax) >> 23) - 14)); }
// Weights of the attention, in f16: p = 2^(s - m + kKv8Lift), s with the exponent of the page's values, m the row's running
// maximum, which moves only where it grows by more than kKv8Lag, so that p <= 2^15. f16 rounds each weight by 2^-12 of itself
// at most (a code carries a rounding of 2^-4 already) down to 2^-25 of the row's largest and flushes below 2^-36: behind a key
// that takes nearly all of the weight, or in pages whose values are that much smaller, the others still count. With
// p = 2^(s - m) <= 2^8 that began at 2^-14 (keys 20 octaves below a sink came out 3% off, 25 octaves lost). The sums of weights
// stay in fp32, of 2^-kKv8Lift p. Roundings between a logit and its exponent go down, so that p <= 2^15 whatever the logits' size, and
// up to 2^26 the largest one's p stays above 2^-14.
constexpr float kKv8Lift = 11.f, kKv8Lag = 4.f, kKv8Unlift = 0x1p-11f;
__device__ __forceinline__ bool kv8_grows(float top, float m) { return top > __fadd_rd(m, kKv8Lag) || m == -__builtin_huge_valf(); }
// What is subtracted from s.
__device__ __forceinline__ float kv8_base(float m) { return m == -__builtin_huge_valf() ? 0.f : __fsub_ru(m, kKv8Lift); }
// Bytes of a word of codes that are NaN, as 0x80 each.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ int64_t larger(int64_t a, int64_t b) { return a > b ? a : b; }
__device__ __forceinline__ int64_t smaller(int64_t a, int64_t b) { return a < b ? a : b; }

// ------------------------------------------------------------------ attention: the row of all work
// An item is a block of query rows of a request on a kv head; its units are the UNIT-key pieces that any of
// the rows sees, and COST units stand ahead of them for what an item takes whatever its length (rows loaded, sums joined
// and stored). All items in a row (request, row block, head) are dealt to the CTAs in equal parts of that, so that
// ragged contexts and causal chunks leave no tail; a CTA does the units in its part. (Without the cost the CTA that got
// the first rows of a prompt of 2048 had 18 short items: 203 us, where the others took 55.)
struct Kv8Item {
    int r, rb, h;
    int L, n, q0;    // context, rows of the request, first of them
    int row0, rows;  // query rows of the block, within the request
    int units;
};

// Context and rows of request r; n = 0 where it is skipped.
__device__ __forceinline__ void kv8_request(const Kv8AttnArgs& a, int r, bool report, int& L, int& n, int& q0) {
    L = a.seq_lens[r];
    q0 = a.q_indptr ? a.q_indptr[r] : r;
    n = a.q_indptr ? a.q_indptr[r + 1] - q0 : 1;
    if (n < 0 || n > a.max_q_len || q0 < 0 || (n > 0 && q0 > a.total_q - n)) {
        if (report) record_error(a.err, MSGL_ERR_BOUNDS, 901);
        n = 0;
    }
    if (n > 0 && (L < 0 || L > a.max_len)) {
        if (report) record_error(a.err, MSGL_ERR_BOUNDS, 900);
        L = L < 0 ? 0 : a.max_len;
    }
}

// Units that the rows [row0, row0 + count) of a request see.
template <int UNIT>
__device__ __forceinline__ int kv8_units(int L, int n, int row0, int count) {
    const int last = L - n + min(n, row0 + count) - 1;
    return row0 < n && last >= 0 ? last / UNIT + 1 : 0;
}

template <int UNIT, int COST>
struct Kv8Walk {
    Kv8Item it;
    int64_t first;  // place of the item's first unit
    int64_t begin, end, per;  // of the CTA's part; of a part

    __device__ __forceinline__ void set_block(int per_block) {
        it.row0 = it.rb * per_block;
        it.rows = min(per_block, it.n - it.row0);
        it.units = kv8_units<UNIT>(it.L, it.n, it.row0, per_block);
    }
    // The CTA's units of the item; there are some in every item of the walk.
    __device__ __forceinline__ int u0() const { return static_cast<int>(larger(0, begin - first)); }
    __device__ __forceinline__ int u1() const { return static_cast<int>(smaller(it.units, end - first)); }
    // CTAs that share the item: their first and last
    __device__ __forceinline__ int cta0() const { return static_cast<int>(first / per); }
    __device__ __forceinline__ int cta1() const { return static_cast<int>((first + it.units - 1) / per); }
    // To the next item of which the CTA has a unit; false where there is none.
    __device__ __forceinline__ bool next(const Kv8AttnArgs& a, int per_block) {
        first += it.units + COST;
        if (first >= end) return false;
        if (++it.h < a.hkv) return true;
        it.h = 0;
        do {
            if ((it.rb + 1) * per_block < it.n) {
                ++it.rb;
            } else {
                it.rb = 0;
                do {
                    if (++it.r >= a.num_reqs) return false;
                    kv8_request(a, it.r, false, it.L, it.n, it.q0);
                } while (it.n <= 0);
            }
            set_block(per_block);
        } while (it.units == 0);
        return true;
    }
};

// Scratch of kv8_part.
template <int THREADS>
struct Kv8Scan {
    int64_t sums[THREADS / 32], first_sums[THREADS / 32], before;
    Kv8Item item;
    int found;
};

// Zeros for the first `rows` query rows from q0 on.
__device__ __forceinline__ void zero_rows(const Kv8AttnArgs& a, int q0, int rows) {
    const int64_t from = static_cast<int64_t>(q0) * a.hq * kKv8Head, to = from + static_cast<int64_t>(rows) * a.hq * kKv8Head;
    for (int64_t i = from; i < to; i += 8) *reinterpret_cast<uint4*>(a.out + i) = make_uint4(0, 0, 0, 0);
}

// This CTA's part of all units and the item that holds its first; false where there is none. Rows before their
// context's first token get zeros on the way, and the workspace is told of an item that the CTA before began. Every
// thread of the block calls it.
template <int THREADS, int UNIT, int COST>
__device__ __forceinline__ bool kv8_part(const Kv8AttnArgs& a, int per_block, Kv8Scan<THREADS>& sh, Kv8Walk<UNIT, COST>& walk) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto block_weight = [&](int L, int n, int row0) {
        const int units = kv8_units<UNIT>(L, n, row0, per_block);
        return units ? static_cast<int64_t>(units + COST) * a.hkv : 0;
    };
    auto weight = [&](int r, bool report, Kv8Item& it) {  // and the request's context and rows
        kv8_request(a, r, report, it.L, it.n, it.q0);
        int64_t s = 0;
        for (int row0 = 0; row0 < it.n; row0 += per_block) s += block_weight(it.L, it.n, row0);
        if (report && it.n > it.L) zero_rows(a, it.q0, it.n - it.L);
        return s;
    };
    // A thread has the weight of one request of the first THREADS, which is all that most calls have.
    Kv8Item own{};
    const int64_t first_weight = tid < a.num_reqs ? weight(tid, blockIdx.x == 0, own) : 0;
    int64_t mine = first_weight, upto = first_weight;  // of all its requests; inclusive sum of a warp's first ones
    for (int r = tid + THREADS; r < a.num_reqs; r += THREADS) {
        Kv8Item other;
        mine += weight(r, blockIdx.x == 0, other);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
        mine += __shfl_xor_sync(0xffffffffu, mine, o);
    }
    if (lane == 0) sh.sums[warp] = mine;
    if (lane == 31) sh.first_sums[warp] = upto;
    if (tid == 0) sh.found = 0;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) total += sh.sums[w];
    const int64_t per = larger((total + gridDim.x - 1) / gridDim.x, a.min_units), begin = per * blockIdx.x, end = smaller(total, begin + per);
    walk.per = per;
    walk.begin = begin;
    walk.end = end;
    bool any = begin < end;
    if (any) {
        int64_t base = 0, w = first_weight;
        for (int r0 = 0; r0 < a.num_reqs; r0 += THREADS) {  // blocks of requests, until their sum passes `begin`
            const int r = r0 + tid;
            if (r0 > 0) {
                w = upto = r < a.num_reqs ? weight(r, false, own) : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += y;
                }
                if (lane == 31) sh.first_sums[warp] = upto;
                __syncthreads();
            }
            int64_t ahead = base + upto - w;
            for (int v = 0; v < THREADS / 32; ++v) {
                if (v < warp) ahead += sh.first_sums[v];
                base += sh.first_sums[v];
            }
            if (w > 0 && begin >= ahead && begin < ahead + w) {
                own.r = r;
                sh.item = own;
                sh.before = ahead;
                sh.found = 1;
            }
            __syncthreads();
            if (sh.found) break;
        }
        // in the request: the row block, then the head
        walk.it = sh.item;
        int64_t at = sh.before;
        int rb = 0;
        for (int64_t w; (w = block_weight(walk.it.L, walk.it.n, rb * per_block)) <= begin - at; ++rb) at += w;
        walk.it.rb = rb;
        walk.set_block(per_block);
        walk.it.h = static_cast<int>((begin - at) / (walk.it.units + COST));
        walk.first = at + static_cast<int64_t>(walk.it.h) * (walk.it.units + COST) + COST;
        any = walk.first < end;  // else the part lies in what an item costs
    }
    if (tid == 0) {
        const bool goes_on = any && walk.first < begin;
        const Kv8Item& it = walk.it;
        a.ws_shared[blockIdx.x] = goes_on ? Kv8Shared{walk.cta0(), walk.cta1(), it.q0 + static_cast<int64_t>(it.row0), it.h, it.rows * (a.hq / a.hkv)}
                                          : Kv8Shared{0, -1, 0, 0, 0};
    }
    return any;
}

}  // namespace msgl
