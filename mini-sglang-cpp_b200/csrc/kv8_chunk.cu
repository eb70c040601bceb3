// kv8_chunk.cu -- attention of long chunks over the 8-bit key / value pool, on tcgen05.
//
// One CTA per (256 rows, kv head, request): two tiles of 128 rows (128 / group query tokens x the group's
// heads), keys in blocks of 128 (8 pages). Codes are brought from global memory into registers, converted
// to f16 (exactly) and laid into shared memory as the operands' canonical tiles, once for both row tiles;
// q is scaled to f16 by a power of two per row (2^-25 of its largest value). A page's scales enter the
// exponent: s = (q . k) 2^(q + k exponents) scale log2(e) + (exponent of v), p = 2^(s - m) <= 2^8 in f16, so
// that O needs no scaling by page, and l adds p 2^-(exponent of v).
//
//   warps 0-3, 4-7   softmax of row tile 0 / 1: a thread per row. S from tensor memory, p as f16 pairs over
//                    the first half of S, l and m in registers; O in tensor memory is rescaled only where
//                    the maximum grew by more than 8;
//   warps 8-11       keys and values of the block: 16-byte loads a block ahead, conversion, tiles;
//   warp 12          one lane issues the MMAs: PV of a tile as soon as its p is there, then that tile's next
//                    S, while the other tile's softmax runs.
// Tensor memory: S0, S1, O0, O1 of 128 columns each. The keys of a page take the order in which the pool
// stores their values (4 (t % 8 / 2) + 2 (t / 8) + t % 2), so that a value tile's rows are its dimensions
// and both operands are K-major.
//
// Bound: tensor (4 x 128 FLOP a row and key) and the exponentials (one a row and key, 16 a clock and SM)
// take the same time.
#include <algorithm>

#include "kv8.cuh"

namespace msgl {
namespace {

constexpr int kPage = kKv8Page;
constexpr int kHd = kKv8Head;
constexpr int kKeys = 128;                 // of a block
constexpr int kPages = kKeys / kPage;      // of a block
constexpr int kRows = 128;                 // of a tile
constexpr int kHalfTile = 128 * 128;       // 128 rows x 64 f16
constexpr int kTile = 2 * kHalfTile;       // 32 KB
constexpr int kStages = 2;
constexpr int kInfo = 4;                   // blocks whose page scales are kept
constexpr int kThreads = 512;
constexpr int kSoftRegs = 184, kConvRegs = 104, kMmaRegs = 40;  // 2 x 184 + 104 + 40 = 4 x 128 of the launch
constexpr size_t kSmem = 1024 + (2 + 2 * kStages) * kTile;
constexpr float kNegInf = -__builtin_huge_valf();

__host__ __device__ constexpr uint32_t idesc_f16(int M, int N) {  // A, B f16 K-major, D fp32
    return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ float exp2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <int N>
__device__ __forceinline__ void more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Token of a page at place i of its order.
__host__ __device__ constexpr int token_at(int i) { return (i % 4 / 2) * 8 + (i / 4) * 2 + i % 2; }

// Scales of a page of the block: keys' factor, values' exponent and inverse factor.
struct PageScale {
    float k, v_exp, v_inv, pad;
};

struct Shared {
    uint64_t q_full[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t s_full[2], p_full[2], o_done[2], info_full[kInfo];
    uint32_t tmem;
    int nan_seen;  // a value hidden from some rows of the CTA was NaN
    PageScale info[kInfo][kPages];
};

// Bytes of a word of codes that are NaN, as 0x80 each.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// One block of a row: 128 S columns into p. EDGE: keys behind `lim` do not count.
template <bool EDGE>
__device__ __forceinline__ void softmax_block(uint32_t (&s0)[64], uint32_t (&s1)[64], const PageScale* info, float qs, int key0,
                                              int lim, float& m, float& l, float& alpha) {
    float mx4[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
    for (int p = 0; p < kPages; ++p) {
        const float f = qs * info[p].k, v = info[p].v_exp;
#pragma unroll
        for (int i = 0; i < kPage; ++i) {
            uint32_t& s = p < 4 ? s0[(p & 3) * 16 + i] : s1[(p & 3) * 16 + i];
            float x = fmaf(__uint_as_float(s), f, v);
            if (EDGE && key0 + p * kPage + token_at(i) > lim) x = kNegInf;
            s = __float_as_uint(x);
            mx4[i & 3] = fmaxf(mx4[i & 3], x);
        }
    }
    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
    // The maximum moves only where it grows by more than 8: p stays below 2^8, which f16 holds as well.
    const float next = m == kNegInf || mx > m + 8.f ? fmaxf(m, mx) : m;
    const float base = next == kNegInf ? 0.f : next;
    alpha = next == m ? 1.f : exp2_ftz(m - next);
    float sum = 0.f;
#pragma unroll
    for (int p = 0; p < kPages; ++p) {
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int i = 0; i < kPage; i += 2) {
            const int c = (p & 3) * 16 + i;
            const float x = exp2_ftz(__uint_as_float(p < 4 ? s0[c] : s1[c]) - base);
            const float y = exp2_ftz(__uint_as_float(p < 4 ? s0[c + 1] : s1[c + 1]) - base);
            a += x;
            b += y;
            s0[p * 8 + i / 2] = half2_of(x, y);  // columns 2 i of the pairs: always behind what is still needed
        }
        sum = fmaf(a + b, info[p].v_inv, sum);
    }
    l = fmaf(l, alpha, sum);
    m = next;
}

__global__ void __launch_bounds__(kThreads, 1)
attend_chunk_kernel(const Kv8AttnArgs a) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ Shared sh;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;                      // 2 tiles
    uint8_t* sK = smem + 2 * kTile;          // [kStages]
    uint8_t* sV = sK + kStages * kTile;      // [kStages]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.hq / a.hkv, per_tile = kRows / group;
    const int r = blockIdx.z, h = blockIdx.y;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.q_full[i], 4);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], 4);
            mbar_init(&sh.o_done[i], 1);
        }
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&sh.k_full[i], 4);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_full[i], 4);
            mbar_init(&sh.v_empty[i], 1);
        }
        for (int i = 0; i < kInfo; ++i) mbar_init(&sh.info_full[i], 1);
        fence_barrier_init();
        sh.nan_seen = 0;
    }
    pdl_wait();
    pdl_trigger();
    int L = a.seq_lens[r];
    const int q0 = a.q_indptr[r], n = a.q_indptr[r + 1] - q0;
    const bool report = tid == 0 && blockIdx.x == 0 && h == 0;
    if (n < 0 || n > a.max_q_len || q0 < 0 || q0 > a.total_q - n) {
        if (report) record_error(a.err, MSGL_ERR_BOUNDS, 901);
        return;
    }
    const int row0 = (gridDim.x - 1 - blockIdx.x) * 2 * per_tile;  // first query row; the longest walks first
    if (n > 0 && (L < 0 || L > a.max_len)) {
        if (report) record_error(a.err, MSGL_ERR_BOUNDS, 900);
        L = L < 0 ? 0 : a.max_len;
    }
    if (row0 >= n) return;
    const int first_lim = L - n + row0;  // last key that the CTA's first row sees
    int blocks[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int last = L - n + min(n, row0 + (t + 1) * per_tile) - 1;
        blocks[t] = row0 + t * per_tile < n && last >= 0 ? last / kKeys + 1 : 0;
    }
    const int last_lim = L - n + min(n, row0 + 2 * per_tile) - 1;  // last key that any row sees
    const int total = max(blocks[0], blocks[1]);
    if (warp == 12) {
        tmem_alloc(&sh.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;

    if (warp < 8) {
        more_regs<kSoftRegs>();
        // ---------------- softmax of tile t: a thread per row
        const int t = warp >> 2, m_row = (warp & 3) * 32 + lane;
        const int i_row = row0 + t * per_tile + m_row / group;
        const bool live = i_row < n;
        const int lim = live ? L - n + i_row : -1;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + t * 128 + lanes, tO = tmem + 256 + t * 128 + lanes;
        const int64_t out_at = (static_cast<int64_t>(q0 + (live ? i_row : 0)) * a.hq + h * group + m_row % group) * kHd;
        const int nblk = blocks[t];
        float qs = 0.f, m = kNegInf, l = 0.f;
        bool ok = true;
        if (nblk > 0) {
            {
                const uint4* src = reinterpret_cast<const uint4*>(a.q + out_at);
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
                const int stored = max(1, min(253, static_cast<int>(__float_as_uint(amax) >> 23)));
                const float inv = kv8_inverse(stored);
                // a row with an infinity or a NaN has no defined logit: NaN throughout
                qs = bad ? __int_as_float(0x7fffffff) : kv8_power(stored) * a.sl2e;
                uint8_t* dst = sQ + t * kTile + m_row * 128;
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const uint32_t w[4] = {u[v].x, u[v].y, u[v].z, u[v].w};
                    uint32_t f[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[e] = bad ? 0u : half2_of(bf16lo(w[e]) * inv, bf16hi(w[e]) * inv);
                    *reinterpret_cast<uint4*>(dst + (v >> 3) * kHalfTile + (((v & 7) ^ (m_row & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full[t]);
            const int tile_first = L - n + row0 + t * per_tile;  // last key of the tile's first row
            for (int j = 0; j < nblk && ok; ++j) {
                ok = __all_sync(0xffffffffu, mbar_wait(&sh.info_full[j % kInfo], (j / kInfo) & 1, a.err, 905) &&
                                                 mbar_wait(&sh.s_full[t], j & 1, a.err, 906));
                if (!ok) break;
                tc_fence_after();
                uint32_t s0[64], s1[64];
                tmem_ld64(tS, s0);
                tmem_ld64(tS + 64, s1);
                tmem_ld_wait();
                float alpha;
                if ((j + 1) * kKeys - 1 > tile_first) softmax_block<true>(s0, s1, sh.info[j % kInfo], qs, j * kKeys, lim, m, l, alpha);
                else softmax_block<false>(s0, s1, sh.info[j % kInfo], qs, j * kKeys, lim, m, l, alpha);
                tmem_st64(tS, s0);
                if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                    // O *= alpha once P(j - 1) V(j - 1) has landed, and before P(j) V(j) is issued
                    ok = __all_sync(0xffffffffu, mbar_wait(&sh.o_done[t], (j - 1) & 1, a.err, 907));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t o[64];
                        tmem_ld64(tO + half * 64, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 64; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st64(tO + half * 64, o);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[t]);
            }
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&sh.o_done[t], (nblk - 1) & 1, a.err, 907));
        }
        __syncthreads();  // the converting warps' word on hidden NaN values
        if (ok) {
            tc_fence_after();
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const bool nan_seen = sh.nan_seen != 0;
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                uint32_t o[64];
                if (nblk > 0) {
                    tmem_ld64(tO + part * 64, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 64; ++e) o[e] = 0u;
                }
                if (nan_seen) {  // NaN values between the CTA's first row and this one: their dimensions are NaN
                    uint64_t gone = 0;
                    for (int k = max(0, first_lim + 1); k <= lim; ++k) {
                        int page = a.page_table[static_cast<int64_t>(r) * a.max_pages + k / kPage];
                        if (page < 0 || page >= a.num_pages) page = 0;
                        const int tk = k % kPage;
                        const uint8_t* v = a.kv8 + (static_cast<int64_t>(page) * a.hkv + h) * kKv8Bytes + kKv8Values +
                                           tk % 8 / 2 * 16 + tk / 8 * 2 + tk % 2;
                        for (int d = 0; d < 64; ++d)
                            if ((v[(part * 16 + d / 4) * 64 + d % 4 * 4] & 0x7f) == 0x7f) gone |= 1ull << d;
                    }
#pragma unroll
                    for (int e = 0; e < 64; ++e)
                        if (gone >> e & 1) o[e] = 0x7fffffffu;
                }
                if (live) {
                    uint4* dst = reinterpret_cast<uint4*>(a.out + out_at + part * 64);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = pack_bf16x2(__uint_as_float(o[8 * c + 2 * e]) * inv, __uint_as_float(o[8 * c + 2 * e + 1]) * inv);
                        dst[c] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
        }
        tc_fence_before();
    } else if (warp < 12) {
        fewer_regs<kConvRegs>();
        // ---------------- keys and values of each block into f16 tiles
        const int cw = warp - 8, ct = tid - 256;
        // keys: page i of the block, half, token, 16 dimensions of it; the row is the token's place
        const int k_half = ct >> 6, k_tok = (ct >> 2) & 15, k_c = ct & 3;
        const int k_place = k_tok % 8 / 2 * 4 + k_tok / 8 * 2 + k_tok % 2;
        // values: pages 4 i + v_page, groups of four dimensions v_dq + 16 i' ..., 8 keys of the page (half v_b)
        const int v_b = lane & 1, v_page = (lane >> 1) & 3, v_dq = cw * 4 + (lane >> 3);
        const int seen_pages = last_lim / kPage + 1;
        const int* pt = a.page_table + static_cast<int64_t>(r) * a.max_pages;
        const uint8_t* pool = a.kv8 + static_cast<int64_t>(h) * kKv8Bytes;
        const int64_t page_bytes = static_cast<int64_t>(a.hkv) * kKv8Bytes;
        auto page_id = [&](int j) {  // lane p: page p of block j; -1 behind the last one that a row sees
            const int p = j * kPages + lane;
            int id = -1;
            if (lane < kPages && j < total && p < seen_pages) {
                id = pt[p];
                if (id < 0 || id >= a.num_pages) {
                    record_error(a.err, MSGL_ERR_BOUNDS, 902);
                    id = 0;
                }
            }
            return id;
        };
        uint4 kreg[kPages];
        uint4 vreg[4][2];
        auto load_keys = [&](int ids) {
#pragma unroll
            for (int i = 0; i < kPages; ++i) {
                const int id = __shfl_sync(0xffffffffu, ids, i);
                kreg[i] = id >= 0 ? __ldg(reinterpret_cast<const uint4*>(pool + id * page_bytes + k_half * 1024 + k_tok * 64 + k_c * 16))
                                  : make_uint4(0, 0, 0, 0);
            }
        };
        auto load_values = [&](int ids) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // pages 4 (i / 2) + v_page, dimension groups v_dq + 16 (i % 2)
                const int id = __shfl_sync(0xffffffffu, ids, 4 * (i >> 1) + v_page);
                const uint4* src = reinterpret_cast<const uint4*>(pool + id * page_bytes + kKv8Values + (v_dq + 16 * (i & 1)) * 64 + v_b * 32);
#pragma unroll
                for (int u = 0; u < 2; ++u) vreg[i][u] = id >= 0 ? __ldg(src + u) : make_uint4(0, 0, 0, 0);
            }
        };
        int ids = page_id(0), ids_next = page_id(1);
        if (total > 0) load_keys(ids);
        bool ok = true;
        for (int j = 0; j < total && ok; ++j) {
            const int st = j % kStages;
            load_values(ids);
            if (cw == 0) {
                uint32_t sc = 0x7f7f;
                if (lane < kPages && ids >= 0)
                    sc = *reinterpret_cast<const uint16_t*>(a.scales + (static_cast<int64_t>(ids) * a.hkv + h) * 2);
                if (lane < kPages) {
                    const int ve = sc >> 8;
                    sh.info[j % kInfo][lane] = {kv8_power(sc & 0xff), static_cast<float>(ve - 127), kv8_inverse(ve), 0.f};
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.info_full[j % kInfo]);
            }
            ok = j < kStages || __all_sync(0xffffffffu, mbar_wait(&sh.k_empty[st], (j / kStages - 1) & 1, a.err, 908));
            if (!ok) break;
            uint8_t* kd = sK + st * kTile + k_half * kHalfTile;
#pragma unroll
            for (int i = 0; i < kPages; ++i) {
                const int row = i * kPage + k_place;
                uint32_t f[8];
                e4m3x4_to_half(kreg[i].x, f[0], f[1]);
                e4m3x4_to_half(kreg[i].y, f[2], f[3]);
                e4m3x4_to_half(kreg[i].z, f[4], f[5]);
                e4m3x4_to_half(kreg[i].w, f[6], f[7]);
                *reinterpret_cast<uint4*>(kd + row * 128 + (((2 * k_c) ^ (row & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
                *reinterpret_cast<uint4*>(kd + row * 128 + (((2 * k_c + 1) ^ (row & 7)) << 4)) = make_uint4(f[4], f[5], f[6], f[7]);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.k_full[st]);
            ids = ids_next;
            ids_next = page_id(j + 2);
            if (j + 1 < total) load_keys(ids);
            if ((j + 1) * kKeys - 1 > first_lim) {  // some row does not see all of the block
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int key = j * kKeys + (4 * (i >> 1) + v_page) * kPage, c = 2 * v_b + u;
                        uint32_t hidden = 0, seen = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int k = key + token_at(4 * c + e);
                            if (k > first_lim) hidden |= 0x80u << (8 * e);
                            if (k <= last_lim) seen |= 0x80u << (8 * e);
                        }
                        uint32_t w[4] = {vreg[i][u].x, vreg[i][u].y, vreg[i][u].z, vreg[i][u].w};
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint32_t bad = nan_bytes(w[x]) & hidden;
                            if (bad & seen) sh.nan_seen = 1;
                            w[x] &= ~((bad >> 7) * 0xffu);
                        }
                        vreg[i][u] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
            }
            ok = j < kStages || __all_sync(0xffffffffu, mbar_wait(&sh.v_empty[st], (j / kStages - 1) & 1, a.err, 909));
            if (!ok) break;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint8_t* vd = sV + st * kTile + (i >> 1) * kHalfTile;
                const uint32_t w0[4] = {vreg[i][0].x, vreg[i][0].y, vreg[i][0].z, vreg[i][0].w};
                const uint32_t w1[4] = {vreg[i][1].x, vreg[i][1].y, vreg[i][1].z, vreg[i][1].w};
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int dim = (v_dq + 16 * (i & 1)) * 4 + x;
                    uint32_t f[4];
                    e4m3x4_to_half(w0[x], f[0], f[1]);
                    e4m3x4_to_half(w1[x], f[2], f[3]);
                    *reinterpret_cast<uint4*>(vd + dim * 128 + (((2 * v_page + v_b) ^ (dim & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.v_full[st]);
        }
        __syncthreads();
    } else {
        fewer_regs<kMmaRegs>();
        if (warp == 12 && lane == 0 && total > 0) {
            // ---------------- MMA issuer
            constexpr uint32_t id = idesc_f16(kRows, 128);
            const int users = blocks[1] > 0 ? 2 : 1;  // tile 1 walks at least as far as tile 0
            bool ok = true;
            auto issue_s = [&](int t, int j) {
                const int st = j % kStages;
                ok = ok && mbar_wait(&sh.k_full[st], (j / kStages) & 1, a.err, 908);
                if (!ok) return;
                tc_fence_after();
                const uint32_t aQ = smem_u32(sQ + t * kTile), aK = smem_u32(sK + st * kTile);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    umma_bf16(tmem + t * 128, umma_desc_sw128(aQ + (k >> 2) * kHalfTile + (k & 3) * 32),
                              umma_desc_sw128(aK + (k >> 2) * kHalfTile + (k & 3) * 32), id, k > 0 ? 1u : 0u);
                umma_commit(&sh.s_full[t]);
                if (t == users - 1) umma_commit(&sh.k_empty[st]);
            };
            for (int t = 0; t < users && ok; ++t)
                if (blocks[t] > 0) {
                    ok = mbar_wait(&sh.q_full[t], 0, a.err, 905);
                    if (ok) issue_s(t, 0);
                }
            for (int j = 0; j < total && ok; ++j) {
                const int st = j % kStages;
                for (int t = 0; t < users && ok; ++t) {
                    if (j >= blocks[t]) continue;
                    ok = mbar_wait(&sh.v_full[st], (j / kStages) & 1, a.err, 909) && mbar_wait(&sh.p_full[t], j & 1, a.err, 906);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t aV = smem_u32(sV + st * kTile), tP = tmem + t * 128, tO = tmem + 256 + t * 128;
#pragma unroll
                    for (int k = 0; k < 8; ++k)  // 16 keys each: 8 columns of p
                        umma_bf16_ta(tO, tP + k * 8, umma_desc_sw128(aV + (k >> 2) * kHalfTile + (k & 3) * 32), id,
                                     (j > 0 || k > 0) ? 1u : 0u);
                    umma_commit(&sh.o_done[t]);
                    if (t == users - 1) umma_commit(&sh.v_empty[st]);
                    if (j + 1 < blocks[t]) {  // p is read once PV is done: then its columns take the next S
                        ok = mbar_wait(&sh.o_done[t], j & 1, a.err, 907);
                        if (ok) issue_s(t, j + 1);
                    }
                }
            }
        }
        __syncwarp();
        __syncthreads();
    }
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace

int launch_attend_chunk(const Kv8AttnArgs& a, msgl_stream_t stream) {
    static std::atomic<int> optin[kMaxDevices];
    const cudaError_t e = smem_optin(attend_chunk_kernel, kSmem, optin);
    if (e != cudaSuccess) return set_error(MSGL_ERR_CUDA, cudaGetErrorString(e));
    const int per_cta = 2 * kRows / (a.hq / a.hkv);
    const dim3 grid((a.max_q_len + per_cta - 1) / per_cta, a.hkv, a.num_reqs);
    launch_pdl(attend_chunk_kernel, grid, dim3(kThreads), kSmem, stream, a);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

}  // namespace msgl
