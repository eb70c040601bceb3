// batch.cu -- device-side decode batch metadata.
//
//  * msgl_decode_advance   the decode branch of Scheduler::step's host flatten
//                          (src/scheduler/scheduler.cpp:83-106: input ids, positions) plus the
//                          slot formula of launch_store_kv_page (kernels/cuda/radix.cu:19-22)
//                          and KVCachePool::allocate (src/cache/kvcache.cpp:21-28, LIFO pops)
//                          for the page a request enters, all on the device, so consecutive
//                          decode steps need no host page tables and no host-to-device copies.
//
//  * msgl_decode_advance_masked / msgl_decode_finish
//                          the same with finished requests held in place, and the stop rules
//                          (max_tokens, stop ids, ignore_eos) applied on the device.
//
//  * msgl_step_tables      a step of any rows per request (chunks, drafted tokens, none): pages
//                          given back and taken, page table, row ranges, positions and slots.
//
// One CTA of up to 1024 threads walks the requests in blocks of blockDim; a block-wide scan
// gives each request that starts a new page its rank among this step's allocations, so pages
// leave the free stack in request order, as the host pool hands them out. The step is
// all-or-nothing: if the free stack cannot serve every new page, or a new page would land past
// the page-table width, nothing is written and the error word records why.
#include "common.cuh"

namespace msgl {
namespace {

constexpr int kAdvThreads = 1024;

// finished (optional, [B]): requests with a nonzero entry are held where they are -- no page,
// no new position, same input id -- so the next step recomputes their last step (writing the
// same K/V to the same slot) and their output is ignored.
__global__ void __launch_bounds__(kAdvThreads)
decode_advance_kernel(const int* __restrict__ next_tokens, int* __restrict__ input_ids,
                      int* __restrict__ positions, int* __restrict__ slot_mapping,
                      int* __restrict__ page_table, int max_pages, int* __restrict__ seq_lens,
                      const int* __restrict__ free_pages, int* __restrict__ free_top, int B,
                      int page_size, const int* __restrict__ finished, int* err) {
    __shared__ int sh[32];
    __shared__ int bad;
    pdl_wait();
    pdl_trigger();
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    const int top = *free_top;
    // pass 1: count the new pages and check every request (no writes)
    int base = 0;
    for (int r0 = 0; r0 < B; r0 += blockDim.x) {
        const int r = r0 + threadIdx.x;
        int need = 0;
        if (r < B && !(finished && finished[r])) {
            const int L = seq_lens[r];  // tokens in the cache after this step's token is added
            need = (L % page_size) == 0;
            if (L < 0 || L / page_size >= max_pages) atomicOr(&bad, 2);
        }
        int total;
        const int k = base + block_excl_scan(need, sh, total);
        if (need && top - 1 - k < 0) atomicOr(&bad, 1);
        base += total;
    }
    __syncthreads();
    if (bad) {
        if (threadIdx.x == 0) {
            if (bad & 2) record_error(err, MSGL_ERR_BOUNDS, 701);
            else record_error(err, MSGL_ERR_WORKSPACE, 700);
        }
        return;
    }
    // pass 2: pop pages in request order, write the next step's metadata
    base = 0;
    for (int r0 = 0; r0 < B; r0 += blockDim.x) {
        const int r = r0 + threadIdx.x;
        int need = 0, L = 0;
        const bool held = r < B && finished && finished[r];
        if (r < B && !held) {
            L = seq_lens[r];
            need = (L % page_size) == 0;
        }
        int total;
        const int k = base + block_excl_scan(need, sh, total);
        if (r < B && !held) {
            int* row = page_table + static_cast<int64_t>(r) * max_pages;
            const int pi = L / page_size;
            if (need) row[pi] = free_pages[top - 1 - k];
            input_ids[r] = next_tokens[r];
            positions[r] = L;
            slot_mapping[r] = row[pi] * page_size + L % page_size;
            seq_lens[r] = L + 1;
        }
        base += total;
    }
    if (threadIdx.x == 0) *free_top = top - base;
}

// Stop rules of one step (Scheduler::step, scheduler.cpp:126-131, with SamplingParams,
// types.h:12-20): a request that had not finished takes next_tokens[r] as its new token
// (token_out[r]), counts it, and finishes once it has generated max_new_tokens[r] tokens or,
// unless ignore_eos[r], when the token is one of the stop ids (the reference checks length
// only, D17). A request that had finished gets token_out[r] = -1.
__global__ void decode_finish_kernel(const int* __restrict__ next_tokens, int* __restrict__ token_out,
                                     const int* __restrict__ max_new_tokens,
                                     const int* __restrict__ ignore_eos,
                                     const int* __restrict__ stop_ids, int num_stop,
                                     int* __restrict__ finished, int* __restrict__ generated, int B) {
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.x * blockDim.x + threadIdx.x;
    if (r >= B) return;
    if (finished[r]) {
        token_out[r] = -1;
        return;
    }
    const int t = next_tokens[r];
    token_out[r] = t;
    const int g = generated[r] + 1;
    generated[r] = g;
    bool stop = g >= max_new_tokens[r];
    if (!(ignore_eos && ignore_eos[r]))
        for (int i = 0; i < num_stop; ++i) stop |= t == stop_ids[i];
    if (stop) finished[r] = 1;
}

// ------------------------------------------------------------------ step tables
// seq = kept + new, pages = ceil(seq / page). Requests that hold more pages than that give the others
// back (rejected drafts, finished requests), then requests that hold fewer take theirs; both in request
// order. A request's pages go back last column first, so that the next to be taken are in the order in
// which they were held. Latency bound: a scan of the requests, then one gather per row.
//
// One cluster. Its first CTA does what hangs on the order: three scans over the requests (pages given
// back, pages taken, rows) in one pass, then pages and rows are dealt to the threads by their place in
// the scans, so that one long prompt among single tokens costs no serial walk. All CTAs fill positions
// and slots: one up to 2048 rows, else eight (64 requests x 16 rows 9.6 us, with eight 10.8; x 33 rows 10.2, with one 11.2;
// 32k rows 12.0, with one 27.5).
constexpr int kStepThreads = 1024;

struct StepArgs {
    const int *kept, *add;
    int* table;
    int width;
    int* held;
    int* free_pages;
    int capacity;
    int* free_top;
    int B, tokens, page, shift;  // page = 2^shift, or shift < 0
    int *seq_lens, *indptr, *positions, *slots, *last;
    int* err;
};

// First index i of ends[0 .. n) (ascending) with ends[i] > x; n if there is none.
__device__ __forceinline__ int first_above(const int* ends, int n, int x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kStepThreads)
step_tables_kernel(const StepArgs a) {
    __shared__ int give_end[kStepThreads], take_end[kStepThreads], row_end[kStepThreads + 1];
    __shared__ int s_need[kStepThreads], s_kept[kStepThreads];
    __shared__ int warp_sums[3][32];
    __shared__ int bad;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = cluster_ctarank(), size = cluster_nctarank();
    if (tid == 0) bad = 0;
    pdl_wait();
    pdl_trigger();
    if (rank == 0) {
        const int blocks = (a.B + kStepThreads - 1) / kStepThreads;
        int give_all, take_all, rows_all;
        // Requests [r0, r0 + 1024): inclusive sums of pages given, taken and rows into shared memory.
        auto load = [&](int r0) {
            const int r = r0 + tid;
            int k = 0, n = 0, h = 0, need = 0, fault = 0;
            if (r < a.B) {
                k = a.kept[r];
                n = a.add[r];
                h = a.held[r];
                if (k < 0 || n < 0 || h < 0 || h > a.width ||
                    static_cast<int64_t>(k) + n > static_cast<int64_t>(a.width) * a.page) {
                    fault = 2;
                    k = n = h = 0;
                } else if (n > a.tokens) {
                    fault = 4;
                    k = n = h = 0;
                }
                need = (k + n + a.page - 1) / a.page;
            }
            int x[3] = {max(h - need, 0), max(need - h, 0), n};
#pragma unroll
            for (int o = 1; o < 32; o <<= 1)
#pragma unroll
                for (int v = 0; v < 3; ++v) {
                    const int y = __shfl_up_sync(0xffffffffu, x[v], o);
                    if (lane >= o) x[v] += y;
                }
            __syncthreads();  // the sums of the block before are no longer read, and `bad` is cleared
            if (fault) atomicOr(&bad, fault);
            if (lane == 31)
#pragma unroll
                for (int v = 0; v < 3; ++v) warp_sums[v][warp] = x[v];
            __syncthreads();
            if (warp < 3) {
                int t = warp_sums[warp][lane];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, t, o);
                    if (lane >= o) t += y;
                }
                warp_sums[warp][lane] = t;
            }
            __syncthreads();
#pragma unroll
            for (int v = 0; v < 3; ++v) x[v] += warp ? warp_sums[v][warp - 1] : 0;
            give_end[tid] = x[0];
            take_end[tid] = x[1];
            row_end[tid] = x[2];
            s_need[tid] = need;
            s_kept[tid] = k;
            give_all = warp_sums[0][31];
            take_all = warp_sums[1][31];
            rows_all = warp_sums[2][31];
            __syncthreads();
        };
        // pass 1: totals, every check; nothing is written
        const int top0 = *a.free_top;
        int64_t gives = 0, takes = 0, rows = 0;
        for (int blk = 0; blk < blocks; ++blk) {
            load(blk * kStepThreads);
            gives += give_all;
            takes += take_all;
            rows += rows_all;
        }
        if (tid == 0) {
            if (rows > a.tokens) bad |= 4;
            if (top0 < 0 || top0 + gives > a.capacity) bad |= 8;
            if (top0 + gives < takes) bad |= 1;
            if (bad)
                record_error(a.err, bad & 2 ? MSGL_ERR_BOUNDS : bad & 4 ? MSGL_ERR_BOUNDS
                                    : bad & 8 ? MSGL_ERR_BOUNDS : MSGL_ERR_WORKSPACE,
                             bad & 2 ? 711 : bad & 4 ? 712 : bad & 8 ? 713 : 710);
        }
        __syncthreads();
        if (!bad) {
            // pass 2: pages back onto the stack
            int top = top0;
            for (int blk = 0; blk < blocks && gives; ++blk) {
                if (blocks > 1) load(blk * kStepThreads);
                const int n = min(kStepThreads, a.B - blk * kStepThreads);
                for (int i = tid; i < give_all; i += kStepThreads) {
                    const int q = first_above(give_end, n, i);
                    const int c = s_need[q] + (give_end[q] - 1 - i);  // the last column first
                    a.free_pages[top + i] = a.table[static_cast<int64_t>(blk * kStepThreads + q) * a.width + c];
                }
                top += give_all;
            }
            __syncthreads();
            // pass 3: pages taken, the requests' outputs
            int row0 = 0;
            for (int blk = 0; blk < blocks; ++blk) {
                if (blocks > 1) load(blk * kStepThreads);
                const int r0 = blk * kStepThreads, n = min(kStepThreads, a.B - r0);
                for (int i = tid; i < take_all; i += kStepThreads) {
                    const int q = first_above(take_end, n, i);
                    const int c = s_need[q] - (take_end[q] - i);
                    a.table[static_cast<int64_t>(r0 + q) * a.width + c] = a.free_pages[top - 1 - i];
                }
                if (tid < n) {
                    const int end = row_end[tid], begin = tid ? row_end[tid - 1] : 0;
                    a.seq_lens[r0 + tid] = s_kept[tid] + end - begin;
                    a.held[r0 + tid] = s_need[tid];
                    a.indptr[r0 + tid + 1] = row0 + end;
                    a.last[r0 + tid] = end > begin ? row0 + end - 1 : -1;
                }
                top -= take_all;
                row0 += rows_all;
            }
            if (tid == 0) {
                a.indptr[0] = 0;
                *a.free_top = top;
            }
        }
    }
    __syncthreads();
    cluster_sync_all();  // the tables of the first CTA, and whether it wrote them
    int failed = bad;
    if (rank != 0) failed = __float_as_int(ld_dsmem_f32(mapa_shared(smem_u32(&bad), 0)));
    if (!failed) {
        // rows' request: ends and kept lengths in shared memory where they fit
        const int* ends = a.indptr + 1;
        const int* kept = a.kept;
        __syncthreads();
        if (a.B <= kStepThreads) {
            if (tid < a.B) {
                row_end[tid + 1] = ends[tid];
                s_kept[tid] = kept[tid];
            }
            if (tid == 0) row_end[0] = 0;
            __syncthreads();
            ends = row_end + 1;
            kept = s_kept;
        }
        const int total = ends[a.B - 1];
        for (int i = rank * kStepThreads + tid; i < a.tokens; i += size * kStepThreads) {
            int pos = 0, slot = -1;
            if (i < total) {
                const int r = first_above(ends, a.B, i);
                pos = kept[r] + i - (r ? ends[r - 1] : 0);
                const int column = a.shift >= 0 ? pos >> a.shift : pos / a.page;
                slot = a.table[static_cast<int64_t>(r) * a.width + column] * a.page + pos - column * a.page;
            }
            a.positions[i] = pos;
            a.slots[i] = slot;
        }
    }
    cluster_sync_all();  // the first CTA's shared memory was read
}

}  // namespace
}  // namespace msgl

using namespace msgl;

extern "C" {

int msgl_decode_advance(const int* next_tokens, int* input_ids, int* positions, int* slot_mapping,
                        int* page_table, int max_pages, int* seq_lens, const int* free_pages,
                        int* free_top, int num_reqs, int page_size, msgl_stream_t stream) {
    if (num_reqs < 0 || max_pages <= 0 || page_size <= 0)
        return set_error(MSGL_ERR_INVALID_ARG, "decode_advance: bad sizes");
    if (num_reqs == 0) return MSGL_OK;
    if (!next_tokens || !input_ids || !positions || !slot_mapping || !page_table || !seq_lens ||
        !free_pages || !free_top)
        return set_error(MSGL_ERR_INVALID_ARG, "decode_advance: null pointer");
    int* err = device_error_word();
    if (!err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    const int threads = num_reqs >= kAdvThreads ? kAdvThreads : ((num_reqs + 31) / 32) * 32;
    launch_pdl(decode_advance_kernel, dim3(1), dim3(threads), 0, stream, next_tokens, input_ids,
               positions, slot_mapping, page_table, max_pages, seq_lens, free_pages, free_top,
               num_reqs, page_size, static_cast<const int*>(nullptr), err);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

int msgl_decode_advance_masked(const int* next_tokens, int* input_ids, int* positions,
                               int* slot_mapping, int* page_table, int max_pages, int* seq_lens,
                               const int* free_pages, int* free_top, const int* finished,
                               int num_reqs, int page_size, msgl_stream_t stream) {
    if (num_reqs < 0 || max_pages <= 0 || page_size <= 0)
        return set_error(MSGL_ERR_INVALID_ARG, "decode_advance: bad sizes");
    if (num_reqs == 0) return MSGL_OK;
    if (!next_tokens || !input_ids || !positions || !slot_mapping || !page_table || !seq_lens ||
        !free_pages || !free_top)
        return set_error(MSGL_ERR_INVALID_ARG, "decode_advance: null pointer");
    int* err = device_error_word();
    if (!err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    const int threads = num_reqs >= kAdvThreads ? kAdvThreads : ((num_reqs + 31) / 32) * 32;
    launch_pdl(decode_advance_kernel, dim3(1), dim3(threads), 0, stream, next_tokens, input_ids,
               positions, slot_mapping, page_table, max_pages, seq_lens, free_pages, free_top,
               num_reqs, page_size, finished, err);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

int msgl_step_tables(const int* kept_lens, const int* new_lens, int* page_table, int max_pages, int* held_pages,
                     int* free_pages, int free_capacity, int* free_top, int num_reqs, int num_tokens,
                     int page_size, int* seq_lens, int* q_indptr, int* positions, int* slot_mapping,
                     int* last_idx, msgl_stream_t stream) {
    if (num_reqs < 0 || num_tokens < 0 || max_pages <= 0 || page_size <= 0 || free_capacity < 0)
        return set_error(MSGL_ERR_INVALID_ARG, "step_tables: bad sizes");
    if (num_tokens > 1 << 20 || static_cast<int64_t>(num_reqs) * max_pages > INT32_MAX ||
        static_cast<int64_t>(max_pages) * page_size > INT32_MAX)
        return set_error(MSGL_ERR_UNSUPPORTED_SHAPE, "step_tables: more than 2^20 rows, 2^31 page-table entries or 2^31 tokens a request");
    if (num_reqs == 0) return MSGL_OK;
    if (!kept_lens || !new_lens || !page_table || !held_pages || !free_pages || !free_top || !seq_lens ||
        !q_indptr || !last_idx || (num_tokens > 0 && (!positions || !slot_mapping)))
        return set_error(MSGL_ERR_INVALID_ARG, "step_tables: null pointer");
    if (seq_lens == kept_lens || seq_lens == new_lens)
        return set_error(MSGL_ERR_INVALID_ARG, "step_tables: seq_lens must not be an input");
    int shift = -1;
    if ((page_size & (page_size - 1)) == 0)
        for (shift = 0; 1 << shift < page_size;) ++shift;
    StepArgs a = {kept_lens, new_lens, page_table, max_pages, held_pages, free_pages, free_capacity, free_top,
                  num_reqs, num_tokens, page_size, shift, seq_lens, q_indptr, positions, slot_mapping, last_idx,
                  device_error_word()};
    if (!a.err) return set_error(MSGL_ERR_CUDA, "device error word unavailable");
    const int size = num_tokens > 2 * kStepThreads ? 8 : 1;
    launch_cluster(step_tables_kernel, size, kStepThreads, size, 0, stream, a);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

int msgl_decode_finish(const int* next_tokens, int* token_out, const int* max_new_tokens,
                       const int* ignore_eos, const int* stop_ids, int num_stop_ids, int* finished,
                       int* generated, int num_reqs, msgl_stream_t stream) {
    if (num_reqs < 0 || num_stop_ids < 0 || (num_stop_ids > 0 && !stop_ids))
        return set_error(MSGL_ERR_INVALID_ARG, "decode_finish: bad sizes");
    if (num_reqs == 0) return MSGL_OK;
    if (!next_tokens || !token_out || !max_new_tokens || !finished || !generated)
        return set_error(MSGL_ERR_INVALID_ARG, "decode_finish: null pointer");
    launch_pdl(decode_finish_kernel, dim3((num_reqs + 127) / 128), dim3(128), 0, stream,
               next_tokens, token_out, max_new_tokens, ignore_eos, stop_ids, num_stop_ids,
               finished, generated, num_reqs);
    MSGL_LAUNCH_CHECK();
    return MSGL_OK;
}

}  // extern "C"
