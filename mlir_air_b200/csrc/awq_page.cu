// The paged cache of many requests: a step's plan (pages, slots, positions, ancestor masks), RoPE into the cache, and the
// accepted tokens of a step kept.  All three move a few bytes to a few hundred megabytes and compute next to nothing: they
// are bound by the latency of one launch, or by memory.
#include "awq_request.cuh"

#include <cuda_fp16.h>

namespace awq {

int check_kv_cache(const char *who, const awq_b200_kv_cache_t *c, KvCacheView *out) {
    AWQ_REQUIRE(c && c->k && c->v, "%s: null cache", who);
    AWQ_REQUIRE(c->format == ACT_BF16 || c->format == ACT_F16, "%s: unknown cache format %d", who, c->format);
    AWQ_REQUIRE(c->n_pages > 0 && c->page_size > 0 && c->n_kv_heads > 0 && c->head_dim > 0, "%s: bad cache size", who);
    AWQ_REQUIRE((long long)c->n_pages * c->page_size <= 0x7fffffffLL, "%s: the cache has more than 2^31 - 1 slots", who);
    AWQ_REQUIRE(c->head_dim % 16 == 0 && c->head_dim <= 256, "%s: head_dim (%d) must be a multiple of 16, at most 256", who, c->head_dim);
    AWQ_REQUIRE(aligned16(c->k) && aligned16(c->v), "%s: the cache must be 16-byte aligned", who);
    const long long s[6] = {c->k_page_stride, c->k_slot_stride, c->k_head_stride, c->v_page_stride, c->v_slot_stride, c->v_head_stride};
    for (long long v : s) AWQ_REQUIRE(v >= 0 && v % 8 == 0, "%s: cache strides must be multiples of 8 elements", who);
    // (the stride of a dimension of one is never used; a box of a tensor map cannot have one of 0)
    const int n[3] = {c->n_pages, c->page_size, c->n_kv_heads};
    for (int i = 0; i < 6; ++i) AWQ_REQUIRE(s[i] > 0 || n[i % 3] == 1, "%s: a cache stride of 0 needs a dimension of one", who);
    *out = KvCacheView{reinterpret_cast<const uint16_t *>(c->k), reinterpret_cast<const uint16_t *>(c->v), s[0], s[1], s[2], s[3], s[4], s[5],
                       c->n_pages, c->page_size, c->n_kv_heads, c->head_dim};
    return AWQ_OK;
}

// Pages of `tokens` tokens: both below 2^31, their sum need not be.
__device__ __forceinline__ int pages_of(int tokens, int page) { return (int)(((unsigned)tokens + (unsigned)page - 1u) / (unsigned)page); }

// Exclusive sums of a pair over the block's threads (256), and the totals.
__device__ __forceinline__ void block_scan_pair(long long &a, long long &b, long long &total_a, long long &total_b) {
    __shared__ long long sa[8], sb[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long ia = a, ib = b;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long ua = __shfl_up_sync(0xffffffffu, ia, d), ub = __shfl_up_sync(0xffffffffu, ib, d);
        if (lane >= d) ia += ua, ib += ub;
    }
    __syncthreads();
    if (lane == 31) sa[warp] = ia, sb[warp] = ib;
    __syncthreads();
    long long ba = 0, bb = 0;
    total_a = total_b = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        if (w < warp) ba += sa[w], bb += sb[w];
        total_a += sa[w], total_b += sb[w];
    }
    a = ba + ia - a;
    b = bb + ib - b;
}

// =====================================================================================
// page_plan.  held = ceil(len / page), need = ceil((len + new) / page) - held; the free pages are a stack of which the
// requests take their new pages one request after another, topmost first.  Row t is token j of its request and goes to
// slot table[r][(len + j) / page] * page + (len + j) % page.  In a tree the bits of token j are those of its parent and
// bit j, its position is the length plus the number of its ancestors.
//
// Every CTA scans all requests (two sums over at most 4096 pairs) and then works on its share of the rows and of the new
// pages: a second launch or a wait between CTAs would cost more than the scan.  The step goes through whole or not at all.
// Measured: 4 requests 3.8 us, 512 requests with trees 6 us: launch, lengths, scan.
// =====================================================================================
constexpr int PLAN_THREADS = 256;
struct PlanArgs {
    const int32_t *lens, *fresh;
    int32_t *table;
    long long table_stride;
    const int32_t *free_pages, *count, *parents;
    int32_t *count_out, *q_start, *slots, *positions;
    long long *mask;
    int R, T, table_width, pool, page, max_pages;  // max_pages: as many as int32 slots can number
    RequestHeader *header;
};

__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(PlanArgs a) {
    extern __shared__ int plan_smem[];
    int *start = plan_smem, *first = plan_smem + a.R + 1;  // [R + 1] each: rows, new pages before request r
    const int tid = threadIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    const int count = *a.count;
    // a thread takes consecutive requests, so that one scan over the threads is enough
    const int per = (a.R + PLAN_THREADS - 1) / PLAN_THREADS, r0 = min(tid * per, a.R), r1 = min(r0 + per, a.R);
    const long long capacity = (long long)a.table_width * a.page;
    long long rows = 0, need = 0;
    bool bad = false;
    for (int r = r0; r < r1; ++r) {
        const int len = a.lens[r], n = a.fresh[r];
        if (len < 0 || n < 0 || (long long)len + n > capacity || (a.parents && n > REQ_MAX_TREE)) {
            bad = true;
            continue;
        }
        rows += n;
        need += pages_of(len + n, a.page) - pages_of(len, a.page);
    }
    long long all_rows, all_need;
    block_scan_pair(rows, need, all_rows, all_need);
    bad = __syncthreads_or(bad) || all_rows > a.T || count < 0 || count > a.pool;
    const bool short_of_pages = !bad && all_need > count;
    const bool refused = bad || short_of_pages;
    if (tid == 0 && blockIdx.x == 0 && refused) req_error(&a.header->error, bad ? REQ_ERR_STEP : REQ_ERR_NO_PAGES);
    if (!refused) {
        for (int r = r0; r < r1; ++r) {
            const int len = a.lens[r], n = a.fresh[r];
            start[r] = (int)rows;
            first[r] = (int)need;
            rows += n;
            need += pages_of(len + n, a.page) - pages_of(len, a.page);
        }
        if (tid == 0) start[a.R] = (int)all_rows, first[a.R] = (int)all_need;
    } else {
        for (int r = tid; r <= a.R; r += PLAN_THREADS) start[r] = first[r] = 0;
        all_rows = all_need = 0;
    }
    __syncthreads();
    const int step = gridDim.x * PLAN_THREADS, me = blockIdx.x * PLAN_THREADS + tid;
    for (int r = me; r <= a.R; r += step) a.q_start[r] = start[r];
    for (int k = me; k < (int)all_need; k += step) {
        const int r = request_of_row(first, a.R, k);
        int page = a.free_pages[count - 1 - k];
        if ((unsigned)page >= (unsigned)a.max_pages) {
            req_error(&a.header->error, REQ_ERR_PAGE);
            page = -1;
        }
        a.table[r * a.table_stride + pages_of(a.lens[r], a.page) + k - first[r]] = page;
    }
    for (int t = me; t < a.T; t += step) {
        if (t >= (int)all_rows) {  // rows behind the last request
            a.slots[t] = -1;
            a.positions[t] = 0;
            if (a.mask) a.mask[t] = 0;
            continue;
        }
        const int r = request_of_row(start, a.R, t), j = t - start[r], len = a.lens[r];
        const int at = len + j, block = at / a.page, held = pages_of(len, a.page);
        // a new page is not read from the table, which another CTA may not have written yet
        int page = block < held ? a.table[r * a.table_stride + block] : a.free_pages[count - 1 - (first[r] + block - held)];
        if ((unsigned)page >= (unsigned)a.max_pages) {
            req_error(&a.header->error, REQ_ERR_PAGE);
            page = -1;
        }
        a.slots[t] = page < 0 ? -1 : page * a.page + at % a.page;
        int position = at;
        if (a.parents) {
            unsigned long long bits = 1ull << j;
            int p = j;
            position = len;
            while (true) {
                const int up = a.parents[start[r] + p];
                if (up == -1) break;
                if (up < 0 || up >= p) {
                    req_error(&a.header->error, REQ_ERR_PARENT);
                    break;
                }
                p = up;
                bits |= 1ull << p;
                ++position;
            }
            a.mask[t] = (long long)bits;
        }
        a.positions[t] = position;
    }
    // every CTA has read the count before the last one writes it (count_out may be count)
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        if (atomicAdd(&a.header->plan_arrived, 1) == (int)gridDim.x - 1) {
            a.header->plan_arrived = 0;
            *a.count_out = count - (int)all_need;
        }
    }
}

// =====================================================================================
// rope_append.  Row t: Q and K rotated by the [cos | sin] row of its position (halves of a head against each other, products
// and sums in f32, one rounding, as in rope_halfsplit), K and V written to its slot.  A row whose slot is -1 is left out.
// A slot that several rows name keeps the last of them, whatever order the CTAs run in: each row looks through the
// slots behind its own.
// Measured: one row 2.5 us; 8 prompts of 333 to 1999 tokens, 32/8 heads of 128 (227 MB read and written), 44 us, 5.1 TB/s (34.5 us at a
// copy's rate).  The look through later slots is quadratic: 16000 rows take 78 us (60 for the bytes), 32000 179 (120), 64000 498 (240).
// =====================================================================================
constexpr int RA_THREADS = 128;
struct AppendArgs {
    const uint16_t *q, *k, *v, *lut;
    long long q_row, q_head, k_row, k_head, v_row, v_head;
    const int32_t *positions, *slots;
    uint16_t *q_out;
    long long o_row, o_head;
    KvCacheView cache;
    int T, n_heads, n_positions;
    RequestHeader *header;
};

template <bool F16>
__device__ __forceinline__ void rope_pair(const uint4 &a4, const uint4 &b4, const uint4 &c4, const uint4 &s4, uint4 &o1, uint4 &o2) {
    const uint32_t a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
    const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
    uint32_t u[4], w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 x = unpack16x2<F16>(a[e]), y = unpack16x2<F16>(b[e]);
        const float2 co = make_float2(bf16x2_lo(c[e]), bf16x2_hi(c[e])), si = make_float2(bf16x2_lo(s[e]), bf16x2_hi(s[e]));
        u[e] = pack16x2<F16>(__fsub_rn(__fmul_rn(x.x, co.x), __fmul_rn(y.x, si.x)), __fsub_rn(__fmul_rn(x.y, co.y), __fmul_rn(y.y, si.y)));
        w[e] = pack16x2<F16>(__fadd_rn(__fmul_rn(x.x, si.x), __fmul_rn(y.x, co.x)), __fadd_rn(__fmul_rn(x.y, si.y), __fmul_rn(y.y, co.y)));
    }
    o1 = make_uint4(u[0], u[1], u[2], u[3]);
    o2 = make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool F16>
__global__ void __launch_bounds__(RA_THREADS, 10) rope_append_kernel(AppendArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int t = blockIdx.x;
    const int slot = a.slots[t], position = a.positions[t];
    if (slot == -1) return;
    const int n_slots = a.cache.n_pages * a.cache.page_size;
    if ((unsigned)slot >= (unsigned)n_slots || (unsigned)position >= (unsigned)a.n_positions) {
        if (threadIdx.x == 0) req_error(&a.header->error, REQ_ERR_SLOT);
        return;
    }
    bool later = false;
    for (int i = t + 1 + threadIdx.x; i < a.T; i += RA_THREADS) later |= a.slots[i] == slot;
    // A row that is left out for its position takes no slot from others.  (Looked up in the loop above, 44.4 us become 48.6; here too, with the
    // 64 registers that the kernel takes if it may.)
    if (__syncthreads_or(later)) {
        later = false;
#pragma unroll 1
        for (int i = t + 1 + threadIdx.x; i < a.T; i += RA_THREADS)
            later |= a.slots[i] == slot && (unsigned)a.positions[i] < (unsigned)a.n_positions;
        later = __syncthreads_or(later);
    }
    const int D = a.cache.head_dim, half = D >> 1, chunks = half >> 3;
    const int page = slot / a.cache.page_size, off = slot - page * a.cache.page_size;
    uint16_t *kd = const_cast<uint16_t *>(a.cache.k) + page * a.cache.k_page + off * a.cache.k_slot;
    uint16_t *vd = const_cast<uint16_t *>(a.cache.v) + page * a.cache.v_page + off * a.cache.v_slot;
    const int items = (a.n_heads + 2 * a.cache.n_kv) * chunks;
    for (int i = threadIdx.x; i < items; i += RA_THREADS) {
        const int c = i % chunks;
        int h = i / chunks;
        const uint16_t *src;
        uint16_t *dst;
        bool turn = true;
        if (h < a.n_heads) {
            src = a.q + t * a.q_row + h * a.q_head;
            dst = a.q_out + t * a.o_row + h * a.o_head;
        } else {
            if (later) continue;
            h -= a.n_heads;
            if (h < a.cache.n_kv) {
                src = a.k + t * a.k_row + h * a.k_head;
                dst = kd + h * a.cache.k_head;
            } else {
                h -= a.cache.n_kv;
                src = a.v + t * a.v_row + h * a.v_head;
                dst = vd + h * a.cache.v_head;
                turn = false;
            }
        }
        uint4 lo = *reinterpret_cast<const uint4 *>(src + 8 * c), hi = *reinterpret_cast<const uint4 *>(src + 8 * c + half);
        if (turn) {
            const uint16_t *l = a.lut + (long long)position * D + 8 * c;
            uint4 o1, o2;
            rope_pair<F16>(lo, hi, *reinterpret_cast<const uint4 *>(l), *reinterpret_cast<const uint4 *>(l + half), o1, o2);
            lo = o1;
            hi = o2;
        }
        *reinterpret_cast<uint4 *>(dst + 8 * c) = lo;
        *reinterpret_cast<uint4 *>(dst + 8 * c + half) = hi;
    }
}

// =====================================================================================
// page_keep.  The i-th kept row of a request moves from len + path[i] to len + i in every layer.  path ascends, so
// path[i] >= i: a thread that owns some columns of all of a request's rows and moves them in order overwrites nothing that
// is still wanted.  Then len += kept, and the pages behind the new length go back onto the stack of free pages; the last
// CTA to finish does that, when no CTA needs the old lengths any more.  A request that keeps nothing because its count or path is
// wrong gives its new pages back; one whose rows or lengths are wrong is left as it is, pages and all.
// Measured: one request, 16 layers, 6.4 us; 32 requests of 6 to 32 tokens, 5 kept, 8 layers, 8.4 us: paths, pages, rows and the last CTA's
// turn one after another (the bytes alone 1.6 us).
// =====================================================================================
constexpr int KEEP_THREADS = 256;
struct KeepArgs {
    uint16_t *kv;
    long long s_layer, s_kv, s_page, s_slot, s_head;
    const int32_t *table;
    long long table_stride;
    const int32_t *lens, *q_start, *kept, *path;
    int32_t *lens_out, *free_pages, *count_out;
    const int32_t *count;
    int R, T, table_width, pool, n_pages, page, layers, n_kv, head_dim;
    RequestHeader *header;
};

struct KeepRequest {
    int len, fresh, kept, start;
    bool ends, bad, unknown;  // unknown: its lengths or rows are not what the buffers hold; nothing of it is touched
};
__device__ __forceinline__ KeepRequest keep_request(const KeepArgs &a, int r) {
    KeepRequest q;
    q.len = a.lens[r];
    q.start = a.q_start[r];
    const int end = a.q_start[r + 1];
    q.fresh = end - q.start;
    q.kept = a.kept[r];
    q.ends = q.kept == -1;
    q.unknown = q.len < 0 || q.start < 0 || q.fresh < 0 || end > a.T || (long long)q.len + q.fresh > (long long)a.table_width * a.page;
    q.bad = q.unknown || q.kept < -1 || q.kept > q.fresh || (a.path && q.kept > REQ_MAX_TREE);
    if (q.bad || q.ends) q.kept = 0;
    return q;
}
// Whether the path of a request ascends and stays inside its rows (kept <= 64): called by a whole warp.
__device__ __forceinline__ bool keep_path_ok(const KeepArgs &a, const KeepRequest &q, int lane) {
    bool ok = true;
    for (int i = lane; i < q.kept; i += 32) {
        const int p = a.path[q.start + i];
        ok = ok && p >= 0 && p < q.fresh && (i == 0 || a.path[q.start + i - 1] < p);
    }
    return __all_sync(0xffffffffu, ok);
}

__global__ void __launch_bounds__(KEEP_THREADS) page_keep_kernel(KeepArgs a) {
    __shared__ long long src[REQ_MAX_TREE], dst[REQ_MAX_TREE];
    __shared__ int last, path_ok;
    const int tid = threadIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    if (a.path) {
        for (long long item = blockIdx.x; item < (long long)a.R * a.layers * 2; item += gridDim.x) {
            const int r = (int)(item / (a.layers * 2)), lk = (int)(item % (a.layers * 2));
            const KeepRequest q = keep_request(a, r);
            if (q.kept == 0) continue;
            __syncthreads();
            if (tid < 32) {
                const bool ok = keep_path_ok(a, q, tid);
                if (tid == 0) path_ok = ok;
            }
            __syncthreads();
            if (!path_ok) continue;
            if (tid < q.kept) {
                const int from = q.len + a.path[q.start + tid], to = q.len + tid;
                const int pf = a.table[r * a.table_stride + from / a.page], pt = a.table[r * a.table_stride + to / a.page];
                const bool bad = (unsigned)pf >= (unsigned)a.n_pages || (unsigned)pt >= (unsigned)a.n_pages;
                if (bad) req_error(&a.header->error, REQ_ERR_PAGE);
                src[tid] = bad || from == to ? -1 : pf * a.s_page + (from % a.page) * a.s_slot;
                dst[tid] = pt * a.s_page + (to % a.page) * a.s_slot;
            }
            __syncthreads();
            uint16_t *base = a.kv + (lk >> 1) * a.s_layer + (lk & 1) * a.s_kv;
            const int per_head = a.head_dim >> 3;
            for (int c = tid; c < a.n_kv * per_head; c += KEEP_THREADS) {
                uint16_t *column = base + (c / per_head) * a.s_head + 8 * (c % per_head);
                for (int i = 0; i < q.kept; ++i)
                    if (src[i] >= 0) *reinterpret_cast<uint4 *>(column + dst[i]) = *reinterpret_cast<const uint4 *>(column + src[i]);
            }
        }
    }
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        last = atomicAdd(&a.header->keep_arrived, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    extern __shared__ int keep_smem[];
    int *first = keep_smem, *after = keep_smem + a.R + 1;  // [R + 1] pages freed before request r; its new length
    const int per = (a.R + KEEP_THREADS - 1) / KEEP_THREADS, r0 = min(tid * per, a.R), r1 = min(r0 + per, a.R);
    const int count = *a.count;
    long long gone = 0, unused = 0, all_gone, all_unused;
    for (int r = r0; r < r1; ++r) {
        KeepRequest q = keep_request(a, r);
        for (int i = 0; a.path && i < q.kept; ++i) {
            const int p = a.path[q.start + i];
            q.bad = q.bad || p < 0 || p >= q.fresh || (i > 0 && a.path[q.start + i - 1] >= p);
        }
        if (q.bad) req_error(&a.header->error, REQ_ERR_KEPT);
        after[r] = q.unknown ? q.len : q.ends ? 0 : q.len + (q.bad ? 0 : q.kept);
        first[r] = q.unknown ? 0 : pages_of(q.len + q.fresh, a.page) - pages_of(after[r], a.page);
        gone += first[r];
    }
    block_scan_pair(gone, unused, all_gone, all_unused);
    for (int r = r0; r < r1; ++r) {
        const int n = first[r];
        first[r] = (int)gone;
        gone += n;
    }
    const bool fits = count >= 0 && all_gone <= (long long)a.pool - count;
    if (tid == 0) {
        first[a.R] = (int)all_gone;
        if (!fits) req_error(&a.header->error, REQ_ERR_KEPT);
    }
    __syncthreads();
    for (int k = tid; fits && k < (int)all_gone; k += KEEP_THREADS) {
        const int r = request_of_row(first, a.R, k);
        a.free_pages[count + k] = a.table[r * a.table_stride + pages_of(after[r], a.page) + k - first[r]];
    }
    for (int r = r0; r < r1; ++r) a.lens_out[r] = after[r];
    if (tid == 0) {
        *a.count_out = fits ? count + (int)all_gone : count;
        a.header->keep_arrived = 0;
    }
}

}  // namespace awq

using namespace awq;

extern "C" size_t awq_b200_request_workspace_bytes(void) { return request_workspace_bytes(); }

extern "C" int awq_b200_request_check(void *workspace, awq_stream_t stream) {
    AWQ_REQUIRE(workspace, "request_check: null workspace");
    int flag = 0;
    int rc = check_cuda(cudaMemcpyAsync(&flag, workspace, sizeof(int), cudaMemcpyDeviceToHost, as_stream(stream)), "request_check copy");
    if (rc) return rc;
    if ((rc = check_cuda(cudaStreamSynchronize(as_stream(stream)), "request_check sync"))) return rc;
    if (flag == 0) return AWQ_OK;
    if ((rc = check_cuda(cudaMemsetAsync(workspace, 0, sizeof(int), as_stream(stream)), "request_check clear"))) return rc;
    if (flag & REQ_ERR_TIMEOUT)
        return set_error(AWQ_ERR_DEVICE_TIMEOUT, "tree_attention: a device-side wait gave up; re-initialise the workspace");
    return set_error(AWQ_ERR_INVALID_ARGUMENT, "an operator on requests met what its buffers do not hold (its results are not valid):%s%s%s%s%s%s%s%s",
                     flag & REQ_ERR_NO_PAGES ? " page_plan: not enough free pages, the step was not planned;" : "",
                     flag & REQ_ERR_STEP ? " page_plan: lengths or counts beyond the batch, the block table or 64 tokens of a tree, the step was not planned;" : "",
                     flag & REQ_ERR_PARENT ? " page_plan: a parent that is not an earlier token of its tree;" : "",
                     flag & REQ_ERR_PAGE ? " a page outside the cache;" : "",
                     flag & REQ_ERR_SLOT ? " rope_append: a slot outside the cache or a position outside the table of angles;" : "",
                     flag & REQ_ERR_KEPT ? " page_keep: a count or path that does not fit its request;" : "",
                     flag & REQ_ERR_ADAPTER ? " lora: an adapter that does not exist;" : "",
                     flag & REQ_ERR_REQUEST ? " tree_attention: lengths or starts beyond the batch, the block table or 64 tokens of a tree;" : "");
}

extern "C" int awq_b200_page_plan(const int32_t *lens, const int32_t *fresh, int32_t *table, long long table_stride, int table_width,
                                  const int32_t *free_pages, int pool, const int32_t *free_count, int32_t *free_count_out,
                                  const int32_t *parents, int page_size, int32_t *q_start, int32_t *slots, int32_t *positions,
                                  long long *mask, int R, int T, void *workspace, size_t workspace_bytes, awq_stream_t stream) {
    AWQ_REQUIRE(R >= 0 && T >= 0 && table_width >= 0 && pool >= 0, "page_plan: negative size");
    AWQ_REQUIRE(R <= REQ_MAX_REQUESTS && T <= REQ_MAX_ROWS, "page_plan: at most %d requests and %d rows", REQ_MAX_REQUESTS, REQ_MAX_ROWS);
    AWQ_REQUIRE(page_size > 0 && (long long)pool * page_size <= 0x7fffffffLL && (long long)table_width * page_size <= 0x7fffffffLL,
                "page_plan: page_size must be positive and the cache below 2^31 slots");
    AWQ_REQUIRE(table_stride >= table_width, "page_plan: the stride of the block table is below its width");
    AWQ_REQUIRE(q_start && free_count && free_count_out, "page_plan: null pointer");
    AWQ_REQUIRE(R == 0 || (lens && fresh && table && free_pages), "page_plan: null pointer");
    AWQ_REQUIRE(T == 0 || (slots && positions), "page_plan: null pointer");
    AWQ_REQUIRE((parents == nullptr) == (mask == nullptr), "page_plan: parents and mask go together");
    AWQ_REQUIRE_REQUEST_WORKSPACE("page_plan", workspace, workspace_bytes);
    PlanArgs a{lens, fresh, table, table_stride, free_pages, free_count, parents, free_count_out, q_start, slots, positions, mask, R, T,
               table_width, pool, page_size, 0x7fffffff / page_size, request_workspace(workspace).header};
    const int grid = max(1, min((T + PLAN_THREADS - 1) / PLAN_THREADS, device_sm_count()));
    return check_cuda(launch_pdl(page_plan_kernel, dim3(grid), dim3(PLAN_THREADS), (size_t)(2 * R + 2) * 4, as_stream(stream), a), "page_plan launch");
}

extern "C" int awq_b200_rope_append(const void *q, long long q_row_stride, long long q_head_stride, const void *k, long long k_row_stride,
                                    long long k_head_stride, const void *v, long long v_row_stride, long long v_head_stride,
                                    const uint16_t *lut, int n_positions, const int32_t *positions, const int32_t *slots, void *q_out,
                                    long long q_out_row_stride, long long q_out_head_stride, const awq_b200_kv_cache_t *cache, int T,
                                    int n_heads, void *workspace, size_t workspace_bytes, awq_stream_t stream) {
    KvCacheView view;
    int rc = check_kv_cache("rope_append", cache, &view);
    if (rc) return rc;
    AWQ_REQUIRE(T >= 0 && T <= REQ_MAX_ROWS && n_heads >= 0 && n_positions > 0, "rope_append: bad size");
    const long long s[8] = {q_row_stride, q_head_stride, k_row_stride, k_head_stride, v_row_stride, v_head_stride, q_out_row_stride, q_out_head_stride};
    for (long long x : s) AWQ_REQUIRE(x >= 0 && x % 8 == 0, "rope_append: strides must be multiples of 8 elements");
    if (T == 0) return AWQ_OK;
    AWQ_REQUIRE((T == 1 || q_out_row_stride > 0) && (n_heads <= 1 || q_out_head_stride > 0), "rope_append: an output stride of 0 needs a dimension of one");
    AWQ_REQUIRE(q && k && v && lut && positions && slots && q_out, "rope_append: null pointer");
    AWQ_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(lut) && aligned16(q_out), "rope_append: pointers must be 16-byte aligned");
    AWQ_REQUIRE_REQUEST_WORKSPACE("rope_append", workspace, workspace_bytes);
    AppendArgs a{reinterpret_cast<const uint16_t *>(q), reinterpret_cast<const uint16_t *>(k), reinterpret_cast<const uint16_t *>(v), lut,
                 s[0], s[1], s[2], s[3], s[4], s[5], positions, slots, reinterpret_cast<uint16_t *>(q_out), s[6], s[7], view, T, n_heads, n_positions,
                 request_workspace(workspace).header};
    auto kernel = cache->format == ACT_F16 ? rope_append_kernel<true> : rope_append_kernel<false>;
    return check_cuda(launch_pdl(kernel, dim3(T), dim3(RA_THREADS), 0, as_stream(stream), a), "rope_append launch");
}

extern "C" int awq_b200_page_keep(void *kv, long long layer_stride, long long kv_stride, long long page_stride, long long slot_stride,
                                  long long head_stride, int layers, int n_pages, int page_size, int n_kv_heads, int head_dim,
                                  const int32_t *table, long long table_stride, int table_width, const int32_t *lens, int32_t *lens_out,
                                  const int32_t *q_start, const int32_t *kept, const int32_t *path, int32_t *free_pages, int pool,
                                  const int32_t *free_count, int32_t *free_count_out, int R, int T, void *workspace,
                                  size_t workspace_bytes, awq_stream_t stream) {
    AWQ_REQUIRE(R >= 0 && R <= REQ_MAX_REQUESTS && T >= 0 && T <= REQ_MAX_ROWS && table_width >= 0 && pool >= 0, "page_keep: bad size");
    AWQ_REQUIRE(layers >= 0 && layers <= 4096 && n_pages > 0 && page_size > 0 && n_kv_heads > 0 && head_dim > 0 && head_dim % 8 == 0,
                "page_keep: bad cache size");
    AWQ_REQUIRE((long long)n_pages * page_size <= 0x7fffffffLL && (long long)table_width * page_size <= 0x7fffffffLL,
                "page_keep: the cache has more than 2^31 - 1 slots");
    AWQ_REQUIRE(table_stride >= table_width, "page_keep: the stride of the block table is below its width");
    const long long s[5] = {layer_stride, kv_stride, page_stride, slot_stride, head_stride};
    for (long long x : s) AWQ_REQUIRE(x >= 0 && x % 8 == 0, "page_keep: strides must be multiples of 8 elements");
    AWQ_REQUIRE(free_count && free_count_out, "page_keep: null pointer");
    AWQ_REQUIRE(R == 0 || (table && lens && lens_out && q_start && kept && free_pages), "page_keep: null pointer");
    AWQ_REQUIRE(!path || kv, "page_keep: a path needs the cache");
    const int n[5] = {layers, 2, n_pages, page_size, n_kv_heads};
    for (int i = 0; path && i < 5; ++i) AWQ_REQUIRE(s[i] > 0 || n[i] <= 1, "page_keep: a stride of 0 needs a dimension of one");
    AWQ_REQUIRE(aligned16(kv), "page_keep: the cache must be 16-byte aligned");
    AWQ_REQUIRE_REQUEST_WORKSPACE("page_keep", workspace, workspace_bytes);
    KeepArgs a{reinterpret_cast<uint16_t *>(kv), s[0], s[1], s[2], s[3], s[4], table, table_stride, lens, q_start, kept, path, lens_out, free_pages,
               free_count_out, free_count, R, T, table_width, pool, n_pages, page_size, layers, n_kv_heads, head_dim,
               request_workspace(workspace).header};
    const long long items = path ? (long long)R * layers * 2 : 1;
    const int grid = (int)max(1LL, min(items, 4096LL));
    return check_cuda(launch_pdl(page_keep_kernel, dim3(grid), dim3(KEEP_THREADS), (size_t)(2 * R + 1) * 4, as_stream(stream), a), "page_keep launch");
}
