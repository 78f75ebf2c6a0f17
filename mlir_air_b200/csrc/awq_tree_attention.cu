// Attention of a step's rows over a paged cache.
//
//   out[t, h] = sum_p w_p v_p / sum_p w_p,   w_p = exp(scale q . k_p - max),   p over the keys that row t sees:
//   the len cached tokens of its request, and of the request's own n new tokens those in the row's mask (bit j: token j)
//   or, without masks, those up to itself.  A row that sees nothing is 0.
#include "awq_request.cuh"

#include <cuda_fp16.h>
#include <math.h>

#include "awq_tcgen05.cuh"

namespace awq {

int encode_tensor_map_4d(CUtensorMap *map, int dtype, const void *base, const uint64_t (&dims)[4], const uint64_t (&strides_bytes)[3],
                         const uint32_t (&box)[4], int swizzle);

struct AttendArgs {
    const uint16_t *q;
    long long q_row, q_head;
    KvCacheView cache;
    const int32_t *table;
    long long table_stride;
    const int32_t *lens, *q_start;
    const long long *mask;
    uint16_t *out;
    long long o_row, o_head;
    float scale_log2;  // scale / ln 2: the exponentials are powers of two
    int R, T, n_heads, table_width;
    int page_shift;    // log2 of the page size, -1: not a power of two
    RequestHeader *header;
    uint8_t *scratch;
};

// The rows [q0, q1) and the number of cached tokens of request r, cut to what the buffers hold.
struct AttendRequest {
    int q0, n, len;
    bool bad;
};
__device__ __forceinline__ AttendRequest attend_request(const AttendArgs &a, int r) {
    AttendRequest q;
    const int s = a.q_start[r], e = a.q_start[r + 1], len = a.lens[r];
    q.q0 = min(max(s, 0), a.T);
    q.n = min(max(e, q.q0), a.T) - q.q0;
    const long long capacity = min((long long)a.table_width * a.cache.page_size, 0x7fff0000LL);  // (keys of a last tile still fit 32 bits)
    q.len = (int)min((long long)max(len, 0), max(capacity - q.n, 0LL));
    q.bad = q.q0 != s || q.q0 + q.n != e || q.len != len || (a.mask && q.n > REQ_MAX_TREE) || q.n > capacity;
    if (q.n > capacity) q.n = 0;
    return q;
}

__device__ __forceinline__ float exp2_fast(float x) {  // 2 units in the last place
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Weights that are multiplied as 16-bit values are 2^WEIGHT_LIFT times exp(score - maximum); their f32 sum is as many times too large, so that
// the factor goes with the division.  fp16 ends at 2^-24, and a long context's small weights count together: 32000 keys 16 nats behind one were
// off by 6 %, 17.5 nats behind were nothing.  Seven up, and with a maximum that may lie 8 behind, the largest is 2^15; what a weight may lose
// is 2^-32 of the largest.  bf16 has f32's exponents.
template <bool F16>
constexpr float WEIGHT_LIFT = F16 ? 7.f : 0.f;
__device__ __forceinline__ int page_index(const AttendArgs &a, int key) { return a.page_shift >= 0 ? key >> a.page_shift : key / a.cache.page_size; }

// Head sizes above 128: a CTA per row and head, a warp per 32 keys, four of them at a time; f32 throughout.  Rows of a group do not share
// their loads.  Bound by instructions (64 requests of 500 to 4000 tokens, 8/4 heads of 256: 752 us, 0.75 TB/s).
constexpr int AA_WARPS = 4;
template <bool F16>
__global__ void __launch_bounds__(AA_WARPS * 32) tree_attention_any_kernel(AttendArgs a) {
    constexpr int AHEAD = 4;
    __shared__ float2 accs[AA_WARPS][128];
    __shared__ float tops[AA_WARPS], totals[AA_WARPS];
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, t = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads;
    int lo = 0, hi = a.R;  // the request of row t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] <= t) lo = mid; else hi = mid;
    }
    const AttendRequest q = attend_request(a, lo);
    if (blockIdx.x == 0)
        for (int r = tid; r < a.R; r += AA_WARPS * 32)
            if (attend_request(a, r).bad) req_error(&a.header->error, REQ_ERR_REQUEST);
    const int j = t - q.q0;
    if (j < 0 || j >= q.n) return;  // behind the last request
    const int D = a.cache.head_dim, pairs = D >> 1, hk = h / (a.n_heads / a.cache.n_kv);
    const unsigned long long bits = a.mask ? (unsigned long long)a.mask[t] : 0;
    const uint32_t *qp = reinterpret_cast<const uint32_t *>(a.q + t * a.q_row + h * a.q_head);
    const uint32_t *kb = reinterpret_cast<const uint32_t *>(a.cache.k + hk * a.cache.k_head) + lane;
    const uint32_t *vb = reinterpret_cast<const uint32_t *>(a.cache.v + hk * a.cache.v_head) + lane;
    float2 qv[4], acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane + 32 * i;
        qv[i] = c < pairs ? unpack16x2<F16>(qp[c]) : make_float2(0.f, 0.f);
        acc[i] = make_float2(0.f, 0.f);
    }
    float top = -INFINITY, total = 0.f;
    for (int p0 = warp * 32; p0 < q.len + q.n; p0 += AA_WARPS * 32) {
        const int p = p0 + lane, d = p - q.len;
        long long k_at = -1, v_at = -1;  // of this lane's key, in pairs
        if (p < q.len + q.n && (d < 0 || (a.mask ? d < 64 && (bits >> d & 1) : d <= j))) {
            const int block = page_index(a, p), page = a.table[lo * a.table_stride + block], off = p - block * a.cache.page_size;
            if ((unsigned)page < (unsigned)a.cache.n_pages)
                k_at = (page * a.cache.k_page + off * a.cache.k_slot) >> 1, v_at = (page * a.cache.v_page + off * a.cache.v_slot) >> 1;
            else
                req_error(&a.header->error, REQ_ERR_PAGE);
        }
        const uint32_t seen = __ballot_sync(0xffffffffu, k_at >= 0);
        for (int i0 = 0; i0 < 32; i0 += AHEAD) {
            if (!(seen >> i0 & ((1u << AHEAD) - 1))) continue;
            uint32_t kw[AHEAD][4], vw[AHEAD][4];
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) {
                const long long ko = __shfl_sync(0xffffffffu, k_at, i0 + n), vo = __shfl_sync(0xffffffffu, v_at, i0 + n);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool there = ko >= 0 && lane + 32 * i < pairs;
                    kw[n][i] = there ? __ldg(kb + ko + 32 * i) : 0;
                    vw[n][i] = there ? __ldg(vb + vo + 32 * i) : 0;
                }
            }
            float s[AHEAD], m = top;
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) {
                s[n] = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 k = unpack16x2<F16>(kw[n][i]);
                    s[n] = fmaf(qv[i].x, k.x, fmaf(qv[i].y, k.y, s[n]));
                }
#pragma unroll
                for (int x = 16; x; x >>= 1) s[n] += __shfl_xor_sync(0xffffffffu, s[n], x);
                s[n] = seen >> (i0 + n) & 1 ? s[n] * a.scale_log2 : -INFINITY;
                m = fmaxf(m, s[n]);
            }
            const float ref = m == -INFINITY ? 0.f : m, keep = exp2f(top - ref);
            top = m;
            total *= keep;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = make_float2(acc[i].x * keep, acc[i].y * keep);
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) {
                const float w = exp2f(s[n] - ref);
                total += w;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 v = unpack16x2<F16>(vw[n][i]);
                    acc[i] = make_float2(fmaf(w, v.x, acc[i].x), fmaf(w, v.y, acc[i].y));
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) accs[warp][lane + 32 * i] = acc[i];
    if (lane == 0) tops[warp] = top, totals[warp] = total;
    __syncthreads();
    float m = -INFINITY, sum = 0.f;
    float2 o = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < AA_WARPS; ++w) m = fmaxf(m, tops[w]);
#pragma unroll
    for (int w = 0; w < AA_WARPS; ++w) {
        if (tops[w] == -INFINITY) continue;  // saw nothing
        const float f = exp2f(tops[w] - m);
        sum = fmaf(f, totals[w], sum);
        o = make_float2(fmaf(f, accs[w][tid].x, o.x), fmaf(f, accs[w][tid].y, o.y));
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (tid < pairs) reinterpret_cast<uint32_t *>(a.out + t * a.o_row + h * a.o_head)[tid] = pack16x2<F16>(o.x * inv, o.y * inv);
}

// =====================================================================================
// Few rows per cache head (one token, small trees): bound by the cache's bytes.
//
// A unit of work is a tile of keys of a segment = (request, cache head, 16 rows); rows are (token, head of the group) pairs,
// padded to the 16 rows of one mma.sync.  The CTAs split the units of all segments evenly (stream-K), whatever the lengths;
// a segment that several CTAs share is joined by the last of them to finish, in the order of its keys, so no CTA waits and
// results do not depend on timing.
//
// Inside a tile every warp has 16 keys of its own and keeps its own running maximum and sum.  K and V come in by asynchronous
// copies into shared memory of the warp's own, two blocks ahead, so that 12 warps an SM have up to 190 KB on their way.  Eight
// lanes fetch 128 bytes of a key at once: with requests of half a line, which a lane's own pieces would be, 64 long requests took 343 us, not
// 269.  In shared memory the pieces lie where mma.sync's lanes find them without bank conflicts:
//   scores: the order of the products over the head is free, so 16 bytes of a key are a lane's operands of two k-steps if the
//           rows of Q are taken in the same order; odd keys have the halves of their lines swapped;
//   output: a lane has 16 bytes of four keys (its k-indices) and pairs them up with byte permutes; column n of block j is then
//           head element 8 n + j, so that a lane's results are 16 neighbours; pieces are shifted by pairs of keys.
// Weights are multiplied as two 16-bit pieces, p = hi + lo: the tensor cores have time to spare, and the result keeps 16 (bf16) or 22 bits
// of a weight; in fp16 those below 2^-21 of the largest keep what lies above 2^-32 of it (WEIGHT_LIFT).
//
// Measured, bf16, heads of 128: one token of 64 requests of 1000 to 16000, 64/8 heads, 262 to 278 us, 5.5 to 5.9 TB/s (85 to 90 % of a copy's
// rate; keys straight to registers 389); one token of 256 requests of 500 to 2000, 32/8 heads, 226 us, 5.9 TB/s.  Small steps are a chain of
// latencies: starts and lengths, pages, keys, the join (one token behind 777, 32/8 heads of 64: 9.8 us).
// =====================================================================================
constexpr int AR_WARPS = 4, AR_TILE = AR_WARPS * 16, AR_PER_SM = 3, AR_ROWS = 16;
constexpr int AR_MAX_CTAS = 192 * AR_PER_SM;

template <int TO, int FROM>  // at fixed distances (bytes) from dst and src; zeros where bytes is 0, not 16
__device__ __forceinline__ void copy16(uint32_t dst, const uint16_t *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0 + %3], [%1 + %4], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes), "n"(TO), "n"(FROM) : "memory");
}
// N copies, the i-th at AT + i TO and i FROM.
template <int N, int TO, int FROM, int AT = 0, int I = 0>
__device__ __forceinline__ void copies16(uint32_t dst, const uint16_t *src, int bytes) {
    if constexpr (I < N) {
        copy16<AT + I * TO, I * FROM>(dst, src, bytes);
        copies16<N, TO, FROM, AT, I + 1>(dst, src, bytes);
    }
}
template <bool F16>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        mma_bf16_16816(d, a0, a1, a2, a3, b0, b1);
}
template <bool F16>
__device__ __forceinline__ bool not_finite16x2(uint32_t v) {
    constexpr uint32_t e = F16 ? 0x7c00u : 0x7f80u;
    return (v & e) == e || ((v >> 16) & e) == e;
}

// acc + 0 v for two 16-bit values: not a number once v was infinite or none.
template <bool F16>
__device__ __forceinline__ uint32_t at_zero_fma(uint32_t v, uint32_t acc) {
    if (F16) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v), "r"(0u));
    else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v), "r"(0u));
    return acc;
}
// Of the block's threads before this one, and of all.
template <int THREADS>
__device__ __forceinline__ long long exclusive_sum(long long mine, long long &total) {
    __shared__ long long sums[THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += u;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    long long base = incl - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) base += sums[w];
        total += sums[w];
    }
    return base;
}
// Units of all requests before each one, in shared memory; returns their number.  Requests that do not fit are reported by
// CTA 0 and have what attend_request leaves of them.
template <int THREADS, typename F>
__device__ __forceinline__ long long scan_units(const AttendArgs &a, long long *cum, F units_of) {
    const int tid = threadIdx.x, per = (a.R + THREADS - 1) / THREADS, r0 = min(tid * per, a.R), r1 = min(r0 + per, a.R);
    long long mine = 0;
    for (int r = r0; r < r1; ++r) {
        const AttendRequest q = attend_request(a, r);
        if (q.bad && blockIdx.x == 0) req_error(&a.header->error, REQ_ERR_REQUEST);
        const long long units = q.n ? units_of(q, r) : 0;
        cum[r] = units;
        mine += units;
    }
    long long total, base = exclusive_sum<THREADS>(mine, total);
    for (int r = r0; r < r1; ++r) {
        const long long u = cum[r];
        cum[r] = base;
        base += u;
    }
    if (tid == 0) cum[a.R] = total;
    __syncthreads();
    return total;
}
// (64-bit divisions cost some hundred cycles; units rarely need them)
__device__ __forceinline__ long long at_div(long long x, long long y) { return (x | y) >> 32 ? x / y : (long long)((uint32_t)x / (uint32_t)y); }
__device__ __forceinline__ int request_of_unit(const long long *cum, int n, long long x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cum[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

// Shared memory: Q in operand order | places of the keys | K and V, later the warps' results | units.  The same for any number of
// requests (three CTAs fit an SM): a thread adds up the units of several, and who has some of them looks through these requests again.
constexpr int AR_PLACES = 4 * 16 * 16 + 64;  // of a warp: four blocks of 16 keys, and which of them there are (stages start on 128 bytes)
template <int D>
constexpr int AR_STAGE = 16 * D * 4;  // K and V of a warp's block
template <int D>
constexpr int AR_STAGES = AR_WARPS * (2 * AR_STAGE<D> > AR_ROWS * (D + 2) * 4 ? 2 * AR_STAGE<D> : AR_ROWS * (D + 2) * 4);
constexpr int AR_CUM = (AR_WARPS * 32 + 1) * 8;  // units before each thread's requests
template <int D>
constexpr int AR_SMEM = D * 32 + AR_WARPS * AR_PLACES + AR_STAGES<D> + AR_CUM;
static_assert(AR_SMEM<128> + 64 <= 224 * 1024 / AR_PER_SM - 1024, "three CTAs an SM (76096 bytes a CTA measured two)");

// PADDED: heads of other sizes below D; what lies behind them is 0 in shared memory and neither read nor written (64 requests of 500 to
// 4000 tokens, 32/8 heads of 96: 100 us, a warp per row and head took 4968).
template <bool F16, int D, bool PADDED>
__global__ void __launch_bounds__(AR_WARPS * 32, AR_PER_SM) tree_attention_rows_kernel(AttendArgs a) {
    const int head = PADDED ? a.cache.head_dim : D;
    constexpr int THREADS = AR_WARPS * 32, QC = D / 32, VC = D / 64;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    uint4 *qs = reinterpret_cast<uint4 *>(smem);  // [QC][2][32]
    longlong2 *places = reinterpret_cast<longlong2 *>(smem + D * 32 + warp * AR_PLACES);
    uint32_t *there = reinterpret_cast<uint32_t *>(places + 64);
    uint8_t *stages = smem + D * 32 + AR_WARPS * AR_PLACES;
    uint8_t *mine = stages + warp * 2 * AR_STAGE<D>;  // [2][K [16][D], V [16][D]]
    // copies: lane l brings pieces l % 8 (and l % 8 + 8) of keys l / 8 + 4 i
    const int ck = lane >> 3, cp = lane & 7;
    const uint32_t copy_k = smem_u32(mine) + ck * 2 * D + (cp ^ ((ck & 1) << 2)) * 16;
    const uint32_t copy_v = smem_u32(mine) + 32 * D + ck * 2 * D;  // + the piece, in its place for even and odd i
    const uint32_t piece_v[2] = {(uint32_t)(cp ^ (ck & 2)) * 16, (uint32_t)(cp ^ (ck & 2) ^ 4) * 16};
    float *ow = reinterpret_cast<float *>(stages);                           // [WARPS][16][D]
    float *mw = ow + AR_WARPS * AR_ROWS * D, *lw = mw + AR_WARPS * AR_ROWS;   // [WARPS][16]
    long long *cum = reinterpret_cast<long long *>(smem + AR_SMEM<D> - AR_CUM);
    __shared__ int s_last;
    pdl_wait();
    pdl_launch_dependents();
    const int group = a.n_heads / a.cache.n_kv;
    long long pad = 1;  // a segment takes a multiple of this
    auto segments_of = [&](const AttendRequest &q) { return (((long long)q.n * group + AR_ROWS - 1) / AR_ROWS) * a.cache.n_kv; };
    auto units_of = [&](const AttendRequest &q, long long pad) {
        const int tiles = (q.len + q.n + AR_TILE - 1) / AR_TILE;
        return segments_of(q) * (pad > 1 ? at_div(tiles + pad - 1, pad) * pad : tiles);
    };
    const int of_thread = (a.R + THREADS - 1) / THREADS;  // requests
    AttendRequest own{};
    auto sum_over_requests = [&](auto f) {
        long long sum = 0, total;
        for (int r = tid * of_thread; r < min((tid + 1) * of_thread, a.R); ++r) {
            if (of_thread > 1) own = attend_request(a, r);
            sum += f(own);
        }
        __syncthreads();  // (the last sums have been read)
        cum[tid] = exclusive_sum<THREADS>(sum, total);
        if (tid == 0) cum[THREADS] = total;
        __syncthreads();
        return total;
    };
    if (of_thread == 1 && tid < a.R) own = attend_request(a, tid);
    if (blockIdx.x == 0)
        for (int r = tid; r < a.R; r += THREADS)
            if (attend_request(a, r).bad) req_error(&a.header->error, REQ_ERR_REQUEST);
    long long units = sum_over_requests([&](const AttendRequest &q) { return units_of(q, 1); });
    long long per = max(at_div(units + gridDim.x - 1, gridDim.x), 1LL);
    // A CTA that goes on with another segment pays for a chain of loads again (starts, pages, keys), about as long as four tiles take.
    // Where CTAs have few tiles anyway, every segment begins at one of its own, if that makes none of them much longer: one token of 16
    // requests of 100 to 2000, 32/8 heads of 128, 23.4 -> 18.7 us.
    if (per > 1 && per <= 16) {
        const long long segments = sum_over_requests(segments_of);
        for (long long p = per; segments <= gridDim.x && pad == 1 && p <= per + at_div(4 * segments, gridDim.x); ++p)
            if (sum_over_requests([&](const AttendRequest &q) { return units_of(q, p); }) <= p * gridDim.x) pad = p;
        if (pad > 1)
            per = pad, units = cum[THREADS];
        else
            units = sum_over_requests([&](const AttendRequest &q) { return units_of(q, 1); });
    }
    long long x = blockIdx.x * per;
    const long long end = min(x + per, units);
    const int page_size = a.cache.page_size;
    float *parts = reinterpret_cast<float *>(a.scratch + 4 * AR_MAX_CTAS);
    int *counters = reinterpret_cast<int *>(a.scratch);
    constexpr int PART = AR_ROWS * (D + 2);

    while (x < end) {
        int r = request_of_unit(cum, THREADS, x);  // the thread whose requests these are
        long long rem = x - cum[r];
        AttendRequest rq;
        if (of_thread == 1) {
            rq = attend_request(a, r);
        } else {
            for (int r0 = r * of_thread;; r0 += 32) {  // (units of one of them lie behind x)
                const AttendRequest q = r0 + lane < a.R ? attend_request(a, r0 + lane) : AttendRequest{};
                const long long u = units_of(q, pad);
                long long incl = u;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const long long v = __shfl_up_sync(0xffffffffu, incl, d);
                    if (lane >= d) incl += v;
                }
                const uint32_t behind = __ballot_sync(0xffffffffu, incl > rem);
                const int l = behind ? __ffs(behind) - 1 : 31;
                r = r0 + l;
                rem -= __shfl_sync(0xffffffffu, behind ? incl - u : incl, l);
                rq = {__shfl_sync(0xffffffffu, q.q0, l), __shfl_sync(0xffffffffu, q.n, l), __shfl_sync(0xffffffffu, q.len, l), false};
                if (behind || r0 + 32 >= a.R) break;
            }
        }
        const int total = rq.len + rq.n, n_tiles = (total + AR_TILE - 1) / AR_TILE, m_tiles = (rq.n * group + AR_ROWS - 1) / AR_ROWS;
        const long long n_units = pad > 1 ? at_div(n_tiles + pad - 1, pad) * pad : n_tiles;
        const int seg = (int)at_div(rem, n_units), tile0 = (int)(rem - seg * n_units), hk = seg / m_tiles, row0 = (seg % m_tiles) * AR_ROWS;
        const long long seg_start = x - tile0, seg_end = seg_start + n_tiles;
        const int tiles = (int)(min(end, seg_end) - x);
        x = min(end, seg_start + n_units);
        if (tiles <= 0) continue;
        const int32_t *table = a.table + r * a.table_stride;
        const uint16_t *kbase = a.cache.k + hk * a.cache.k_head + 8 * cp, *vbase = a.cache.v + hk * a.cache.v_head + 8 * cp;

        // a lane looks after one key of two blocks: its page, then its place in K and V (negative: none)
        const int first = tile0 * AR_TILE + warp * 16;
        auto page_of = [&](int i) {
            const int key = first + (i + (lane >> 4)) * AR_TILE + (lane & 15);
            return i + (lane >> 4) < tiles && key < total ? __ldg(table + page_index(a, key)) : -2;
        };
        auto place = [&](int i, int page) {  // i even
            const int key = first + (i + (lane >> 4)) * AR_TILE + (lane & 15), off = key - page_index(a, key) * page_size;
            const bool ok = (unsigned)page < (unsigned)a.cache.n_pages;
            if (!ok && page != -2) req_error(&a.header->error, REQ_ERR_PAGE);
            if (page == -2 && i + (lane >> 4) < tiles && key < total) req_error(&a.header->error, REQ_ERR_PAGE);
            places[(i & 2) * 16 + lane] =
                ok ? make_longlong2(page * a.cache.k_page + off * a.cache.k_slot, page * a.cache.v_page + off * a.cache.v_slot) : make_longlong2(-8, -8);
            const uint32_t b = __ballot_sync(0xffffffffu, ok);
            if (lane == 0) there[(i & 2) >> 1] = b;
            __syncwarp();
        };
        auto copy_lines = [&](uint32_t dst, const uint16_t *src, bool there) {
            if (!PADDED) {
                copies16<D / 64, 128, 128>(dst, src, there ? 16 : 0);
            } else {
                copy16<0, 0>(dst, src, there && 8 * cp < head ? 16 : 0);
                if (D > 64) copy16<128, 128>(dst, src, there && 64 + 8 * cp < head ? 16 : 0);
            }
        };
        auto load_k = [&](int i) {
            __syncwarp();  // the block that was here has been read
            if (i < tiles)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const long long o = places[(i & 3) * 16 + 4 * q + ck].x;
                    copy_lines(copy_k + (i & 1) * AR_STAGE<D> + q * 8 * D, kbase + o, o >= 0);
                }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        auto load_v = [&](int i) {
            __syncwarp();
            if (i < tiles)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const long long o = places[(i & 3) * 16 + 4 * q + ck].y;
                    copy_lines(copy_v + piece_v[q & 1] + (i & 1) * AR_STAGE<D> + q * 8 * D, vbase + o, o >= 0);
                }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        __syncthreads();  // the previous segment's readers of shared memory are done
        const int page0 = page_of(0);
        int next_page = page_of(2);
        // this lane's rows, g and g + 8: token and mask
        int j[2];
        unsigned long long bits[2];
        const uint16_t *qrow[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = row0 + g + 8 * i;
            j[i] = row < rq.n * group ? row / group : -1;
            bits[i] = a.mask && j[i] >= 0 ? (unsigned long long)a.mask[rq.q0 + j[i]] : 0;
            qrow[i] = a.q + (long long)(rq.q0 + max(j[i], 0)) * a.q_row + (long long)(hk * group + row % group) * a.q_head;
        }
        for (int c = warp; c < QC; c += AR_WARPS)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                qs[(c * 2 + i) * 32 + lane] = j[i] >= 0 && (!PADDED || 32 * c + 8 * t4 < head) ? *reinterpret_cast<const uint4 *>(qrow[i] + 32 * c + 8 * t4) : make_uint4(0, 0, 0, 0);
        place(0, page0);
        load_k(0);
        load_v(0);
        load_k(1);
        load_v(1);
        __syncthreads();

        float acc[VC][8][4];
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int b = 0; b < 8; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[c][b][e] = 0.f;
        float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
        for (int i = 0; i < tiles; ++i) {
            if ((i & 1) == 0) {
                place(i + 2, next_page);
                next_page = page_of(i + 4);
            }
            const uint8_t *stage = mine + (i & 1) * AR_STAGE<D>;
            const uint8_t *ks = stage + g * 2 * D + t4 * 16, *vs = stage + 32 * D + 4 * D * t4 + (g ^ (2 * t4)) * 16;
            const int swap = (g & 1) * 64;
            asm volatile("cp.async.wait_group 3;" ::: "memory");
            __syncwarp();
            float s[2][4] = {};
#pragma unroll
            for (int c = 0; c < QC; ++c) {
                const uint4 q0 = qs[(c * 2) * 32 + lane], q1 = qs[(c * 2 + 1) * 32 + lane];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint4 k = *reinterpret_cast<const uint4 *>(ks + 16 * D * b + (64 * c ^ swap));
                    mma16<F16>(s[b], q0.x, q1.x, q0.y, q1.y, k.x, k.y);
                    mma16<F16>(s[b], q0.z, q1.z, q0.w, q1.w, k.z, k.w);
                }
            }
            load_k(i + 2);
            const int key0 = first + i * AR_TILE;
            const uint32_t valid = there[(i & 2) >> 1] >> (16 * (i & 1)) & 0xffffu;
            const bool partly = key0 + 16 > rq.len || valid != 0xffffu;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[b][e] *= a.scale_log2;
            if (partly) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int c = 8 * b + 2 * t4 + (e & 1), d = key0 + c - rq.len;
                        const bool seen = (valid >> c & 1) && (d < 0 || (a.mask ? d < 64 && (bits[e >> 1] >> d & 1) : d <= j[e >> 1]));
                        if (!seen) s[b][e] = -INFINITY;
                    }
            }
            // The weights refer to a maximum that may lie 8 behind: they stay below 2^8 (and the lift), and the sums are rarely rescaled.
            float p[2][4];
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
                float m = fmaxf(fmaxf(s[0][2 * i2], s[0][2 * i2 + 1]), fmaxf(s[1][2 * i2], s[1][2 * i2 + 1]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                if (__any_sync(0xffffffffu, m > top[i2] + 8.f)) {
                    const float to = fmaxf(m, top[i2]), keep = to == -INFINITY ? 1.f : exp2_fast(top[i2] - to);
                    top[i2] = to;
                    sum[i2] *= keep;
#pragma unroll
                    for (int c = 0; c < VC; ++c)
#pragma unroll
                        for (int b = 0; b < 8; ++b) acc[c][b][2 * i2] *= keep, acc[c][b][2 * i2 + 1] *= keep;
                }
                const float ref = (top[i2] == -INFINITY ? 0.f : top[i2]) - WEIGHT_LIFT<F16>;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) sum[i2] += p[b][2 * i2 + e] = exp2_fast(s[b][2 * i2 + e] - ref);
            }
            uint32_t hi[4], lo[4];  // rows g, g + 8 of keys 0-7, then of keys 8-15
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i2 = 0; i2 < 2; ++i2) {
                    const float p0 = p[b][2 * i2], p1 = p[b][2 * i2 + 1];
                    hi[2 * b + i2] = pack16x2<F16>(p0, p1);
                    const float2 h = unpack16x2<F16>(hi[2 * b + i2]);
                    lo[2 * b + i2] = pack16x2<F16>(p0 - h.x, p1 - h.y);
                }
            asm volatile("cp.async.wait_group 3;" ::: "memory");
            __syncwarp();
            bool odd = false;
            if (partly) {  // a value that some rows do not see must not reach them as 0 times infinity or NaN
                uint32_t zeros[4] = {};
#pragma unroll
                for (int w = 0; w < 4 * VC; ++w) {  // (the pieces this lane reads below)
                    const uint4 u = *reinterpret_cast<const uint4 *>(vs + (w & 1) * 2 * D + (w >> 1 & 1) * 16 * D + (w >> 2) * 128);
                    zeros[0] = at_zero_fma<F16>(u.x, zeros[0]), zeros[1] = at_zero_fma<F16>(u.y, zeros[1]);
                    zeros[2] = at_zero_fma<F16>(u.z, zeros[2]), zeros[3] = at_zero_fma<F16>(u.w, zeros[3]);
                }
                const bool any = not_finite16x2<F16>(zeros[0]) || not_finite16x2<F16>(zeros[1]) || not_finite16x2<F16>(zeros[2]) || not_finite16x2<F16>(zeros[3]);
#pragma unroll 1
                for (int w = 0; any && w < 16 * VC; ++w) {
                    uint32_t &u = reinterpret_cast<uint32_t *>(const_cast<uint8_t *>(vs) + (w >> 2 & 1) * 2 * D + (w >> 3 & 1) * 16 * D + (w >> 4) * 128)[w & 3];
                    if (!not_finite16x2<F16>(u)) continue;
                    odd = true;
                    u &= (not_finite16x2<F16>(u & 0xffffu) ? 0xffff0000u : 0xffffffffu) & (not_finite16x2<F16>(u >> 16) ? 0xffffu : 0xffffffffu);
                }
            }
#pragma unroll
            for (int c = 0; c < VC; ++c) {
                uint32_t v[4][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(vs + (e & 1) * 2 * D + (e >> 1) * 16 * D + c * 128);
                    v[e][0] = u.x, v[e][1] = u.y, v[e][2] = u.z, v[e][3] = u.w;
                }
#pragma unroll
                for (int b = 0; b < 8; ++b) {
                    const uint32_t sel = b & 1 ? 0x7632u : 0x5410u;
                    const uint32_t b0 = __byte_perm(v[0][b >> 1], v[1][b >> 1], sel), b1 = __byte_perm(v[2][b >> 1], v[3][b >> 1], sel);
                    mma16<F16>(acc[c][b], hi[0], hi[1], hi[2], hi[3], b0, b1);
                    mma16<F16>(acc[c][b], lo[0], lo[1], lo[2], lo[3], b0, b1);
                }
            }
            if (partly && __any_sync(0xffffffffu, odd)) {  // the rows that do see it, key by key
                for (int key = 0; key < 16; ++key) {
                    const long long o = places[(i & 3) * 16 + key].y;
                    const int from = (lane & 28) + ((key & 7) >> 1);
                    float w[2];  // the weights of rows g and g + 8
#pragma unroll
                    for (int i2 = 0; i2 < 2; ++i2) {
                        const float w0 = __shfl_sync(0xffffffffu, p[0][2 * i2], from), w1 = __shfl_sync(0xffffffffu, p[0][2 * i2 + 1], from);
                        const float w2 = __shfl_sync(0xffffffffu, p[1][2 * i2], from), w3 = __shfl_sync(0xffffffffu, p[1][2 * i2 + 1], from);
                        w[i2] = key < 8 ? (key & 1 ? w1 : w0) : (key & 1 ? w3 : w2);
                    }
                    if (o < 0) continue;  // (zeros)
                    const int d0 = key0 + key - rq.len;
#pragma unroll
                    for (int i2 = 0; i2 < 2; ++i2) {  // a weight that came out as 0 leaves infinity infinity; one that is not seen is none
                        const bool seen = j[i2] >= 0 && (d0 < 0 || (a.mask ? d0 < 64 && (bits[i2] >> d0 & 1) : d0 <= j[i2]));
                        w[i2] = !seen ? 0.f : w[i2] == 0.f ? 1.f : w[i2];
                    }
#pragma unroll
                    for (int c = 0; c < VC; ++c) {
                        if (PADDED && 64 * c + 16 * t4 >= head) continue;
#pragma unroll
                        for (int d = 0; d < 16; ++d) {
                            const uint32_t bitsv = (vbase - 8 * cp + o)[64 * c + 16 * t4 + d];
                            if (!not_finite16x2<F16>(bitsv)) continue;
                            const float v = unpack16x2<F16>(bitsv).x;
#pragma unroll
                            for (int i2 = 0; i2 < 2; ++i2)
                                if (w[i2] != 0.f) acc[c][d & 7][2 * i2 + (d >> 3)] += w[i2] * v;
                        }
                    }
                }
            }
            load_v(i + 2);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // the warps' results take the stages' place
        // ---- join the warps ----
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
            sum[i2] += __shfl_xor_sync(0xffffffffu, sum[i2], 1);
            sum[i2] += __shfl_xor_sync(0xffffffffu, sum[i2], 2);
            const int row = g + 8 * i2;
            if (t4 == 0) mw[warp * 16 + row] = top[i2], lw[warp * 16 + row] = sum[i2];
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float *o = ow + (warp * 16 + row) * D + 64 * c + 16 * t4 + 8 * e;
                    *reinterpret_cast<float4 *>(o) = make_float4(acc[c][0][2 * i2 + e], acc[c][1][2 * i2 + e], acc[c][2][2 * i2 + e], acc[c][3][2 * i2 + e]);
                    *reinterpret_cast<float4 *>(o + 4) = make_float4(acc[c][4][2 * i2 + e], acc[c][5][2 * i2 + e], acc[c][6][2 * i2 + e], acc[c][7][2 * i2 + e]);
                }
        }
        __syncthreads();
        const int c0 = (int)at_div(seg_start, per), c1 = (int)at_div(seg_end - 1, per), rows = min(AR_ROWS, rq.n * group - row0);
        const bool whole = c0 == c1;
        float *part = parts + (long long)(2 * blockIdx.x + ((int)blockIdx.x == c0 ? 1 : 0)) * PART;
        auto store = [&](int row, int d, const float (&o)[4], float total_w) {
            if (PADDED && d >= head) return;
            const float inv = total_w == 0.f ? 0.f : 1.f / total_w;
            uint16_t *dst = a.out + (long long)(rq.q0 + (row0 + row) / group) * a.o_row + (long long)(hk * group + (row0 + row) % group) * a.o_head + d;
            *reinterpret_cast<uint2 *>(dst) = make_uint2(pack16x2<F16>(o[0] * inv, o[1] * inv), pack16x2<F16>(o[2] * inv, o[3] * inv));
        };
        for (int i = tid; i < rows * (D / 4); i += THREADS) {
            const int row = i / (D / 4), d = 4 * (i % (D / 4));
            float m = -INFINITY, l = 0.f, o[4] = {};
#pragma unroll
            for (int w = 0; w < AR_WARPS; ++w) m = fmaxf(m, mw[w * 16 + row]);
#pragma unroll
            for (int w = 0; w < AR_WARPS; ++w) {
                const float mm = mw[w * 16 + row], f = mm == -INFINITY ? 0.f : exp2_fast(mm - m);
                l += f * lw[w * 16 + row];
                if (mm == -INFINITY) continue;  // saw nothing.  (A warp whose weights come out as 0 goes on: 0 times NaN is NaN)
                const float4 u = *reinterpret_cast<const float4 *>(ow + (w * 16 + row) * D + d);
                o[0] += f * u.x, o[1] += f * u.y, o[2] += f * u.z, o[3] += f * u.w;
            }
            if (whole) {
                store(row, d, o, l);
            } else {
                *reinterpret_cast<float4 *>(part + row * D + d) = make_float4(o[0], o[1], o[2], o[3]);
                if (d == 0) part[AR_ROWS * D + row] = m, part[AR_ROWS * D + AR_ROWS + row] = l;
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = atomicAdd(counters + c0, 1) == c1 - c0;
            __syncthreads();
            if (s_last) {
                __threadfence();
                for (int i = tid; i < rows * (D / 4); i += THREADS) {
                    const int row = i / (D / 4), d = 4 * (i % (D / 4));
                    float m = -INFINITY, l = 0.f, o[4] = {};
                    for (int at = c0; at <= c1; at += 8) {  // eight parts' loads at once
                        float mc[8], lc[8];
                        float4 u[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const int c = min(at + k, c1);
                            const float *src = parts + (long long)(2 * c + (c == c0 ? 1 : 0)) * PART;
                            mc[k] = __ldcg(src + AR_ROWS * D + row), lc[k] = __ldcg(src + AR_ROWS * D + AR_ROWS + row);
                            u[k] = __ldcg(reinterpret_cast<const float4 *>(src + row * D + d));
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (at + k <= c1) {
                                const float m2 = fmaxf(m, mc[k]), ref = m2 == -INFINITY ? 0.f : m2, f = exp2_fast(m - ref), fc = exp2_fast(mc[k] - ref);
                                m = m2;
                                l = l * f + lc[k] * fc;
                                const float add[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[e] = o[e] * f + (mc[k] == -INFINITY ? 0.f : add[e] * fc);
                            }
                    }
                    store(row, d, o, l);
                }
                if (tid == 0) counters[c0] = 0;
            }
        }
    }
}

// =====================================================================================
// Many rows per cache head (trees, prompts): tcgen05, 128 rows at a time.
//
// A unit of work is 64 keys of a segment = (request, cache head, 128 rows), split over the CTAs as above.  Two CTAs an SM;
// in each
//   2 warps  bring K and V by TMA, box by box of slots that lie in one page, two tiles of each held (pages that do not consist of
//            eights of slots: by 16-byte asynchronous copies into the same 128-byte swizzle);
//   1 warp   brings Q of the next segment while the last tiles of this one are weighed;
//   1 warp   issues the products: S = Q K^T into 64 columns of tensor memory, O += P V into D others;
//   4 warps  hold a row per thread: maximum, weights, and P as 16-bit pairs over S's own columns, from where the tensor cores take
//            it as the left operand of the next product.
// S is held twice: the scores of a tile are formed while the one before it is weighed.  What one CTA leaves idle (the tensor
// cores during its softmax, the exponentials during its products) is the other one's.  O stays in tensor memory; it is rescaled
// only when a maximum has grown by more than 8 (powers of two), by the warp that finds it.
// Weights are rounded to the rows' 16-bit type for the product, as they have to be for one tensor-core operand (their sum is
// not): half a step per weight, independent from key to key; in fp16 for weights from 2^-21 of the largest on, smaller ones to 2^-32 of
// it (WEIGHT_LIFT).
//
// Measured, bf16, heads of 128: two trees of 64 over 32000 tokens, 64/8 heads, 166 us (810 TFLOP/s) in ten replayed calls, 188 to 193 (700) in
// calls one after another for some time, when the SMs run slower; 16 trees of 8 to 32 over 300 to 6000 tokens, 32/8 heads, 59 to 62 us; four prompts of
// 512 behind 2000 to 4000 tokens, 32/8 heads, 151 us, 690 TFLOP/s.  Bound by how fast one CTA's chain S -> weights -> O turns over: a tile of 64 keys
// takes some 2300 cycles, while the tensor pipe is active for 37 % of them, instructions issue in 41 %, and DRAM is at 18 %.
// =====================================================================================
constexpr int AT_ROWS = 128, AT_TILE = 64, AT_THREADS = 8 * 32, AT_PER_SM = 2, AT_MAX_CTAS = 192 * AT_PER_SM, AT_COLS = 256;
// A segment that begins in a CTA and goes on behind it: where it ends, and its rows.  The next launch joins its parts.
struct AttendJoin {
    int last, q0, n, hk, m;
};
constexpr long long AT_STEP_BYTES = 100LL << 20;  // of keys and values, from which on segments begin at CTAs of their own
constexpr int AT_JOINS = 4 * AR_MAX_CTAS;  // their place in the scratch, behind the other kernel's counters
// A piece of a segment that one CTA works on: keys from tile0 on, `tiles` of its n_tiles.
struct AttendSegment {
    int r, q0, n, len, hk, m, tile0, tiles, n_tiles, c0, c1;  // c0, c1: the CTAs that have its first and last tile
};
struct AttendTilesShared {
    // mbarriers, of even and odd tiles: K, V there; QK^T, PV (of every fourth) done; P there.  Of a segment: Q there, Q done with, O done.  V that is
    // not ready for the product yet.
    uint64_t k_full[2], v_full[2], scored[2], added[4], weighed[2], q_full, q_free, summed, v_landed, drained;
    uint32_t tmem;
    int odd[4], pad;                       // a segment's: values that are not finite were taken out of V
    uint64_t found[4];                     // mbarriers: a segment's description is there
    AttendSegment segments[4];             // (no tiles: the last one is over)
    unsigned long long bits[2][AT_ROWS];   // of a segment's rows: their tokens' masks
    uint32_t valid[4][2];                  // of a tile: which of its keys there are
    long long places[2][AT_TILE];  // of a copying warp: the keys of its tile
};
template <int D>
constexpr int AT_OPERAND = AT_TILE * D * 2;
template <int D>
constexpr int AT_SMEM = AT_ROWS * D * 2 + 4 * AT_OPERAND<D> + 1024 + (int)sizeof(AttendTilesShared);

// Keys that some of rows [128 m, 128 m + 128) see, from the front on.
__device__ __forceinline__ int at_tiles(const AttendArgs &a, const AttendRequest &q, int group, int m) {
    const int seen = a.mask ? q.n : (int)min((long long)q.n, at_div((long long)(m + 1) * AT_ROWS - 1, group) + 1);
    return (q.len + seen + AT_TILE - 1) / AT_TILE;
}
// 128-byte swizzle, columns of the operand side by side (MN-major): blocks of 64 columns `block` bytes apart, groups of eight k 1024.
__device__ __forceinline__ uint64_t at_desc_mn(uint32_t smem_addr, uint32_t block) {
    return (dg_desc_sw128(smem_addr) & ~((uint64_t)0x3fff << 16)) | (uint64_t)(block >> 4) << 16;
}
__device__ __forceinline__ void at_tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Two f32 fused multiply-adds, and two additions onto a pair of sums, in one instruction each.
__device__ __forceinline__ void at_fma2(float &x0, float &x1, float a0, float a1, float b, float c) {
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(x0), "=f"(x1)
        : "f"(a0), "f"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ void at_add2(uint64_t &sums, float x0, float x1) {
    asm("{\n\t.reg .b64 a;\n\tmov.b64 a, {%1, %2};\n\tadd.rn.f32x2 %0, %0, a;\n\t}" : "+l"(sums) : "f"(x0), "f"(x1));
}
__device__ __forceinline__ float at_sum2(uint64_t sums) {
    return __uint_as_float((uint32_t)sums) + __uint_as_float((uint32_t)(sums >> 32));
}
// Scores of a row against keys it does not see become -inf; vis: the keys that there are.
__device__ __noinline__ void at_see(const AttendArgs &a, int len, int key0, int j, unsigned long long bits, uint32_t (&vis)[2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int d0 = key0 + 32 * c - len;  // token of the step of the word's first key
        if (d0 <= -32) continue;
        unsigned long long b;  // from token max(d0, 0) on
        if (a.mask) b = d0 >= 64 ? 0 : d0 > 0 ? bits >> d0 : bits;
        else b = j - max(d0, 0) >= 63 ? ~0ull : j < max(d0, 0) ? 0 : (2ull << (j - max(d0, 0))) - 1;
        vis[c] &= d0 < 0 ? (uint32_t)(b << -d0) | ((1u << -d0) - 1) : (uint32_t)b;
    }
}
__device__ __forceinline__ void at_mask(const AttendArgs &a, int len, int key0, int j, unsigned long long bits, uint32_t (&vis)[2],
                                        uint32_t (&v)[2][32]) {
    at_see(a, len, key0, j, bits, vis);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 32; ++e) v[c][e] = vis[c] >> e & 1 ? v[c][e] : 0xff800000u;
}

// A CTA's walk over its part of the units, segment by segment.
template <int D>
struct AttendWalk {
    const AttendArgs &a;
    const long long *cum;
    long long x, end;
    int group;
    long long pad;  // units of a segment come in multiples of this
    __device__ __forceinline__ bool next(AttendSegment &s, long long per) {
        while (x < end) {
            s.r = request_of_unit(cum, a.R, x);
            const AttendRequest rq = attend_request(a, s.r);
            s.q0 = rq.q0, s.n = rq.n, s.len = rq.len;
            const long long rem = x - cum[s.r], per_head = at_div(cum[s.r + 1] - cum[s.r], a.cache.n_kv);
            s.hk = (int)at_div(rem, per_head);
            long long left = rem - s.hk * per_head, units;
            if (a.mask) {  // all segments of a request are as long
                s.n_tiles = at_tiles(a, rq, group, 0);
                units = at_padded(s.n_tiles, pad);
                s.m = (int)at_div(left, units);
                left -= s.m * units;
            } else {  // a prompt's grow: 32 at a time (a warp calls this)
                const int lane = threadIdx.x & 31;
                for (s.m = 0;; s.m += 32) {
                    const int mine = at_tiles(a, rq, group, s.m + lane);
                    const long long u = at_padded(mine, pad);
                    long long incl = u;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const long long v = __shfl_up_sync(0xffffffffu, incl, d);
                        if (lane >= d) incl += v;
                    }
                    const uint32_t behind = __ballot_sync(0xffffffffu, incl > left);
                    if (behind) {
                        const int at = __ffs(behind) - 1;
                        s.m += at;
                        s.n_tiles = __shfl_sync(0xffffffffu, mine, at);
                        units = __shfl_sync(0xffffffffu, u, at);
                        left -= __shfl_sync(0xffffffffu, incl, at) - units;
                        break;
                    }
                    left -= __shfl_sync(0xffffffffu, incl, 31);
                }
            }
            s.tile0 = (int)left;
            s.tiles = (int)min(end - x, (long long)s.n_tiles - left);
            s.c0 = (int)at_div(x - left, per);
            s.c1 = (int)at_div(x - left + s.n_tiles - 1, per);
            x += min(end - x, units - left);
            if (s.tiles > 0) return true;
        }
        return false;
    }
    __device__ __forceinline__ static long long at_padded(int tiles, long long pad) { return pad > 1 ? at_div(tiles + pad - 1, pad) * pad : tiles; }
};

// Keys 4 q + (the lane's of four) of a tile for q = Q .. END - 1, in lines of 128 bytes swizzled by key % 8: the lane's piece has one
// place in keys of even q (dst0) and another one in odd (dst1).
template <int D, int Q, int END>
__device__ __forceinline__ void at_copy_keys(uint32_t dst0, uint32_t dst1, const uint16_t *base, const long long *places) {
    if constexpr (Q < END) {
        const long long o = places[4 * Q];
        copies16<D / 64, AT_TILE * 128, 128, Q * 512>(Q & 1 ? dst1 : dst0, base + o, o < 0 ? 0 : 16);
        at_copy_keys<D, Q + 1, END>(dst0, dst1, base, places);
    }
}

template <bool F16, int D>
__device__ __noinline__ void at_clean_values(uint8_t *mine, int from, int row, int *odd) {
#pragma unroll 1
    for (int k = row; k < AT_TILE; k += 4)
#pragma unroll 1
        for (int w = 0; k >= from && w < 4 * (D / 64); ++w) {
            uint32_t &v = reinterpret_cast<uint32_t *>(mine + (w >> 2) * AT_TILE * 128 + (k - row) * 128)[w & 3];
            if (!not_finite16x2<F16>(v)) continue;
            *odd = 1;
            v &= (not_finite16x2<F16>(v & 0xffffu) ? 0xffff0000u : 0xffffffffu) & (not_finite16x2<F16>(v >> 16) ? 0xffffu : 0xffffffffu);
        }
}
// A weight of 0 must not meet infinity or NaN: in V's tile the slots without a token become 0, and of the keys from `from` on, which
// some rows do not see, what is not finite; that is added where it is seen, at the segment's end.  A warp: eight lanes a line.
// (The warp is alone with this, and the product waits for it: a look at every value costs one fused multiply-add for two.)
template <bool F16, int D>
__device__ __forceinline__ void at_clean(uint8_t *tile, const uint32_t (&valid)[2], int from, int lane, int *odd) {
    const int row = lane >> 3;
    uint8_t *mine = tile + row * 128 + (lane & 7) * 16;
    const uint32_t there[2] = {valid[0] >> row, valid[1] >> row};
    uint32_t acc[4] = {};
#pragma unroll
    for (int q = 0; q < AT_TILE / 4; ++q) {
        const bool is = there[q >> 3] >> (4 * (q & 7)) & 1;
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
            uint4 &p = *reinterpret_cast<uint4 *>(mine + h * AT_TILE * 128 + q * 512);
            if (!is) p = make_uint4(0, 0, 0, 0);
            const uint4 v = p;
            acc[0] = at_zero_fma<F16>(v.x, acc[0]), acc[1] = at_zero_fma<F16>(v.y, acc[1]);
            acc[2] = at_zero_fma<F16>(v.z, acc[2]), acc[3] = at_zero_fma<F16>(v.w, acc[3]);
        }
    }
    if (__any_sync(0xffffffffu, not_finite16x2<F16>(acc[0]) || not_finite16x2<F16>(acc[1]) || not_finite16x2<F16>(acc[2]) || not_finite16x2<F16>(acc[3])))
        at_clean_values<F16, D>(mine, from, row, odd);
}

template <bool F16, int D>
__global__ void __launch_bounds__(AT_THREADS, AT_PER_SM) tree_attention_tiles_kernel(AttendArgs a, const __grid_constant__ CUtensorMap k_map,
                                                                                            const __grid_constant__ CUtensorMap v_map, int box, long long limit) {
    constexpr uint32_t IDESC = (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(AT_ROWS >> 4) << 24);
    constexpr uint32_t IDESC_QK = IDESC | ((uint32_t)(AT_TILE >> 3) << 17), IDESC_PV = IDESC | (1u << 16) | ((uint32_t)(D >> 3) << 17);
    constexpr int HALF = AT_TILE * 128, Q_HALF = AT_ROWS * 128;  // bytes of 64 columns of an operand
    constexpr int PART = AT_ROWS * (D + 2);
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *qs = smem, *ks = smem + AT_ROWS * D * 2, *vs = ks + 2 * AT_OPERAND<D>;
    AttendTilesShared &sh = *reinterpret_cast<AttendTilesShared *>(vs + 2 * AT_OPERAND<D>);
    long long *cum = reinterpret_cast<long long *>(&sh + 1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = a.n_heads / a.cache.n_kv, page_size = a.cache.page_size;
    const uint32_t k_full = smem_u32(sh.k_full), v_full = smem_u32(sh.v_full), scored = smem_u32(sh.scored), added = smem_u32(sh.added),
                   weighed = smem_u32(sh.weighed), q_full = smem_u32(&sh.q_full), q_free = smem_u32(&sh.q_free), summed = smem_u32(&sh.summed);
    if (tid == 0) {
        for (int b = 0; b < 16; b += 8) {
            mbar_init(k_full + b, 1);
            mbar_init(v_full + b, 1);
            mbar_init(scored + b, 1);
            mbar_init(added + b, 1);
            mbar_init(added + 16 + b, 1);
            mbar_init(weighed + b, 128);
        }
        mbar_init(q_full, 1);
        mbar_init(q_free, 1);
        mbar_init(summed, 1);
        mbar_init(smem_u32(&sh.v_landed), 1);
        mbar_init(smem_u32(&sh.drained), 1);
        for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&sh.found[i]), 1);
        mbar_fence_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    if (warp == 7) {
        dg_tmem_alloc(smem_u32(&sh.tmem), AT_COLS);
        dg_tmem_relinquish();
    }
    // (few requests without masks may be long prompts, whose segments differ: a warp per request adds theirs up)
    const bool by_warp = !a.mask && a.R <= 64;
    auto all_units = [&](long long pad) {
        for (int r = warp; by_warp && r < a.R; r += AT_THREADS / 32) {
            const AttendRequest q = attend_request(a, r);
            const int m_tiles = (int)at_div((long long)q.n * group + AT_ROWS - 1, AT_ROWS);
            long long tiles = 0;
            for (int m = lane; m < m_tiles; m += 32) tiles += AttendWalk<D>::at_padded(at_tiles(a, q, group, m), pad);
#pragma unroll
            for (int d = 16; d; d >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, d);
            if (lane == 0) cum[r] = tiles * a.cache.n_kv;
        }
        __syncthreads();
        return scan_units<AT_THREADS>(a, cum, [&](const AttendRequest &q, int r) {
            if (by_warp) return cum[r];
            const int m_tiles = (int)at_div((long long)q.n * group + AT_ROWS - 1, AT_ROWS);
            long long tiles = 0;
            if (a.mask) tiles = m_tiles * AttendWalk<D>::at_padded(at_tiles(a, q, group, 0), pad);
            else for (int m = 0; m < m_tiles; ++m) tiles += AttendWalk<D>::at_padded(at_tiles(a, q, group, m), pad);
            return tiles * a.cache.n_kv;
        });
    };
    long long units = all_units(1), per = max((units + gridDim.x - 1) / gridDim.x, 1LL), pad = 1;
    // Segments of the same keys (a request's rows beyond 128) should run in step, so that the keys come from memory once.  They do if
    // every segment begins at a CTA of its own; that takes longer parts, so it is done where the keys, counted once per segment, do not stay in
    // the L2 anyway: two trees of 64 over 32000 tokens, 64/8 heads of 128 (262 MB), 171 us, 197 without; four prompts of 512 behind 2000 to 4000 (50 MB)
    // 153 either way.  Whether any two segments do share keys is not looked at: steps where none do pay for the search, some passes over the
    // requests' lengths, too.
    if (units * (AT_TILE * D * 4LL) > AT_STEP_BYTES) {
        if (all_units(per) <= (per + per / 4) * gridDim.x)
            for (long long p = per; pad == 1 && p <= per + per / 4; p += max(per / 32, 1LL))
                if (all_units(p) <= p * gridDim.x) pad = p;
        if (pad > 1) per = pad;
        units = pad > 1 ? cum[a.R] : all_units(1);
    }
    dg_fence_before();
    __syncthreads();
    dg_fence_after();
    const uint32_t tmem = sh.tmem, tmem_o = tmem + 2 * AT_TILE;
    AttendSegment g;
    bool ok = true;
    int n = 0;  // tiles so far: tile n has place n % 2 of everything that is held twice, in phase n / 2 % 2
    int cleaned = 0;  // of the warp that brings V: tiles that were put right before the product had them
    auto bar_of = [](uint32_t bar, int t) { return bar + 8 * (t & 1); };
    // keys that all rows of a segment see, from the front on
    auto seen_by_all = [&](const AttendSegment &s) { return s.len + (a.mask ? 0 : s.m * AT_ROWS / group + 1); };
    // the next segment, as warp 6 has found it
    auto next = [&](int seg) {
        ok = mbar_wait_bounded_warp(smem_u32(&sh.found[seg & 3]), seg >> 2 & 1, limit);
        if (ok) g = sh.segments[seg & 3];
        return ok && g.tiles > 0;
    };
    auto phase_of = [](int t) { return (uint32_t)(t >> 1 & 1); };
    auto added_of = [&](int t) { return added + 8 * (t & 3); };
    auto added_phase = [](int t) { return (uint32_t)(t >> 2 & 1); };

    if (box && (warp == 4 || warp == 5)) {
        // ---- TMA: warp 4 K, warp 5 V; lane l brings box l of a tile ----
        const bool is_v = warp == 5;
        const CUtensorMap *map = is_v ? &v_map : &k_map;
        const int boxes = AT_TILE / box;
        const uint32_t landed = smem_u32(&sh.v_landed);
        if (lane == 0) tma_prefetch_desc(map);
        for (int seg = 0; ok && next(seg); ++seg) {
            const int total = g.len + g.n;
            const int32_t *table = a.table + g.r * a.table_stride;
            auto page_of = [&](int i) {
                const int key = (g.tile0 + i) * AT_TILE + lane * box;
                return i < g.tiles && lane < boxes && key < total ? __ldg(table + page_index(a, key)) : -1;
            };
            int page = page_of(0);
            for (int i = 0; i < g.tiles; ++i, ++n) {
                const int key0 = (g.tile0 + i) * AT_TILE, first = key0 + lane * box, off = first - page_index(a, first) * page_size;
                const bool there = (unsigned)page < (unsigned)a.cache.n_pages;
                if (lane < boxes && first < total && !there) req_error(&a.header->error, REQ_ERR_PAGE);
                const uint32_t got = __ballot_sync(0xffffffffu, there);
                uint32_t valid[2];
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    valid[k] = __ballot_sync(0xffffffffu, (got >> ((32 * k + lane) / box) & 1) && key0 + 32 * k + lane < total);
                // (A wait tells a phase from the one before it only; that one, of tile n - 4 or n - 6, this warp has seen.)
                if (n > 1 && !(ok = is_v ? mbar_wait_bounded_warp(added_of(n - 2), added_phase(n - 2), limit)
                                         : mbar_wait_bounded_warp(bar_of(scored, n), phase_of(n - 2), limit)))
                    break;
                // (scores of tile n - 2 were asked for behind the weights of tile n - 4, whose place this is)
                if (!is_v && lane == 0) sh.valid[n & 3][0] = valid[0], sh.valid[n & 3][1] = valid[1];
                // V of new tokens and of slots without a token: see below
                const bool clean = is_v && (key0 + AT_TILE > seen_by_all(g) || (valid[0] & valid[1]) != 0xffffffffu);
                const uint32_t bar = clean ? landed : bar_of(is_v ? v_full : k_full, n);
                if (lane == 0) mbar_expect_tx(bar, __popc(got) * box * 128 * (D / 64));
                __syncwarp();
                if (there) {
                    const uint32_t dst = smem_u32((is_v ? vs : ks) + (n & 1) * AT_OPERAND<D>) + lane * box * 128;
#pragma unroll
                    for (int h = 0; h < D / 64; ++h) tma_load_4d(dst + h * HALF, map, 64 * h, g.hk, off, page, bar);
                }
                page = page_of(i + 1);
                if (clean) {
                    // A weight of 0 must not meet infinity or NaN: slots without a token become 0, and of new tokens, which some rows do
                    // not see, what is not finite; it is added where it is seen, at the end.
                    if (!(ok = mbar_wait_bounded_warp(landed, cleaned++ & 1, limit))) break;
                    at_clean<F16, D>(vs + (n & 1) * AT_OPERAND<D>, valid, seen_by_all(g) - key0, lane, &sh.odd[seg & 3]);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_of(v_full, n));
                }
            }
        }
    } else if (warp == 4 || warp == 5) {
        // ---- the same by copies: lanes 8 i to 8 i + 7 bring lines of keys 4 q + i ----
        const bool is_v = warp == 5;
        const int ck = lane >> 3, cp = lane & 7;
        long long *places = sh.places[is_v];
        for (int seg = 0; ok && next(seg); ++seg) {
            const int total = g.len + g.n;
            const int32_t *table = a.table + g.r * a.table_stride;
            const uint16_t *base = (is_v ? a.cache.v + g.hk * a.cache.v_head : a.cache.k + g.hk * a.cache.k_head) + 8 * cp;
            const long long s_page = is_v ? a.cache.v_page : a.cache.k_page, s_slot = is_v ? a.cache.v_slot : a.cache.k_slot;
            for (int i = 0; i < g.tiles; ++i, ++n) {
                const int key0 = (g.tile0 + i) * AT_TILE;
                uint32_t valid[2];
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int key = key0 + 32 * k + lane, block = page_index(a, key);
                    const int page = key < total ? __ldg(table + block) : -1;
                    const bool there = (unsigned)page < (unsigned)a.cache.n_pages;
                    if (key < total && !there) req_error(&a.header->error, REQ_ERR_PAGE);
                    places[32 * k + lane] = there ? page * s_page + (key - block * page_size) * s_slot : -8;
                    valid[k] = __ballot_sync(0xffffffffu, there);
                }
                __syncwarp();
                if (n > 1 && !(ok = is_v ? mbar_wait_bounded_warp(added_of(n - 2), added_phase(n - 2), limit)
                                         : mbar_wait_bounded_warp(bar_of(scored, n), phase_of(n - 2), limit)))
                    break;
                if (!is_v && lane == 0) sh.valid[n & 3][0] = valid[0], sh.valid[n & 3][1] = valid[1];
                const uint32_t to = smem_u32((is_v ? vs : ks) + (n & 1) * AT_OPERAND<D>) + ck * 128;
                at_copy_keys<D, 0, AT_TILE / 4>(to + (cp ^ ck) * 16, to + (cp ^ ck ^ 4) * 16, base, places + ck);
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncwarp();
                if (is_v && (key0 + AT_TILE > seen_by_all(g) || (valid[0] & valid[1]) != 0xffffffffu))
                    at_clean<F16, D>(vs + (n & 1) * AT_OPERAND<D>, valid, seen_by_all(g) - key0, lane, &sh.odd[seg & 3]);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_of(is_v ? v_full : k_full, n));
            }
        }
    } else if (warp == 6) {
        // ---- what comes next: the segment for everyone, then its Q, as soon as the last scores of the one before are there ----
        const int ck = lane >> 3, cp = lane & 7, step_j = 4 / group, step_h = 4 % group;
        AttendWalk<D> walk{a, cum, blockIdx.x * per, min((blockIdx.x + 1) * per, units), group, pad};
        for (int seg = 0; ok; ++seg) {
            const bool more = walk.next(g, per);
            if (!more) g.tiles = 0;
            // (Its place was that of segment seg - 4.  The scores of seg - 2 are there, so that all of seg - 3 has been weighed: everybody has its
            // description, and nobody is still with seg - 4.)
            if (lane == 0) {
                sh.odd[seg & 3] = 0;  // (read for seg - 4 before anything of seg - 3 was weighed)
                sh.segments[seg & 3] = g;
                mbar_arrive(smem_u32(&sh.found[seg & 3]));
            }
            if (!more) break;
            const int rows = (int)min((long long)AT_ROWS, (long long)g.n * group - (long long)g.m * AT_ROWS);
            unsigned long long bits[AT_ROWS / 32];
#pragma unroll
            for (int k = 0; k < AT_ROWS / 32; ++k)
                bits[k] = a.mask && 32 * k + lane < rows ? (unsigned long long)a.mask[g.q0 + (g.m * AT_ROWS + 32 * k + lane) / group] : 0;
            if (seg && !(ok = mbar_wait_bounded_warp(q_free, (seg - 1) & 1, limit))) break;
            const uint32_t to = smem_u32(qs) + ck * 128;
            const uint16_t *base = a.q + (long long)g.q0 * a.q_row + (long long)g.hk * group * a.q_head + 8 * cp;
            int j = (g.m * AT_ROWS + ck) / group, h = (g.m * AT_ROWS + ck) % group;  // token and head of row 4 q + ck
            // (rows that there are not are worked on like the others, and not stored)
#pragma unroll 4
            for (int q = 0; q < (rows + 3) / 4; ++q) {
                if (4 * q + ck < rows) copies16<D / 64, Q_HALF, 128>(to + q * 512 + (cp ^ ((4 * q + ck) & 7)) * 16, base + (j * a.q_row + h * a.q_head), 16);
                h += step_h;
                j += step_j;
                if (h >= group) h -= group, ++j;
            }
#pragma unroll
            for (int k = 0; k < AT_ROWS / 32; ++k) sh.bits[seg & 1][32 * k + lane] = bits[k];
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (a.scale_log2 < 0.f) {  // a negative scale turns Q's signs
                __syncwarp();
                for (int q = 0; q < AT_ROWS / 4; ++q)
#pragma unroll
                    for (int x = 0; x < D / 64; ++x) {
                        uint4 &v = *reinterpret_cast<uint4 *>(qs + x * Q_HALF + (4 * q + ck) * 128 + cp * 16);
                        v = make_uint4(v.x ^ 0x80008000u, v.y ^ 0x80008000u, v.z ^ 0x80008000u, v.w ^ 0x80008000u);
                        // (every piece of a row is some lane's, whatever its place)
                    }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
    } else if (warp == 7) {
        // ---- products: the scores of a tile are asked for before the weighted sum of the one in front of it ----
        const uint64_t q_desc = dg_desc_sw128(smem_u32(qs)), k_desc = dg_desc_sw128(smem_u32(ks)), v_desc = at_desc_mn(smem_u32(vs), HALF);
        auto score = [&](int t, bool last) {
            ok = mbar_wait_bounded_warp(bar_of(k_full, t), phase_of(t), limit);
            if (!ok) return;
            dg_fence_after();
            if (elect_one()) {
                const uint64_t kd = k_desc + (t & 1) * (AT_OPERAND<D> >> 4);
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    dg_umma_bf16(tmem + (t & 1) * AT_TILE, q_desc + (k >> 2) * (Q_HALF >> 4) + 2 * (k & 3), kd + (k >> 2) * (HALF >> 4) + 2 * (k & 3), IDESC_QK, k > 0);
                dg_umma_commit(bar_of(scored, t));
                if (last) dg_umma_commit(q_free);
            }
            __syncwarp();
        };
        for (int seg = 0; ok && next(seg); ++seg) {
            if (!(ok = mbar_wait_bounded_warp(q_full, seg & 1, limit))) break;
            score(n, g.tiles == 1);
            for (int i = 0; ok && i < g.tiles; ++i, ++n) {
                if (i + 1 < g.tiles) score(n + 1, i + 2 == g.tiles);
                if (!ok) break;
                if (!(ok = mbar_wait_bounded_warp(bar_of(v_full, n), phase_of(n), limit) && mbar_wait_bounded_warp(bar_of(weighed, n), phase_of(n), limit))) break;
                dg_fence_after();
                if (elect_one()) {
                    const uint64_t vd = v_desc + (n & 1) * (AT_OPERAND<D> >> 4);
#pragma unroll
                    for (int k = 0; k < AT_TILE / 16; ++k)
                        dg_umma_bf16_ta(tmem_o, tmem + (n & 1) * AT_TILE + 8 * k, vd + k * (2048 >> 4), IDESC_PV, i > 0 || k > 0);
                    dg_umma_commit(added_of(n));
                    if (i + 1 == g.tiles) dg_umma_commit(summed);
                }
                __syncwarp();
            }
        }
    } else if (warp < 4) {
        // ---- a row a thread ----
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const float scale = fmaxf(fabsf(a.scale_log2), 1.17549435e-38f);  // (a negative one has turned Q's signs; 0 times -inf is not a number)
        float *parts = reinterpret_cast<float *>(a.scratch + AT_JOINS + sizeof(AttendJoin) * AT_MAX_CTAS);
        AttendJoin *joins = reinterpret_cast<AttendJoin *>(a.scratch + AT_JOINS);
        bool joined = false;
        for (int seg = 0; ok && next(seg); ++seg) {
            const int rows = (int)min((long long)AT_ROWS, (long long)g.n * group - (long long)g.m * AT_ROWS);
            const bool mine = tid < rows, busy = warp * 32 < rows;
            const int row = g.m * AT_ROWS + tid, j = row / group, head = g.hk * group + row % group;
            unsigned long long bits = 0;
            const int all_see = seen_by_all(g);
            float top = -INFINITY, sum = 0.f;
            for (int i = 0; i < g.tiles; ++i, ++n) {
                if (!(ok = mbar_wait_bounded_warp(bar_of(scored, n), phase_of(n), limit))) break;
                dg_fence_after();
                if (i == 0) bits = sh.bits[seg & 1][tid];  // (there with Q.  Q of the next but one segment may be there too by now: no wait for q_full)
                if (busy) {
                    const uint32_t s_cols = tmem + lanes + (n & 1) * AT_TILE;
                    const int key0 = (g.tile0 + i) * AT_TILE;
                    uint32_t v[2][32];
                    dg_tmem_ld_32x32b_x32(s_cols, v[0]);
                    dg_tmem_ld_32x32b_x32(s_cols + 32, v[1]);
                    uint32_t vis[2] = {sh.valid[n & 3][0], sh.valid[n & 3][1]};
                    dg_tmem_ld_wait();
                    if (key0 + AT_TILE > all_see || (vis[0] & vis[1]) != 0xffffffffu) at_mask(a, g.len, key0, j, bits, vis, v);
                    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 32; ++e) m0 = fmaxf(m0, __uint_as_float(v[0][e])), m1 = fmaxf(m1, __uint_as_float(v[1][e]));
                    float m = fmaxf(m0, m1);
                    if (m != -INFINITY) m *= scale;
                    if (__any_sync(0xffffffffu, m > top + 8.f)) {
                        const float to = fmaxf(m, top), keep = to == -INFINITY ? 1.f : exp2_fast(top - to);
                        top = to;
                        sum *= keep;
                        if (i > 0) {
                            if (!(ok = mbar_wait_bounded_warp(added_of(n - 1), added_phase(n - 1), limit))) break;
                            dg_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D / 16; ++c) {
                                uint32_t u[16];
                                dg_tmem_ld_32x32b_x16(tmem_o + lanes + 16 * c, u);
                                dg_tmem_ld_wait();
#pragma unroll
                                for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(__uint_as_float(u[e]) * keep);
                                at_tmem_st_x16(tmem_o + lanes + 16 * c, u);
                            }
                        }
                    }
                    const float ref = (top == -INFINITY ? 0.f : top) - WEIGHT_LIFT<F16>;
                    uint64_t sums[2] = {0, 0};
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t p[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float x0, x1;
                            at_fma2(x0, x1, __uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1]), scale, -ref);
                            x0 = exp2_fast(x0), x1 = exp2_fast(x1);
                            at_add2(sums[e & 1], x0, x1);
                            p[e] = pack16x2<F16>(x0, x1);
                        }
                        at_tmem_st_x16(s_cols + 16 * c, p);  // (over scores that have been read)
                    }
                    sum += at_sum2(sums[0]) + at_sum2(sums[1]);
                    dg_tmem_st_wait();
                }
                dg_fence_before();
                mbar_arrive(bar_of(weighed, n));
            }
            if (!ok) break;
            if (!(ok = mbar_wait_bounded_warp(summed, seg & 1, limit))) break;
            dg_fence_after();
            // ---- the segment's sums: out, or to the CTA that joins them ----
            const int c0 = g.c0, c1 = g.c1;
            const bool whole = c0 == c1;
            const bool odd = *reinterpret_cast<volatile int *>(&sh.odd[seg & 3]) != 0;
            float *part = parts + (long long)(2 * blockIdx.x + ((int)blockIdx.x == c0 ? 1 : 0)) * PART;  // [D + 2][128]
            uint16_t *out = a.out + (long long)(g.q0 + j) * a.o_row + (long long)head * a.o_head;
            auto store32 = [&](int c, const float (&o)[32], float total) {
                const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
                for (int e = 0; e < 32; e += 8)
                    *reinterpret_cast<uint4 *>(out + 32 * c + e) =
                        make_uint4(pack16x2<F16>(o[e] * inv, o[e + 1] * inv), pack16x2<F16>(o[e + 2] * inv, o[e + 3] * inv),
                                   pack16x2<F16>(o[e + 4] * inv, o[e + 5] * inv), pack16x2<F16>(o[e + 6] * inv, o[e + 7] * inv));
            };
            if (busy) {
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t v[32];
                    float o[32];
                    dg_tmem_ld_32x32b_x32(tmem_o + lanes + 32 * c, v);
                    dg_tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(v[e]);
                    if (odd && mine) {
                        const int first = max(g.tile0 * AT_TILE - g.len, 0), last = min((g.tile0 + g.tiles) * AT_TILE - g.len, g.n);
                        for (int d = first; d < last; ++d) {
                            if (!(a.mask ? d < 64 && (bits >> d & 1) : d <= j)) continue;
                            const int key = g.len + d, page = a.table[g.r * a.table_stride + page_index(a, key)];
                            if ((unsigned)page >= (unsigned)a.cache.n_pages) continue;
                            const uint16_t *src = a.cache.v + page * a.cache.v_page + (key - page_index(a, key) * page_size) * a.cache.v_slot + g.hk * a.cache.v_head + 32 * c;
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (not_finite16x2<F16>(src[e])) o[e] += unpack16x2<F16>(src[e]).x;
                        }
                    }
                    if (whole) {
                        if (mine) store32(c, o, sum);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) part[(32 * c + e) * AT_ROWS + tid] = o[e];
                    }
                }
                if (!whole) part[D * AT_ROWS + tid] = top, part[(D + 1) * AT_ROWS + tid] = sum;
            }
            dg_fence_before();
            // what begins here and goes on is this CTA's last segment
            if (tid == 0 && !whole && (int)blockIdx.x == c0) joins[blockIdx.x] = AttendJoin{c1, g.q0, g.n, g.hk, g.m}, joined = true;
        }
        if (tid == 0 && !joined) joins[blockIdx.x].last = -1;
    }
    if (!ok) {
        // A wait gave up, here or, as its consequence, in other warps one after another: the roles wait for each other at mbarriers alone, all
        // with a limit.  What this warp has on its way into shared or tensor memory must be there before the CTA gives these back.
        if (lane == 0) req_error(&a.header->error, REQ_ERR_TIMEOUT);
        if (box && (warp == 4 || warp == 5)) {
            for (int t = max(n - 2, 0); t < n; ++t) mbar_wait_bounded_warp(bar_of(warp == 5 ? v_full : k_full, t), phase_of(t), WAIT_LIMIT_DEFAULT);
            if (warp == 5 && cleaned > 0) mbar_wait_bounded_warp(smem_u32(&sh.v_landed), (cleaned - 1) & 1, WAIT_LIMIT_DEFAULT);
        } else if (warp == 7) {
            if (elect_one()) dg_umma_commit(smem_u32(&sh.drained));
            __syncwarp();
            mbar_wait_bounded_warp(smem_u32(&sh.drained), 0, WAIT_LIMIT_DEFAULT);
        }
    }
    dg_fence_before();
    __syncthreads();
    dg_fence_after();
    if (warp == 6) dg_tmem_dealloc(tmem, AT_COLS);
}

// The parts of the segments that several CTAs have shared: a CTA per segment and 16 columns, a thread per row.  (Done by the last
// CTA to finish a segment it took that one 10 to 15 us, with its next segment waiting.)
constexpr int AJ_COLS = 16;
template <bool F16, int D>
__global__ void __launch_bounds__(AT_ROWS) tree_attention_join_kernel(AttendArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    constexpr int PART = AT_ROWS * (D + 2);
    const int c0 = blockIdx.x, tid = threadIdx.x, d0 = blockIdx.y * AJ_COLS, group = a.n_heads / a.cache.n_kv;
    const AttendJoin s = reinterpret_cast<const AttendJoin *>(a.scratch + AT_JOINS)[c0];
    const int row = s.m * AT_ROWS + tid;
    if (s.last < 0 || row >= s.n * group) return;
    const float *parts = reinterpret_cast<const float *>(a.scratch + AT_JOINS + sizeof(AttendJoin) * AT_MAX_CTAS);
    float top = -INFINITY, total = 0.f, o[AJ_COLS] = {};
    for (int c = c0; c <= s.last; c += 4) {  // four parts' values on their way at a time
        float m[4], l[4], v[4][AJ_COLS];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float *src = parts + (long long)(2 * min(c + k, s.last) + (c + k == c0)) * PART + tid;
            m[k] = c + k <= s.last ? src[D * AT_ROWS] : -INFINITY;
            l[k] = src[(D + 1) * AT_ROWS];
#pragma unroll
            for (int e = 0; e < AJ_COLS; ++e) v[k][e] = src[(d0 + e) * AT_ROWS];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float to = fmaxf(top, m[k]), ref = to == -INFINITY ? 0.f : to, keep = exp2_fast(top - ref), f = exp2_fast(m[k] - ref);
            top = to;
            total = total * keep + (c + k <= s.last ? l[k] * f : 0.f);
            // (a part that saw nothing has no sums; of one whose weights come out as 0, NaN stays NaN)
#pragma unroll
            for (int e = 0; e < AJ_COLS; ++e) o[e] = o[e] * keep + (m[k] == -INFINITY ? 0.f : v[k][e] * f);
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    uint16_t *out = a.out + (long long)(s.q0 + row / group) * a.o_row + (long long)(s.hk * group + row % group) * a.o_head + d0;
#pragma unroll
    for (int e = 0; e < AJ_COLS; e += 8)
        *reinterpret_cast<uint4 *>(out + e) = make_uint4(pack16x2<F16>(o[e] * inv, o[e + 1] * inv), pack16x2<F16>(o[e + 2] * inv, o[e + 3] * inv),
                                                         pack16x2<F16>(o[e + 4] * inv, o[e + 5] * inv), pack16x2<F16>(o[e + 6] * inv, o[e + 7] * inv));
}

size_t tree_attention_scratch_bytes() {
    const size_t rows = (size_t)2 * AR_MAX_CTAS * AR_ROWS * (128 + 2) * 4,
                 tiles = sizeof(AttendJoin) * AT_MAX_CTAS + (size_t)2 * AT_MAX_CTAS * AT_ROWS * (128 + 2) * 4;
    return 4 * AR_MAX_CTAS + (rows > tiles ? rows : tiles);
}

}  // namespace awq

using namespace awq;

extern "C" int awq_b200_tree_attention(const void *q, long long q_row_stride, long long q_head_stride, const awq_b200_kv_cache_t *cache,
                                       const int32_t *table, long long table_stride, int table_width, const int32_t *lens,
                                       const int32_t *q_start, const long long *mask, float scale, void *out, long long out_row_stride,
                                       long long out_head_stride, int R, int T, int n_heads, void *workspace, size_t workspace_bytes,
                                       awq_stream_t stream) {
    KvCacheView view;
    int rc = check_kv_cache("tree_attention", cache, &view);
    if (rc) return rc;
    AWQ_REQUIRE(R >= 0 && R <= REQ_MAX_REQUESTS && T >= 0 && T <= REQ_MAX_ROWS && table_width >= 0, "tree_attention: at most %d requests and %d rows",
                REQ_MAX_REQUESTS, REQ_MAX_ROWS);
    AWQ_REQUIRE(n_heads > 0 && n_heads % view.n_kv == 0, "tree_attention: n_heads (%d) must be a multiple of the cache's heads (%d)", n_heads, view.n_kv);
    AWQ_REQUIRE(table_stride >= table_width, "tree_attention: the stride of the block table is below its width");
    AWQ_REQUIRE(isfinite(scale), "tree_attention: the scale must be finite");
    const long long s[4] = {q_row_stride, q_head_stride, out_row_stride, out_head_stride};
    for (long long x : s) AWQ_REQUIRE(x >= 0 && x % 8 == 0, "tree_attention: strides must be multiples of 8 elements");
    if (R == 0 || T == 0) return AWQ_OK;
    AWQ_REQUIRE((T == 1 || out_row_stride > 0) && (n_heads == 1 || out_head_stride > 0), "tree_attention: an output stride of 0 needs a dimension of one");
    AWQ_REQUIRE(q && out && table && lens && q_start, "tree_attention: null pointer");
    AWQ_REQUIRE(aligned16(q) && aligned16(out), "tree_attention: pointers must be 16-byte aligned");
    AWQ_REQUIRE_REQUEST_WORKSPACE("tree_attention", workspace, workspace_bytes);
    const RequestWorkspaceView w = request_workspace(workspace);
    AttendArgs a{reinterpret_cast<const uint16_t *>(q), s[0], s[1], view, table, table_stride, lens, q_start, mask,
                 reinterpret_cast<uint16_t *>(out), s[2], s[3], scale * 1.4426950408889634f, R, T, n_heads, table_width,
                 view.page_size & (view.page_size - 1) ? -1 : __builtin_ctz(view.page_size), w.header, w.attention};
    const bool f16 = cache->format == ACT_F16;
    auto launch_rows = [&](auto kernel, int smem) {
        if (int e = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "tree_attention shared memory")) return e;
        const int grid = min(device_sm_count() * AR_PER_SM, AR_MAX_CTAS);
        return check_cuda(launch_pdl(kernel, dim3(grid), dim3(AR_WARPS * 32), smem, as_stream(stream), a), "tree_attention launch");
    };
    if (view.head_dim == 64 || view.head_dim == 128) {
        // More rows than one mma.sync tile has, on average: tcgen05.  32 requests of 2000 to 4000 tokens, 32/8 heads of 128, trees of 4 (16
        // rows per head): mma.sync 79 us, tcgen05 89; trees of 8 (32 rows): 118 and 92.  The host knows the average alone, over all R requests, those
        // that bring no rows too, and one kernel takes the whole step: a prompt's chunk of 1000 rows beside 63 single tokens takes 177 us, the two
        // apart 77 and 66; 8 trees of 32 among 64 requests 64 us, without the idle ones 40.
        if ((long long)T * (n_heads / view.n_kv) > (long long)AR_ROWS * R) {
            auto kernel = view.head_dim == 64 ? (f16 ? tree_attention_tiles_kernel<true, 64> : tree_attention_tiles_kernel<false, 64>)
                                              : (f16 ? tree_attention_tiles_kernel<true, 128> : tree_attention_tiles_kernel<false, 128>);
            const int smem = (view.head_dim == 64 ? AT_SMEM<64> : AT_SMEM<128>) + (R + 1) * 8;
            if ((rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "tree_attention shared memory"))) return rc;
            const int grid = min(device_sm_count() * AT_PER_SM, AT_MAX_CTAS);
            // boxes of slots that never straddle a page or a tile
            int box = AT_TILE;
            while (box >= 8 && view.page_size % box) box >>= 1;
            CUtensorMap maps[2] = {};
            const long long longest = 1LL << 38;  // elements of 2 bytes: TMA strides are below 2^40 bytes
            if (box < 8 || view.k_page > longest || view.v_page > longest || view.k_slot > longest || view.v_slot > longest || view.k_head > longest || view.v_head > longest)
                box = 0;
            for (int i = 0; box && i < 2; ++i) {
                const long long st[3] = {i ? view.v_head : view.k_head, i ? view.v_slot : view.k_slot, i ? view.v_page : view.k_page};
                // (a dimension of one may come with a stride of 0)
                const uint64_t strides[3] = {(uint64_t)max(2 * st[0], 16LL), (uint64_t)max(2 * st[1], 16LL), (uint64_t)max(2 * st[2], 16LL)};
                if ((rc = encode_tensor_map_4d(&maps[i], f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, i ? view.v : view.k,
                                               {(uint64_t)view.head_dim, (uint64_t)view.n_kv, (uint64_t)view.page_size, (uint64_t)view.n_pages}, strides,
                                               {64u, 1u, (uint32_t)box, 1u}, CU_TENSOR_MAP_SWIZZLE_128B)))
                    return rc;
            }
            if ((rc = check_cuda(launch_pdl(kernel, dim3(grid), dim3(AT_THREADS), smem, as_stream(stream), a, maps[0], maps[1], box, wait_limit_cycles()),
                                 "tree_attention launch")))
                return rc;
            auto join = view.head_dim == 64 ? (f16 ? tree_attention_join_kernel<true, 64> : tree_attention_join_kernel<false, 64>)
                                            : (f16 ? tree_attention_join_kernel<true, 128> : tree_attention_join_kernel<false, 128>);
            return check_cuda(launch_pdl(join, dim3(grid, view.head_dim / AJ_COLS), dim3(AT_ROWS), 0, as_stream(stream), a), "tree_attention join launch");
        }
        return launch_rows(view.head_dim == 64 ? (f16 ? tree_attention_rows_kernel<true, 64, false> : tree_attention_rows_kernel<false, 64, false>)
                                               : (f16 ? tree_attention_rows_kernel<true, 128, false> : tree_attention_rows_kernel<false, 128, false>),
                           view.head_dim == 64 ? AR_SMEM<64> : AR_SMEM<128>);
    }
    if (view.head_dim < 128)
        return launch_rows(view.head_dim < 64 ? (f16 ? tree_attention_rows_kernel<true, 64, true> : tree_attention_rows_kernel<false, 64, true>)
                                              : (f16 ? tree_attention_rows_kernel<true, 128, true> : tree_attention_rows_kernel<false, 128, true>),
                           view.head_dim < 64 ? AR_SMEM<64> : AR_SMEM<128>);
    AWQ_REQUIRE((long long)T * n_heads <= 0x7fffffffLL, "tree_attention: too many rows and heads");
    auto kernel = f16 ? tree_attention_any_kernel<true> : tree_attention_any_kernel<false>;
    return check_cuda(launch_pdl(kernel, dim3((unsigned)(T * n_heads)), dim3(AA_WARPS * 32), 0, as_stream(stream), a), "tree_attention launch");
}
