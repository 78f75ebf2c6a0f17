// Attention of a step's rows over a paged cache.
//
//   out[t, h] = sum_p w_p v_p / sum_p w_p,   w_p = exp(scale q . k_p - max),   p over the keys that row t sees:
//   the len cached tokens of its request, and of the request's own n new tokens those in the row's mask (bit j: token j)
//   or, without masks, those up to itself.  A row that sees nothing is 0.
#include "awq_request.cuh"

#include <cuda_fp16.h>
#include <math.h>

namespace awq {

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
    const long long capacity = min((long long)a.table_width * a.cache.page_size, 0x7fffffffLL);
    q.len = (int)min((long long)max(len, 0), max(capacity - q.n, 0LL));
    q.bad = q.q0 != s || q.q0 + q.n != e || q.len != len || (a.mask && q.n > REQ_MAX_TREE) || q.n > capacity;
    if (q.n > capacity) q.n = 0;
    return q;
}

// Any head size: a warp per row and head, one key after another.  Head sizes that have no tensor-core kernel.
template <bool F16>
__global__ void __launch_bounds__(128) tree_attention_any_kernel(AttendArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int t = (int)(item / a.n_heads), h = (int)(item % a.n_heads);
    if (t >= a.T) return;
    int lo = 0, hi = a.R;  // the request of row t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] <= t) lo = mid; else hi = mid;
    }
    const AttendRequest q = attend_request(a, lo);
    if (q.bad && lane == 0) req_error(&a.header->error, REQ_ERR_REQUEST);
    const int j = t - q.q0;
    if (j < 0 || j >= q.n) return;  // behind the last request
    const int D = a.cache.head_dim, pairs = D >> 1, hk = h / (a.n_heads / a.cache.n_kv);
    const unsigned long long bits = a.mask ? (unsigned long long)a.mask[t] : 0;
    const uint16_t *qp = a.q + t * a.q_row + h * a.q_head;
    float2 qv[4], acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane + 32 * i;
        qv[i] = c < pairs ? unpack16x2<F16>(reinterpret_cast<const uint32_t *>(qp)[c]) : make_float2(0.f, 0.f);
        acc[i] = make_float2(0.f, 0.f);
    }
    float top = -INFINITY, total = 0.f;
    for (int p = 0; p < q.len + q.n; ++p) {
        const int d = p - q.len;
        if (d >= 0 && !(a.mask ? d < 64 && (bits >> d & 1) : d <= j)) continue;
        const int page = a.table[lo * a.table_stride + p / a.cache.page_size], off = p % a.cache.page_size;
        if ((unsigned)page >= (unsigned)a.cache.n_pages) {
            if (lane == 0) req_error(&a.header->error, REQ_ERR_PAGE);
            continue;
        }
        const uint32_t *kp = reinterpret_cast<const uint32_t *>(a.cache.k + page * a.cache.k_page + off * a.cache.k_slot + hk * a.cache.k_head);
        const uint32_t *vp = reinterpret_cast<const uint32_t *>(a.cache.v + page * a.cache.v_page + off * a.cache.v_slot + hk * a.cache.v_head);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = lane + 32 * i;
            if (c < pairs) {
                const float2 k = unpack16x2<F16>(kp[c]);
                s = fmaf(qv[i].x, k.x, fmaf(qv[i].y, k.y, s));
            }
        }
#pragma unroll
        for (int d2 = 16; d2; d2 >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d2);
        s *= a.scale_log2;
        const float m = fmaxf(top, s), keep = m == -INFINITY ? 1.f : exp2f(top - m), w = m == -INFINITY ? 0.f : exp2f(s - m);
        top = m;
        total = total * keep + w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = lane + 32 * i;
            if (c < pairs) {
                const float2 v = unpack16x2<F16>(vp[c]);
                acc[i] = make_float2(fmaf(w, v.x, acc[i].x * keep), fmaf(w, v.y, acc[i].y * keep));
            }
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    uint32_t *op = reinterpret_cast<uint32_t *>(a.out + t * a.o_row + h * a.o_head);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane + 32 * i;
        if (c < pairs) op[c] = pack16x2<F16>(acc[i].x * inv, acc[i].y * inv);
    }
}

size_t tree_attention_scratch_bytes() { return 0; }

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
    AWQ_REQUIRE(q && out && table && lens && q_start, "tree_attention: null pointer");
    AWQ_REQUIRE(aligned16(q) && aligned16(out), "tree_attention: pointers must be 16-byte aligned");
    AWQ_REQUIRE_REQUEST_WORKSPACE("tree_attention", workspace, workspace_bytes);
    const RequestWorkspaceView w = request_workspace(workspace);
    AttendArgs a{reinterpret_cast<const uint16_t *>(q), s[0], s[1], view, table, table_stride, lens, q_start, mask,
                 reinterpret_cast<uint16_t *>(out), s[2], s[3], scale * 1.4426950408889634f, R, T, n_heads, table_width, w.header, w.attention};
    const long long items = (long long)T * n_heads;
    AWQ_REQUIRE((items + 3) / 4 <= 0x7fffffffLL, "tree_attention: too many rows and heads");
    auto kernel = cache->format == ACT_F16 ? tree_attention_any_kernel<true> : tree_attention_any_kernel<false>;
    return check_cuda(launch_pdl(kernel, dim3((unsigned)((items + 3) / 4)), dim3(128), 0, as_stream(stream), a), "tree_attention launch");
}
