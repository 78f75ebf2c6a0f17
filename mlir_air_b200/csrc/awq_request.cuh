// What the operators on many requests' rows share (page_plan, rope_append, tree_attention, page_keep, lora): the layout of
// their workspace, the bits of its error word, the paged cache as the kernels see it.
#pragma once

#include "awq_common.cuh"
#include "awq_ptx.cuh"

namespace awq {

// Bits of the error word.  A kernel that meets such an index skips the access, sets the bit and goes on: what the call
// computed for that request is not valid, nothing outside the caller's buffers was touched.
enum RequestError : int {
    REQ_ERR_NO_PAGES = 1,    // page_plan: the step needs more pages than are free
    REQ_ERR_STEP = 2,        // page_plan: lengths or counts that do not fit the batch, the block table or a tree's 64 tokens
    REQ_ERR_PARENT = 4,      // page_plan: a parent that is not an earlier token of its tree
    REQ_ERR_PAGE = 8,        // a page outside the cache
    REQ_ERR_SLOT = 16,       // rope_append: a slot outside the cache or a position outside the table of angles
    REQ_ERR_KEPT = 32,       // page_keep: a count or path that does not fit its request
    REQ_ERR_ADAPTER = 64,    // lora: an adapter that does not exist
    REQ_ERR_REQUEST = 128,   // tree_attention: lengths or starts that do not fit the batch or the block table
    REQ_ERR_TIMEOUT = 256,   // a bounded device-side wait gave up
};

constexpr int REQ_MAX_REQUESTS = 4096;  // a CTA scans all requests' lengths
constexpr int REQ_MAX_ROWS = 1 << 20;
constexpr int REQ_MAX_TREE = 64;        // drafted tokens of a tree: the bits of a mask word

// Workspace: header, then one area per operator (none uses another's, so that launches that follow one another may overlap).
struct RequestHeader {
    int error;
    int plan_arrived, keep_arrived;  // CTAs that are done; back at 0 when the call is
    int pad[61];
};
static_assert(sizeof(RequestHeader) == 256, "header of the request workspace");

struct KvCacheView {  // strides in elements
    const uint16_t *k, *v;
    long long k_page, k_slot, k_head, v_page, v_slot, v_head;
    int n_pages, page_size, n_kv, head_dim;
};

__device__ __forceinline__ void req_error(int *error, int bit) { atomicOr(error, bit); }

// 16-bit floats of either format to f32 and back, two at a time.
template <bool F16>
__device__ __forceinline__ float2 unpack16x2(uint32_t v) {
    if (F16) return __half22float2(*reinterpret_cast<const __half2 *>(&v));
    return make_float2(bf16x2_lo(v), bf16x2_hi(v));
}
template <bool F16>
__device__ __forceinline__ uint32_t pack16x2(float lo, float hi) {
    if (F16) {
        __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&h);
    }
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
}

// The last i in [0, n) with start[i] <= t (start[0] = 0, not decreasing): the request of row t.
__device__ __forceinline__ int request_of_row(const int *start, int n, int t) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

size_t tree_attention_scratch_bytes();
size_t lora_scratch_bytes();
struct RequestWorkspaceView {
    RequestHeader *header;
    uint8_t *attention, *lora;
};
inline size_t request_workspace_bytes() { return sizeof(RequestHeader) + tree_attention_scratch_bytes() + lora_scratch_bytes(); }
inline RequestWorkspaceView request_workspace(void *ws) {
    uint8_t *p = reinterpret_cast<uint8_t *>(ws);
    return {reinterpret_cast<RequestHeader *>(p), p + sizeof(RequestHeader), p + sizeof(RequestHeader) + tree_attention_scratch_bytes()};
}

#define AWQ_REQUIRE_REQUEST_WORKSPACE(who, ws, bytes)                                                                         \
    do {                                                                                                                      \
        if (!(ws) || (bytes) < awq::request_workspace_bytes())                                                                \
            return awq::set_error(AWQ_ERR_WORKSPACE, "%s: workspace of %zu bytes required", who, awq::request_workspace_bytes()); \
        if (!awq::aligned16(ws)) return awq::set_error(AWQ_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", who);    \
    } while (0)

// Argument checks of a cache descriptor; fills `out`.
int check_kv_cache(const char *who, const awq_b200_kv_cache_t *c, KvCacheView *out);

}  // namespace awq
