// Low-rank adapters of many requests beside a shared projection:
//
//   out[t] = bf16(base[t] + scale[a] (x[t] A[a]^T) B[a]^T (+ residual[t])),   a = idx[t], -1: none.
//
// A [n, rank_max, K] and B [n, N, rank_max] hold rank[a] rows / columns of each adapter; what lies behind them is not read.
#include "awq_request.cuh"

#include <math.h>

namespace awq {

struct LoraArgs {
    const uint16_t *x, *A, *B;
    const float *scales;
    const int32_t *ranks, *idx;
    const void *base;
    const uint16_t *residual;
    uint16_t *out;
    long long x_row;
    int base_f32, T, K, N, n, rank_max;
    float *low;  // [T, rank_max] x A^T
    RequestHeader *header;
};

__global__ void __launch_bounds__(128) lora_down_kernel(LoraArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int t = (int)(item / a.rank_max), r = (int)(item % a.rank_max);
    if (t >= a.T) return;
    const int ad = a.idx[t];
    if (ad < 0 || ad >= a.n) {
        if (ad >= a.n && lane == 0) req_error(&a.header->error, REQ_ERR_ADAPTER);
        return;
    }
    const int rank = a.ranks ? min(max(a.ranks[ad], 0), a.rank_max) : a.rank_max;
    if (r >= rank) return;
    const uint16_t *x = a.x + t * a.x_row, *A = a.A + ((long long)ad * a.rank_max + r) * a.K;
    float s = 0.f;
    for (int k = lane; k < a.K; k += 32) s = fmaf(bf16_bits_to_f32(x[k]), bf16_bits_to_f32(A[k]), s);
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0) a.low[(long long)t * a.rank_max + r] = s * a.scales[ad];
}

__global__ void __launch_bounds__(128) lora_up_kernel(LoraArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int t = blockIdx.y, n = blockIdx.x * 128 + threadIdx.x;
    if (n >= a.N) return;
    const int ad = a.idx[t];
    const long long at = (long long)t * a.N + n;
    float s = a.base_f32 ? reinterpret_cast<const float *>(a.base)[at] : bf16_bits_to_f32(reinterpret_cast<const uint16_t *>(a.base)[at]);
    float up = 0.f;
    if (ad >= 0 && ad < a.n) {
        const int rank = a.ranks ? min(max(a.ranks[ad], 0), a.rank_max) : a.rank_max;
        const uint16_t *B = a.B + ((long long)ad * a.N + n) * a.rank_max;
        for (int r = 0; r < rank; ++r) up = fmaf(a.low[(long long)t * a.rank_max + r], bf16_bits_to_f32(B[r]), up);
    }
    s += up;
    if (a.residual) s += bf16_bits_to_f32(a.residual[at]);
    a.out[at] = f32_to_bf16_bits(s);
}

constexpr int LORA_MAX_ROWS = 65535, LORA_MAX_RANK = 128;
size_t lora_scratch_bytes() { return (size_t)LORA_MAX_ROWS * LORA_MAX_RANK * 4; }

}  // namespace awq

using namespace awq;

extern "C" int awq_b200_lora_bf16(const uint16_t *x, long long x_row_stride, const uint16_t *A, const uint16_t *B, const float *scales,
                                  const int32_t *ranks, int n_adapters, int rank_max, const int32_t *idx, const void *base, int base_is_f32,
                                  const uint16_t *residual, uint16_t *out, int T, int K, int N, void *workspace, size_t workspace_bytes,
                                  awq_stream_t stream) {
    AWQ_REQUIRE(T >= 0 && T <= LORA_MAX_ROWS && K > 0 && N >= 0 && n_adapters >= 0, "lora: bad size (at most %d rows)", LORA_MAX_ROWS);
    AWQ_REQUIRE(rank_max > 0 && rank_max <= LORA_MAX_RANK && rank_max % 8 == 0, "lora: rank_max (%d) must be a multiple of 8, at most %d", rank_max,
                LORA_MAX_RANK);
    AWQ_REQUIRE(K % 8 == 0 && N % 8 == 0, "lora: K (%d) and N (%d) must be multiples of 8", K, N);
    AWQ_REQUIRE(x_row_stride >= 0 && x_row_stride % 8 == 0, "lora: the row stride of x must be a multiple of 8 elements");
    if (T == 0 || N == 0) return AWQ_OK;
    AWQ_REQUIRE(x && idx && base && out, "lora: null pointer");
    AWQ_REQUIRE(n_adapters == 0 || (A && B && scales), "lora: null adapter");
    AWQ_REQUIRE(aligned16(x) && aligned16(A) && aligned16(B) && aligned16(base) && aligned16(residual) && aligned16(out),
                "lora: pointers must be 16-byte aligned");
    AWQ_REQUIRE_REQUEST_WORKSPACE("lora", workspace, workspace_bytes);
    const RequestWorkspaceView w = request_workspace(workspace);
    LoraArgs a{x, A, B, scales, ranks, idx, base, residual, out, x_row_stride, base_is_f32, T, K, N, n_adapters, rank_max,
               reinterpret_cast<float *>(w.lora), w.header};
    const long long items = (long long)T * rank_max;
    int rc = check_cuda(launch_pdl(lora_down_kernel, dim3((unsigned)((items + 3) / 4)), dim3(128), 0, as_stream(stream), a), "lora down launch");
    if (rc) return rc;
    return check_cuda(launch_pdl(lora_up_kernel, dim3((N + 127) / 128, T), dim3(128), 0, as_stream(stream), a), "lora up launch");
}
