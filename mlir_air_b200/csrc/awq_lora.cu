// Low-rank adapters of many requests beside a shared projection:
//
//   out[t] = bf16(base[t] + scale[a] (x[t] A[a]^T) B[a]^T (+ residual[t])),   a = idx[t], -1: none.
//
// A [n, rank_max, K] and B [n, N, rank_max] hold rank[a] rows / columns of each adapter; what lies behind them is not read.
//
// Rows are put together by adapter into tiles, so that an adapter is read once per tile and multiplied on the tensor cores
// (mma.sync: the products are small, the bytes of x, base, out and the adapters are what takes time).  A row's result does not
// depend on its tile or its place in it.  Operands go from global memory to registers in 16-byte pieces: the order of the
// products along K (or the rank) is free as long as both operands have the same one, so eight neighbours of a row are a lane's
// operands of two k-steps.  x A^T stays at f32's accuracy between the products: it is summed in f32 and multiplied as two
// bf16 pieces (hi + lo, 2^-17; of an infinite sum hi is the largest finite value, so that lo is what is infinite and no difference of
// infinities arises).
#include "awq_request.cuh"

#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <math.h>

namespace awq {

namespace cg = cooperative_groups;

constexpr int LORA_MAX_ROWS = 65535, LORA_MAX_RANK = 128, LORA_MAX_ADAPTERS = 4096;

struct LoraArgs {
    const uint16_t *x, *A, *B;
    const float *scales;
    const int32_t *ranks, *idx;
    const void *base;
    const uint16_t *residual;
    uint16_t *out;
    long long x_row;
    int base_f32, T, K, N, n, rank_max;
    RequestHeader *header;
    int32_t *order;   // [T] rows by adapter
    int4 *tiles;      // adapter, first of `order`, rows, rank
    int32_t *n_tiles;
    uint16_t *low;    // [T][2][rank_max up to 32] scale x A^T in the order of `order`, hi and lo
};

__device__ __forceinline__ int lora_rank(const LoraArgs &a, int ad) {
    if (ad >= a.n) return 0;
    return a.ranks ? min(max(a.ranks[ad], 0), a.rank_max) : a.rank_max;
}
// The adapter of a row; a.n: none.
__device__ __forceinline__ int lora_adapter(const LoraArgs &a, int t, bool report) {
    const int ad = a.idx[t];
    if (ad >= a.n && report) req_error(&a.header->error, REQ_ERR_ADAPTER);
    return (unsigned)ad < (unsigned)a.n ? ad : a.n;
}
__device__ __forceinline__ uint4 ldg16(const uint16_t *p, bool on) {
    return on ? __ldg(reinterpret_cast<const uint4 *>(p)) : make_uint4(0, 0, 0, 0);
}

// acc[m][b] += x rows x (rank rows of A)^T over chunks first, first + step, ... < last of 32 columns of K.
template <int MT, int NB>
__device__ __forceinline__ void lora_down(float (&acc)[MT][NB][4], const uint16_t *const (&x)[MT][2], const uint16_t *A, int K, int rank, int r0,
                                          int first, int last, int step, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll 2
    for (int c = first; c < last; c += step) {
        const int k = 32 * c + 8 * t;
        uint4 xv[MT][2], av[NB];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i) xv[m][i] = ldg16(x[m][i] + k, x[m][i] != nullptr && k < K);
#pragma unroll
        for (int b = 0; b < NB; ++b) av[b] = ldg16(A + (long long)(r0 + 8 * b + g) * K + k, r0 + 8 * b + g < rank && k < K);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int b = 0; b < NB; ++b) mma_bf16_16816(acc[m][b], xv[m][0].x, xv[m][1].x, xv[m][0].y, xv[m][1].y, av[b].x, av[b].y);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int b = 0; b < NB; ++b) mma_bf16_16816(acc[m][b], xv[m][0].z, xv[m][1].z, xv[m][0].w, xv[m][1].w, av[b].z, av[b].w);
    }
}

// Two sums as pieces.  Of those at `left` and behind, which are ranks that an adapter has not, nothing is left: x may be infinite there and A 0.
__device__ __forceinline__ void lora_pieces(float x, float y, int left, uint32_t &hi, uint32_t &lo) {
    constexpr float MOST = 3.38953139e38f;  // bf16's largest
    if (left < 1) x = 0.f;
    if (left < 2) y = 0.f;
    hi = pack16x2<false>(fminf(fmaxf(x, -MOST), MOST), fminf(fmaxf(y, -MOST), MOST));
    lo = pack16x2<false>(x - bf16x2_lo(hi), y - bf16x2_hi(hi));
}
// The first `left` of eight columns of B, the others zero, whatever is stored there.
__device__ __forceinline__ uint4 lora_mask_rank(uint4 v, int left) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] &= left > 2 * i + 1 ? 0xffffffffu : left > 2 * i ? 0xffffu : 0u;
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 lora_b_piece(const uint16_t *B, int r, int rank, bool on) {
    const uint4 v = ldg16(B + r, on && r < rank);
    return rank & 7 ? lora_mask_rank(v, rank - r) : v;
}
// 32 columns of B as operands: column n of block b is column 8 (n / 2) + 2 b + n % 2, so that a lane's results are 8 neighbours.
template <int RC>
__device__ __forceinline__ void lora_load_b(uint4 (&bv)[4][RC], const LoraArgs &a, int ad, int rank, int n0, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int col = n0 + 8 * (g >> 1) + 2 * b + (g & 1);
#pragma unroll
        for (int c = 0; c < RC; ++c) bv[b][c] = lora_b_piece(a.B + ((long long)ad * a.N + col) * a.rank_max, 32 * c + 8 * t, rank, col < a.N);
    }
}
// Eight neighbours of a row of base (+ residual), in f32.
struct Base8 {
    float v[8];
};
__device__ __forceinline__ Base8 lora_base(const LoraArgs &a, long long at, bool on) {
    Base8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = 0.f;
    if (!on) return o;
    if (a.base_f32) {
        const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(a.base) + at);
        const float4 u = p[0], w = p[1];
        o.v[0] = u.x, o.v[1] = u.y, o.v[2] = u.z, o.v[3] = u.w, o.v[4] = w.x, o.v[5] = w.y, o.v[6] = w.z, o.v[7] = w.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(a.base) + at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) o.v[2 * i] = bf16x2_lo(w[i]), o.v[2 * i + 1] = bf16x2_hi(w[i]);
    }
    return o;
}
__device__ __forceinline__ void lora_store(const LoraArgs &a, long long at, const Base8 &base, const float (&up)[8]) {
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = base.v[i] + up[i];
    if (a.residual) {
        const uint4 u = *reinterpret_cast<const uint4 *>(a.residual + at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) s[2 * i] += bf16x2_lo(w[i]), s[2 * i + 1] += bf16x2_hi(w[i]);
    }
    *reinterpret_cast<uint4 *>(a.out + at) = make_uint4(pack16x2<false>(s[0], s[1]), pack16x2<false>(s[2], s[3]), pack16x2<false>(s[4], s[5]), pack16x2<false>(s[6], s[7]));
}

// =====================================================================================
// Up to LORA_FEW rows: one launch.  A cluster of eight CTAs takes a tile of 16 rows: each an eighth of K, its warps a share of
// that; the partial sums meet in distributed shared memory, and each CTA goes on with its share of the columns of B, whose
// first pieces are on their way before the sums meet.  Every CTA puts the rows in order for itself (a few hundred comparisons a
// thread), which is cheaper than a launch in front.  How many tiles there are only the device knows: as many clusters as run at
// once go through them, and where the tiles are few, several share a tile's columns and each forms x A^T for itself.
//
// Measured: 4 rows on adapters of rank 16, K = N = 2048, 5.5 us, most of it the launch and two passes of latency; 64 rows on 64 adapters of
// rank 16, K = N = 4096, 18 us; 64 on 64 of rank 64, K = N = 8192, 40 us (134 MB of adapters, 3.4 TB/s).
// LORA_FEW, one launch against three, K = N = 4096, in us: 128 rows on 8 adapters of rank 16 9.9 and 11.5, on 64 20.8 and 26.2; 256 rows on 8 adapters
// 14.6 and 12.5, on 64 27.9 and 27.0.
// =====================================================================================
constexpr int LORA_FEW = 128, LF_WARPS = 8, LF_CLUSTER = 8;

template <int RC>  // rank_max up to 32 RC
__global__ void __cluster_dims__(LF_CLUSTER, 1, 1) __launch_bounds__(LF_WARPS * 32, RC == 4 ? 1 : 2) lora_few_kernel(LoraArgs a) {
    constexpr int NB = 4 * RC, RP = 32 * RC, THREADS = LF_WARPS * 32;
    extern __shared__ __align__(16) float lf_smem[];
    float(*red)[16][RP + 4] = reinterpret_cast<float(*)[16][RP + 4]>(lf_smem);  // [WARPS / 2]
    __shared__ __align__(16) float part[16][RP + 4];
    __shared__ uint4 frag[RC][2][2][32];  // chunk, hi / lo, rows g / g + 8, lane
    __shared__ int key[LORA_FEW], start[LORA_FEW], rows[16], s_adapter;
    const cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int rank_in = blockIdx.x % LF_CLUSTER, n_clusters = gridDim.x / LF_CLUSTER;
    pdl_wait();
    pdl_launch_dependents();
    // ---- the tiles: the rows of one adapter, 16 at a time, adapters in order ----
    if (tid < a.T) key[tid] = lora_adapter(a, tid, blockIdx.x == 0);
    __syncthreads();
    int mine = -1, pos = 0, of = -1;  // of row tid: its adapter, its place among that one's rows, its tile
    if (tid < a.T) {
        mine = key[tid];
        for (int u = 0; u < tid; ++u) pos += key[u] == mine;
        start[tid] = pos % 16 == 0 ? mine : -1;
    }
    const int tiles = __syncthreads_count(tid < a.T && pos % 16 == 0);
    if (tid < a.T) {
        of = pos / 16;  // behind the tiles of smaller adapters
        for (int u = 0; u < a.T; ++u) of += start[u] >= 0 && start[u] < mine;
    }
    const int blocks = (a.N + 31) / 32;
    // Columns a warp would have with one cluster per tile, counted in blocks of 32: shared while clusters would idle.
    const int splits = max(1, min(n_clusters / tiles, blocks / (LF_CLUSTER * LF_WARPS)));
    bool reading = false;  // whether other CTAs may still read this one's sums
    for (int item = blockIdx.x / LF_CLUSTER; item < tiles * splits; item += n_clusters) {
        const int tile = item / splits, split = item % splits;
        __syncthreads();  // the last tile's readers are done
        if (tid < 16) rows[tid] = -1;
        __syncthreads();
        if (of == tile) {
            rows[pos % 16] = tid;
            if (pos % 16 == 0) s_adapter = mine;
        }
        __syncthreads();
        const int ad = s_adapter, rank = lora_rank(a, ad), r_lo = rows[g], r_hi = rows[g + 8];
        // ---- x A^T ----
        if (rank > 0) {
            const int chunks = (a.K + 31) / 32, c0 = chunks * rank_in / LF_CLUSTER, c1 = chunks * (rank_in + 1) / LF_CLUSTER;
            const uint16_t *x[1][2] = {{r_lo >= 0 ? a.x + r_lo * a.x_row : nullptr, r_hi >= 0 ? a.x + r_hi * a.x_row : nullptr}};
            float acc[1][NB][4] = {};
            lora_down<1, NB>(acc, x, a.A + (long long)ad * a.rank_max * a.K, a.K, rank, 0, c0 + warp, c1, LF_WARPS, lane);
#pragma unroll
            for (int half = 1; half >= 0; --half) {
                if (warp / (LF_WARPS / 2) == half)
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float &d = red[warp % (LF_WARPS / 2)][g + 8 * (e >> 1)][8 * b + 2 * t4 + (e & 1)];
                            d = half ? acc[0][b][e] : d + acc[0][b][e];
                        }
                __syncthreads();
            }
            if (reading) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            reading = true;
            for (int i = tid; i < 16 * RP; i += THREADS) {
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < LF_WARPS / 2; ++w) s += red[w][i / RP][i % RP];
                part[i / RP][i % RP] = s;
            }
        }
        // ---- this warp's first columns, before the sums meet ----
        const int stride = LF_CLUSTER * splits * LF_WARPS;
        int cb = (split * LF_CLUSTER + rank_in) * LF_WARPS + warp;
        uint4 bv[4][RC];
        Base8 base[2];
        auto fetch = [&]() {
            const int n0 = 32 * cb, col = n0 + 8 * t4;
            lora_load_b<RC>(bv, a, ad, cb < blocks ? rank : 0, n0, lane);
            base[0] = lora_base(a, (long long)r_lo * a.N + col, r_lo >= 0 && cb < blocks && col < a.N);
            base[1] = lora_base(a, (long long)r_hi * a.N + col, r_hi >= 0 && cb < blocks && col < a.N);
        };
        fetch();
        if (rank > 0) {
            cluster.sync();
            const float scale = a.scales[ad];
            for (int i = tid; i < 16 * RP / 2; i += THREADS) {
                const int row = i / (RP / 2), r = 2 * (i % (RP / 2));
                float2 s = make_float2(0.f, 0.f);
#pragma unroll
                for (int c = 0; c < LF_CLUSTER; ++c) {
                    const float2 v = *reinterpret_cast<const float2 *>(cluster.map_shared_rank(&part[row][r], c));
                    s.x += v.x, s.y += v.y;
                }
                s.x *= scale, s.y *= scale;
                uint32_t hi, lo;
                lora_pieces(s.x, s.y, rank - r, hi, lo);
                // element r of the row: chunk, the lane's eight, the word in it
                const int c = r / 32, l = (row % 8) * 4 + r % 32 / 8, w = r % 8 / 2;
                reinterpret_cast<uint32_t *>(&frag[c][0][row / 8][l])[w] = hi;
                reinterpret_cast<uint32_t *>(&frag[c][1][row / 8][l])[w] = lo;
            }
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // done with the other CTAs' sums
            __syncthreads();
        }
        while (cb < blocks) {
            float acc[4][4] = {};
            if (rank > 0) {
#pragma unroll
                for (int c = 0; c < RC; ++c)
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const uint4 u = frag[c][p][0][lane], v = frag[c][p][1][lane];
#pragma unroll
                        for (int b = 0; b < 4; ++b) mma_bf16_16816(acc[b], u.x, v.x, u.y, v.y, bv[b][c].x, bv[b][c].y);
#pragma unroll
                        for (int b = 0; b < 4; ++b) mma_bf16_16816(acc[b], u.z, v.z, u.w, v.w, bv[b][c].z, bv[b][c].w);
                    }
            }
            const int col = 32 * cb + 8 * t4;
            const Base8 b0 = base[0], b1 = base[1];
            cb += stride;
            fetch();
            if (col < a.N) {
                const float u[8] = {acc[0][0], acc[0][1], acc[1][0], acc[1][1], acc[2][0], acc[2][1], acc[3][0], acc[3][1]};
                const float v[8] = {acc[0][2], acc[0][3], acc[1][2], acc[1][3], acc[2][2], acc[2][3], acc[3][2], acc[3][3]};
                if (r_lo >= 0) lora_store(a, (long long)r_lo * a.N + col, b0, u);
                if (r_hi >= 0) lora_store(a, (long long)r_hi * a.N + col, b1, v);
            }
        }
    }
    if (reading) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// =====================================================================================
// Many rows, three launches: rows by adapter into tiles of 64; x A^T of a tile by a cluster of eight CTAs (an eighth of K each,
// the sums meeting in distributed shared memory); and the columns of B, 64 rows x 256 columns a CTA, which is where the bytes
// of base and out go by.
//
// Measured, 9 prompts of 3583 rows together, K 4096, N 14336, 7 adapters of rank 8 to 64: 79 us (3.1 TB/s; 37 us for the bytes alone).  The
// columns of B take most of it, 58 us alone, with DRAM at 38 %, the tensor pipe at 35 %, instructions in 40 % of the cycles, L1 at 68 %: of the
// 8.8 cycles that one of the 16 warps an SM has room for spends per instruction, it waits 2.9 for base, 2.0 for the instruction before, 1.0 for
// the tensor pipe.
// Base by asynchronous copies with 16 warps (102 us) and through shared memory in whole lines (89) were slower.
// =====================================================================================
constexpr int LM_ROWS = 64, LM_MT = LM_ROWS / 16, LG_THREADS = 1024, LD_WARPS = 8, LU_WARPS = 4;
constexpr int LORA_MAX_TILES = (LORA_MAX_ROWS + LM_ROWS - 1) / LM_ROWS + LORA_MAX_ADAPTERS + 1;

__global__ void __launch_bounds__(LG_THREADS) lora_group_kernel(LoraArgs a) {
    extern __shared__ int lora_smem[];
    int *count = lora_smem, *first = lora_smem + a.n + 1;  // [n + 1] each; adapter n: none
    int *place = reinterpret_cast<int *>(a.low);           // [T] a row's place among its adapter's (`low` is not in use yet)
    __shared__ int sums[LG_THREADS / 32][2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i <= a.n; i += LG_THREADS) count[i] = 0;
    pdl_wait();
    pdl_launch_dependents();
    __syncthreads();
    // (rows of one adapter are counted together: a prompt's rows would otherwise queue for one counter)
#pragma unroll 4
    for (int base = 0; base < a.T; base += LG_THREADS) {
        const int t = base + tid, ad = t < a.T ? lora_adapter(a, t, true) : -1;
        const unsigned same = __match_any_sync(0xffffffffu, ad);
        int at = 0;
        if (ad >= 0 && lane == __ffs(same) - 1) at = atomicAdd(&count[ad], __popc(same));
        at = __shfl_sync(0xffffffffu, at, __ffs(same) - 1) + __popc(same & ((1u << lane) - 1));
        if (ad >= 0) place[t] = at;
    }
    __syncthreads();
    const int per = (a.n + LG_THREADS) / LG_THREADS, a0 = min(tid * per, a.n + 1), a1 = min(a0 + per, a.n + 1);
    int r = 0, w = 0;  // rows and tiles
    for (int i = a0; i < a1; ++i) r += count[i], w += (count[i] + LM_ROWS - 1) / LM_ROWS;
    int ir = r, iw = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int ur = __shfl_up_sync(0xffffffffu, ir, d), uw = __shfl_up_sync(0xffffffffu, iw, d);
        if (lane >= d) ir += ur, iw += uw;
    }
    if (lane == 31) sums[warp][0] = ir, sums[warp][1] = iw;
    __syncthreads();
    int br = ir - r, bw = iw - w, all = 0;
    for (int i = 0; i < LG_THREADS / 32; ++i) {
        if (i < warp) br += sums[i][0], bw += sums[i][1];
        all += sums[i][1];
    }
    for (int i = a0; i < a1; ++i) {
        const int c = count[i], rank = c ? lora_rank(a, i) : 0;
        first[i] = br;
        for (int k = 0; k < c; k += LM_ROWS) a.tiles[bw++] = make_int4(i, br + k, min(LM_ROWS, c - k), rank);
        br += c;
    }
    if (tid == 0) *a.n_tiles = all;
    __syncthreads();
#pragma unroll 4
    for (int t = tid; t < a.T; t += LG_THREADS) a.order[first[lora_adapter(a, t, false)] + place[t]] = t;
}

// x A^T of a tile of 64 rows by a cluster of 1 to 8 CTAs, each with a share of K, which it runs through in stages of 128: x and A
// come in by 16-byte asynchronous copies, three stages deep, so that the memory has 64 KB per CTA to fetch whatever the warps
// do; a warp multiplies a quarter of a stage by half the ranks.  Rows in shared memory are 256 bytes with their two halves
// swapped in odd rows: a quarter warp's 16-byte reads then touch every bank once.
constexpr int LD_STAGE = 128, LD_STAGES = 3;
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

template <int NB>  // blocks of eight ranks a warp has; a CTA has twice that at a time
__global__ void __launch_bounds__(LD_WARPS * 32, 2) lora_down_kernel(LoraArgs a) {
    constexpr int RP = 16 * NB, THREADS = LD_WARPS * 32, PARTS = LD_WARPS / 2, ROWS = LM_ROWS + RP, BYTES = ROWS * 2 * LD_STAGE;
    extern __shared__ __align__(128) uint8_t ld_smem[];  // [STAGES][64 rows of x, RP of A][256]; then [PARTS][64][RP + 4] f32
    const cg::cluster_group cluster = cg::this_cluster();
    const int n_ctas = (int)cluster.num_blocks(), rank_in = (int)cluster.block_rank(), tile = blockIdx.x / n_ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3, half = warp & 1, part = warp >> 1;
    pdl_wait();
    pdl_launch_dependents();
    const int4 w = a.tiles[tile];  // (behind the last tile: not looked at)
    if (tile >= *a.n_tiles) return;  // (the whole cluster)
    const int rank = w.w, wide = (a.rank_max + 31) / 32 * 32;
    if (rank == 0) return;
    const float scale = a.scales[w.x];
    const int all = (a.K + LD_STAGE - 1) / LD_STAGE, s0 = all * rank_in / n_ctas, s1 = all * (rank_in + 1) / n_ctas;
    // a thread copies piece tid % 16 of rows tid / 16 + 16 i
    const int piece = tid & 15, r16 = tid >> 4, swapped = piece ^ ((r16 & 1) << 2);
    const uint16_t *src[ROWS / 16];
#pragma unroll
    for (int i = 0; i < LM_ROWS / 16; ++i) src[i] = r16 + 16 * i < w.z ? a.x + a.order[w.y + r16 + 16 * i] * a.x_row : nullptr;
    const uint32_t smem = smem_u32(ld_smem), dst = smem + r16 * 256 + swapped * 16;
    float *sums = reinterpret_cast<float *>(ld_smem);
    for (int r0 = 0; r0 < rank; r0 += RP) {
#pragma unroll
        for (int i = 0; i < RP / 16; ++i)
            src[LM_ROWS / 16 + i] = r0 + r16 + 16 * i < rank ? a.A + ((long long)w.x * a.rank_max + r0 + r16 + 16 * i) * a.K : nullptr;
        auto load = [&](int s) {
            const int k = s * LD_STAGE + 8 * piece;
            if (s < s1)
#pragma unroll
                for (int i = 0; i < ROWS / 16; ++i) {
                    const bool on = src[i] != nullptr && k < a.K;
                    cp_async16(dst + (s - s0) % LD_STAGES * BYTES + i * 16 * 256, on ? src[i] + k : a.A, on);
                }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (int s = 0; s < LD_STAGES - 1; ++s) load(s0 + s);
        float acc[LM_MT][NB][4] = {};
        for (int s = s0; s < s1; ++s) {
            asm volatile("cp.async.wait_group %0;" ::"n"(LD_STAGES - 2) : "memory");
            __syncthreads();
            load(s + LD_STAGES - 1);
            const uint32_t at = smem + (s - s0) % LD_STAGES * BYTES + g * 256 + ((4 * part + t4) ^ ((g & 1) << 2)) * 16;
            uint4 av[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) av[b] = lds128(at + (LM_ROWS + 8 * (NB * half + b)) * 256);
#pragma unroll
            for (int m = 0; m < LM_MT; ++m) {
                if (r0 + 8 * NB * half >= rank) break;  // (no ranks for this warp)
                const uint4 x0 = lds128(at + 16 * m * 256), x1 = lds128(at + (16 * m + 8) * 256);
#pragma unroll
                for (int b = 0; b < NB; ++b) mma_bf16_16816(acc[m][b], x0.x, x1.x, x0.y, x1.y, av[b].x, av[b].y);
#pragma unroll
                for (int b = 0; b < NB; ++b) mma_bf16_16816(acc[m][b], x0.z, x1.z, x0.w, x1.w, av[b].z, av[b].w);
            }
        }
        __syncthreads();  // (the copies still pending are empty groups)
        float *mine = sums + part * LM_ROWS * (RP + 4) + half * 8 * NB;
#pragma unroll
        for (int m = 0; m < LM_MT; ++m)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    *reinterpret_cast<float2 *>(mine + (16 * m + 8 * e + g) * (RP + 4) + 8 * b + 2 * t4) = make_float2(acc[m][b][2 * e], acc[m][b][2 * e + 1]);
        __syncthreads();
        for (int i = tid; i < LM_ROWS * RP / 4; i += THREADS) {
            float4 *p = reinterpret_cast<float4 *>(sums + (i / (RP / 4)) * (RP + 4)) + i % (RP / 4);
            float4 s = *p;
#pragma unroll
            for (int k = 1; k < PARTS; ++k) {
                const float4 v = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + k * LM_ROWS * (RP + 4));
                s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
            }
            *p = s;
        }
        cluster.sync();
        // 64 / n_ctas rows a CTA
        for (int i = tid; i < LM_ROWS / n_ctas * (RP / 4); i += THREADS) {
            const int row = LM_ROWS / n_ctas * rank_in + i / (RP / 4), r = 4 * (i % (RP / 4));
            if (row >= w.z || r0 + r >= wide) continue;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = 0; c < n_ctas; ++c) {
                const float4 v = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(sums + row * (RP + 4) + r, c));
                s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
            }
            s.x *= scale, s.y *= scale, s.z *= scale, s.w *= scale;
            uint2 hi, lo;
            lora_pieces(s.x, s.y, rank - r0 - r, hi.x, lo.x);
            lora_pieces(s.z, s.w, rank - r0 - r - 2, hi.y, lo.y);
            uint16_t *d = a.low + (long long)(w.y + row) * 2 * wide + r0 + r;
            *reinterpret_cast<uint2 *>(d) = hi;
            *reinterpret_cast<uint2 *>(d + wide) = lo;
        }
        cluster.sync();
    }
}

// A CTA has a tile's x A^T in shared memory, in the order of mma operands, and goes through `loops` times 32 columns per warp; the
// base of the next columns is on its way while these are multiplied, and the products are summed on top of it.  Lanes without
// a row or column of their own read some other one's and store nothing.
template <int RC, bool F32>
__global__ void __launch_bounds__(LU_WARPS * 32, RC == 4 ? 2 : F32 ? 3 : 4) lora_up_kernel(LoraArgs a, int loops) {
    extern __shared__ __align__(16) uint4 lu_frag[];  // [MT][RC][hi / lo][rows g / g + 8][32]
    __shared__ int rows[LM_ROWS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    pdl_wait();
    pdl_launch_dependents();
    const int4 w = a.tiles[blockIdx.y];
    if ((int)blockIdx.y >= *a.n_tiles) return;
    const int rank = w.w, wide = (a.rank_max + 31) / 32 * 32, used = (rank + 31) / 32;
    if (tid < LM_ROWS) rows[tid] = a.order[w.y + min(tid, w.z - 1)];
    for (int i = tid; i < LM_MT * RC * 128; i += LU_WARPS * 32) {
        const int l = i & 31, row = 16 * (i / (128 * RC)) + 8 * (i >> 5 & 1) + (l >> 2), r = 32 * (i / 128 % RC) + 8 * (l & 3);
        // (columns behind the rank need not have been written)
        lu_frag[i] = ldg16(a.low + ((long long)(w.y + row) * 2 + (i >> 6 & 1)) * wide + r, row < w.z && r < rank);
    }
    __syncthreads();
    int n0 = (blockIdx.x * loops * LU_WARPS + warp) * 32, col = min(n0 + 8 * t4, a.N - 8);
    long long at[LM_MT][2];  // the lane's rows
#pragma unroll
    for (int m = 0; m < LM_MT; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) at[m][i] = (long long)rows[16 * m + 8 * i + g] * a.N;
    const int parts = (w.z + 15) / 16;
    uint4 raw[LM_MT][2][F32 ? 2 : 1];
    auto fetch = [&](int m, int c) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int k = 0; k < (F32 ? 2 : 1); ++k)
                raw[m][i][k] = F32 ? reinterpret_cast<const uint4 *>(reinterpret_cast<const float *>(a.base) + at[m][i] + c)[k]
                                   : *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(a.base) + at[m][i] + c);
    };
#pragma unroll
    for (int m = 0; m < LM_MT; ++m)
        if (m < parts) fetch(m, col);
    for (int l = 0; l < loops && n0 < a.N; ++l) {
        uint4 bv[4][RC];
        lora_load_b<RC>(bv, a, w.x, rank, n0, lane);
        const bool here = n0 + 8 * t4 < a.N;
        const int this_col = col;
        n0 += 32 * LU_WARPS;
        const bool more = l + 1 < loops && n0 < a.N;
        if (more) col = min(n0 + 8 * t4, a.N - 8);
#pragma unroll
        for (int m = 0; m < LM_MT; ++m) {
            if (m >= parts) break;
            float acc[4][4];  // base, then the sums
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const uint4 u = raw[m][i][F32 ? b >> 1 : 0];
                    if (F32) {
                        acc[b][2 * i] = __uint_as_float(b & 1 ? u.z : u.x), acc[b][2 * i + 1] = __uint_as_float(b & 1 ? u.w : u.y);
                    } else {
                        const uint32_t e = b == 0 ? u.x : b == 1 ? u.y : b == 2 ? u.z : u.w;
                        acc[b][2 * i] = bf16x2_lo(e), acc[b][2 * i + 1] = bf16x2_hi(e);
                    }
                }
            if (more) fetch(m, col);
#pragma unroll
            for (int c = 0; c < RC; ++c) {
                if (c >= used) break;
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const uint4 u = lu_frag[((m * RC + c) * 2 + p) * 64 + lane], v = lu_frag[((m * RC + c) * 2 + p) * 64 + 32 + lane];
#pragma unroll
                    for (int b = 0; b < 4; ++b) mma_bf16_16816(acc[b], u.x, v.x, u.y, v.y, bv[b][c].x, bv[b][c].y);
#pragma unroll
                    for (int b = 0; b < 4; ++b) mma_bf16_16816(acc[b], u.z, v.z, u.w, v.w, bv[b][c].z, bv[b][c].w);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (!here || 16 * m + 8 * i + g >= w.z) continue;
                const long long o = at[m][i] + this_col;
                if (a.residual) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(a.residual + o);
                    const uint32_t e[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int b = 0; b < 4; ++b) acc[b][2 * i] += bf16x2_lo(e[b]), acc[b][2 * i + 1] += bf16x2_hi(e[b]);
                }
                *reinterpret_cast<uint4 *>(a.out + o) = make_uint4(pack16x2<false>(acc[0][2 * i], acc[0][2 * i + 1]), pack16x2<false>(acc[1][2 * i], acc[1][2 * i + 1]),
                                                                   pack16x2<false>(acc[2][2 * i], acc[2][2 * i + 1]), pack16x2<false>(acc[3][2 * i], acc[3][2 * i + 1]));
            }
        }
    }
}

size_t lora_scratch_bytes() {
    return 256 + (size_t)LORA_MAX_TILES * 16 + ((size_t)LORA_MAX_ROWS + 1) * 4 + ((size_t)LORA_MAX_ROWS + 1) * LORA_MAX_RANK * 4;
}

template <int NB>
static int launch_lora_down(const LoraArgs &a, int tiles, cudaStream_t stream) {
    constexpr int stages = LD_STAGES * (LM_ROWS + 16 * NB) * 2 * LD_STAGE, sums = LD_WARPS / 2 * LM_ROWS * (16 * NB + 4) * 4, smem = stages > sums ? stages : sums;
    int rc = check_cuda(cudaFuncSetAttribute(lora_down_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "lora shared memory");
    if (rc) return rc;
    // as many shares of K as let every CTA be resident at once
    const int busy = (a.T + LM_ROWS - 1) / LM_ROWS, most = 2 * device_sm_count();
    const int n_ctas = busy * 8 <= most ? 8 : busy * 4 <= most ? 4 : busy * 2 <= most ? 2 : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * n_ctas);
    cfg.blockDim = dim3(LD_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)n_ctas, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return check_cuda(cudaLaunchKernelEx(&cfg, lora_down_kernel<NB>, a), "lora down launch");
}
template <int RC>
static int launch_lora_up(const LoraArgs &a, int tiles, cudaStream_t stream) {
    // as many columns a CTA as leave about two CTAs to each of the four places on an SM (nine prompts, K 4096, N 14336: 79 us;
    // four 84, one 82)
    const int blocks = (a.N + 32 * LU_WARPS - 1) / (32 * LU_WARPS), busy = (a.T + LM_ROWS - 1) / LM_ROWS;
    const int loops = max(1, min(16, (int)((long long)blocks * busy / (7 * device_sm_count()))));
    const dim3 grid((blocks + loops - 1) / loops, tiles), block(LU_WARPS * 32);
    const int smem = LM_MT * RC * 128 * 16;
    auto kernel = a.base_f32 ? lora_up_kernel<RC, true> : lora_up_kernel<RC, false>;
    return check_cuda(launch_pdl(kernel, grid, block, smem, stream, a, loops), "lora up launch");
}

static int launch_lora(LoraArgs a, cudaStream_t stream) {
    const int rc32 = (a.rank_max + 31) / 32;
    if (a.T <= LORA_FEW) {
        // as many clusters as find room at once (two CTAs an SM), or as there may be tiles and shares of their columns
        const int shares = max(1, (a.N + 31) / 32 / (LF_CLUSTER * LF_WARPS)), tiles = min(a.T, (a.T + 15) / 16 + a.n + 1);
        const dim3 grid(LF_CLUSTER * min(2 * device_sm_count() / LF_CLUSTER, shares * tiles)), block(LF_WARPS * 32);
        auto kernel = rc32 == 1 ? lora_few_kernel<1> : rc32 == 2 ? lora_few_kernel<2> : lora_few_kernel<4>;
        const int smem = LF_WARPS / 2 * 16 * ((rc32 == 3 ? 4 : rc32) * 32 + 4) * 4;
        int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "lora shared memory");
        if (rc) return rc;
        return check_cuda(launch_pdl(kernel, grid, block, smem, stream, a), "lora launch");
    }
    const int tiles = min(a.T, (a.T + LM_ROWS - 1) / LM_ROWS + a.n + 1);
    const int smem = 2 * (a.n + 1) * 4;
    int rc = check_cuda(launch_pdl(lora_group_kernel, dim3(1), dim3(LG_THREADS), smem, stream, a), "lora group launch");
    if (rc) return rc;
    if (a.n > 0) {
        rc = a.rank_max <= 16 ? launch_lora_down<1>(a, tiles, stream) : a.rank_max <= 32 ? launch_lora_down<2>(a, tiles, stream) : launch_lora_down<4>(a, tiles, stream);
        if (rc) return rc;
    }
    return rc32 == 1 ? launch_lora_up<1>(a, tiles, stream) : rc32 == 2 ? launch_lora_up<2>(a, tiles, stream) : launch_lora_up<4>(a, tiles, stream);
}

}  // namespace awq

using namespace awq;

extern "C" int awq_b200_lora_bf16(const uint16_t *x, long long x_row_stride, const uint16_t *A, const uint16_t *B, const float *scales,
                                  const int32_t *ranks, int n_adapters, int rank_max, const int32_t *idx, const void *base, int base_is_f32,
                                  const uint16_t *residual, uint16_t *out, int T, int K, int N, void *workspace, size_t workspace_bytes,
                                  awq_stream_t stream) {
    AWQ_REQUIRE(T >= 0 && T <= LORA_MAX_ROWS && K > 0 && N >= 0 && n_adapters >= 0 && n_adapters <= LORA_MAX_ADAPTERS,
                "lora: bad size (at most %d rows and %d adapters)", LORA_MAX_ROWS, LORA_MAX_ADAPTERS);
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
    // CTAs read all of x, A and B, and each the base and residual of the elements that it writes.
    auto apart = [&](const void *p, long long elements, int size) {
        const uintptr_t from = reinterpret_cast<uintptr_t>(p), to = reinterpret_cast<uintptr_t>(out);
        return !p || from + (uintptr_t)elements * size <= to || to + 2 * (uintptr_t)T * N <= from;
    };
    const long long whole = (long long)T * N;
    AWQ_REQUIRE(apart(x, (T - 1) * x_row_stride + K, 2) && apart(A, (long long)n_adapters * rank_max * K, 2) && apart(B, (long long)n_adapters * rank_max * N, 2),
                "lora: out must not overlap x or the adapters");
    AWQ_REQUIRE((!base_is_f32 && base == out) || apart(base, whole, base_is_f32 ? 4 : 2), "lora: out may be a bf16 base, but not overlap base otherwise");
    AWQ_REQUIRE(residual == out || apart(residual, whole, 2), "lora: out may be the residual, but not overlap it otherwise");
    const RequestWorkspaceView w = request_workspace(workspace);
    LoraArgs a{};
    a.x = x, a.A = A, a.B = B, a.scales = scales, a.ranks = ranks, a.idx = idx, a.base = base, a.residual = residual, a.out = out;
    a.x_row = x_row_stride, a.base_f32 = base_is_f32, a.T = T, a.K = K, a.N = N, a.n = n_adapters, a.rank_max = rank_max;
    a.header = w.header;
    uint8_t *p = w.lora;
    a.n_tiles = reinterpret_cast<int32_t *>(p), p += 256;
    a.tiles = reinterpret_cast<int4 *>(p), p += (size_t)LORA_MAX_TILES * 16;
    a.order = reinterpret_cast<int32_t *>(p), p += ((size_t)LORA_MAX_ROWS + 1) * 4;
    a.low = reinterpret_cast<uint16_t *>(p);
    return launch_lora(a, as_stream(stream));
}
