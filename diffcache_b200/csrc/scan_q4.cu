// Score scan over keys held in 4 bits: the ranking keys of score_scan (scan.cu; nsw.rs:601-607 with QKDist,
// nsw.rs:129-139) for stored keys s * c,  dist = 65536 - sum_g s_g * sum_{d in g} q_d c_d,  in fp32.
//
// 16 rows at a time go through m16n8k16 tensor-core products: the codes, as fp16 subnormals, are A; column j of B is the
// query with every group but group j set to zero, so that ONE chain of head_dim / 16 products leaves the partial dot of
// group j in column j, exact up to fp32 accumulation, and the scales are applied once per group in fp32.  The query is
// normalised by a power of two, so that a bf16 query is exact in fp16 as well.  The codes come straight from global
// memory to the fragment registers (the stored order makes a lane's share of a row contiguous), 64 rows per warp at a time.
// Bound: HBM, 9/16 * head_dim bytes a row and 4 of output.  128 problems x 130496 rows of head_dim 128: 208 us = 6.1 TB/s (one
// thread per row on the FMA pipe: 630 us; without the second register set 429; with 1024-row CTAs and the query first 325;
// with the codes converted to integers before the products 225).
#include <algorithm>

#include "q4_mma.cuh"

namespace dc {
namespace {

constexpr int kScanThreads = 256;
constexpr int kScanWarps = kScanThreads / 32;
constexpr int kCtasPerSm = 2;
// 16-row tiles a warp loads at a time: 4, or 2 where a row is 128 bytes of codes and registers would not hold two sets of 4
__host__ __device__ constexpr int scan_tiles(int head_dim) { return head_dim <= 128 ? 4 : 2; }
__host__ __device__ constexpr int scan_pass_rows(int head_dim) { return kScanWarps * 16 * scan_tiles(head_dim); }

// grid = (chunks of rows_per_cta rows, n_prob)
template <int DT, int D>
__global__ void __launch_bounds__(kScanThreads, kCtasPerSm)
q4_scan_kernel(const Q4Rows keys, int64_t prob_rows, int64_t n, const int32_t* __restrict__ n_dev,
               const uint16_t* __restrict__ q, int q_mode, int group, int kv_heads, int64_t q_stride_b,
               uint32_t* __restrict__ scores, int64_t score_stride, uint32_t* __restrict__ minmax, int rows_per_cta) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int NG = D / kQ4Group, W = D / 64;
    constexpr int kTiles = scan_tiles(D), kWarpRows = 16 * kTiles, kPassRows = scan_pass_rows(D);
    __shared__ float s_q[D];
    __shared__ float s_top;
    __shared__ uint32_t s_lo, s_hi;
    // rows valid now (the grid was sized for an upper bound, which is also all the output holds)
    const int64_t n_now = n_dev != nullptr ? min(n, static_cast<int64_t>(*n_dev)) : n;
    const int64_t prob = blockIdx.y;
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * rows_per_cta;
    if (begin >= n_now) return;
    const int64_t end = min(n_now, begin + rows_per_cta);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;

    const uint8_t* codes = keys.codes + prob * prob_rows * (D / 2) + t * (D / 8);
    const uint16_t* scales = keys.scales + prob * prob_rows * NG + 2 * t;
    struct Rows { uint32_t k[kTiles][2][D / 32], sc[kTiles][2]; };
    auto load = [&](Rows& x, int64_t base) {
        if (base + kWarpRows <= end) {         // one address, everything else is a constant away
            const uint8_t* kp = codes + (base + g) * (D / 2);
            const uint16_t* sp = scales + (base + g) * NG;
#pragma unroll
            for (int i = 0; i < kTiles; i++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    ldg_words<D / 32>(x.k[i][r], kp + (16 * i + 8 * r) * (D / 2));
                    x.sc[i][r] = 2 * t < NG ? __ldcs(reinterpret_cast<const uint32_t*>(sp + (16 * i + 8 * r) * NG)) : 0u;
                }
        } else {
#pragma unroll
            for (int i = 0; i < kTiles; i++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const int64_t row = min(base + 16 * i + 8 * r + g, end - 1);   // rows beyond the end repeat the last one
                    ldg_words<D / 32>(x.k[i][r], codes + row * (D / 2));
                    x.sc[i][r] = 2 * t < NG ? *reinterpret_cast<const uint32_t*>(scales + row * NG) : 0u;
                }
        }
    };
    // the first rows are on their way while the query is prepared
    int64_t base = begin + warp * kWarpRows;
    Rows x, y;
    if (base < end) load(x, base);

    if (threadIdx.x == 0) { s_lo = 0xFFFFFFFFu; s_hi = 0u; }
    if (threadIdx.x < 32) {
        float top = 0.0f;
        for (int c = threadIdx.x; c < D / 8; c += 32) {
            float f[8];
            load_query8<DT>(query_base(q, prob, D, q_mode, group, kv_heads, q_stride_b), D, q_mode, group, c * 8, f);
#pragma unroll
            for (int j = 0; j < 8; j++) { s_q[c * 8 + j] = f[j]; top = fmaxf(top, fabsf(f[j])); }
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
        if (threadIdx.x == 0) s_top = top;
    }
    __syncthreads();
    float down, up;
    q4_normalise(s_top, down, up);

    // query fragments: column g of B holds group g, i.e. only the products with that group's codes are not zero
    uint32_t qb[D / 16][2];
    float q_sum = 0.0f;                        // of column g, over this lane's rows of B
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int d = 32 * (g % NG) + 2 * (2 * t + c) + e;   // + 16: the group's other tile
            const float f = e ? down * 0.0625f : down;
            const uint32_t v = pack2<false>(s_q[d] * f, s_q[d + 16] * f);
            const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&v));
            q_sum += (r.x + r.y) * (e ? 16.0f : 1.0f);
#pragma unroll
            for (int i = 0; i < NG; i++) qb[2 * i + c][e] = g == i ? v : 0u;
        }
    q_sum += __shfl_xor_sync(0xFFFFFFFFu, q_sum, 1);
    q_sum += __shfl_xor_sync(0xFFFFFFFFu, q_sum, 2);
    // the sums start from - 8 * 2^-24 times their column's query sum (columns 2t, 2t + 1 of this lane)
    const float start0 = -0x1p-21f * __shfl_sync(0xFFFFFFFFu, q_sum, 8 * t), start1 = -0x1p-21f * __shfl_sync(0xFFFFFFFFu, q_sum, 8 * t + 4);
    const float start[4] = {2 * t < NG ? start0 : 0.0f, 2 * t < NG ? start1 : 0.0f, 2 * t < NG ? start0 : 0.0f, 2 * t < NG ? start1 : 0.0f};

    uint32_t* out = scores + prob * score_stride;
    uint32_t lo = 0xFFFFFFFFu, hi = 0u;
    auto compute = [&](const Rows& x, int64_t base) {
        float mine[2] = {0.0f, 0.0f};          // of tile t: rows g and g + 8
#pragma unroll
        for (int i = 0; i < kTiles; i++) {
            float acc[4];
#pragma unroll
            for (int w = 0; w < W; w++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t p[4], r[4];
                    codes_subnormal(x.k[i][0][c * W + w], p);
                    codes_subnormal(x.k[i][1][c * W + w], r);
                    if (w == 0 && c == 0) mma_from(acc, start, p[0], r[0], p[1], r[1], qb[0][0], qb[0][1]);
                    else mma<false>(acc, p[0], r[0], p[1], r[1], qb[4 * w + c][0], qb[4 * w + c][1]);
                    mma<false>(acc, p[2], r[2], p[3], r[3], qb[4 * w + 2 + c][0], qb[4 * w + 2 + c][1]);
                }
#pragma unroll
            for (int r = 0; r < 2; r++) {      // columns 2t, 2t + 1 are groups (zeros beyond the last); the t lanes of a row add up
                float dot = fmaf(low_elem<DT>(x.sc[i][r]), acc[2 * r], high_elem<DT>(x.sc[i][r]) * acc[2 * r + 1]);
                if (NG > 2) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, 1);
                if (NG > 4) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, 2);
                // the sum is complete in lane t = 0 (NG 2), t = 0, 1 (NG 4) or all of them; lane t takes tile t
                if (NG <= 4) dot = __shfl_sync(0xFFFFFFFFu, dot, lane & ~3);
                if (t == i) mine[r] = dot;
            }
        }
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int64_t row = base + 16 * t + 8 * r + g;
            if (t < kTiles && row < end) {
                const uint32_t b = dist_bits(mine[r] * up * 0x1p24f);   // up * 2^24 may overflow
                out[row] = b;
                lo = min(lo, b);
                hi = max(hi, b);
            }
        }
    };
    if (base < end) {                          // one load ahead, in two sets of registers
        while (true) {
            int64_t next = base + kPassRows;
            if (next < end) load(y, next);
            compute(x, base);
            if (next >= end) break;
            base = next;
            next += kPassRows;
            if (next < end) load(x, next);
            compute(y, base);
            if (next >= end) break;
            base = next;
        }
    }
    if (minmax != nullptr) {
        lo = __reduce_min_sync(0xFFFFFFFFu, lo);
        hi = __reduce_max_sync(0xFFFFFFFFu, hi);
        if (lane == 0) { atomicMin(&s_lo, lo); atomicMax(&s_hi, hi); }
        __syncthreads();
        if (threadIdx.x == 0 && s_lo <= s_hi) { atomicMin(&minmax[2 * prob], s_lo); atomicMax(&minmax[2 * prob + 1], s_hi); }
    }
}

// Rows per CTA.  A CTA costs about as much as 600 rows before it streams (the query), so CTAs are long; the length is chosen
// so that the launch fills whole waves of the CTAs that fit.
int rows_per_cta(int64_t n, int n_prob, int unit) {
    const int64_t slots = static_cast<int64_t>(kCtasPerSm) * sm_count();
    int64_t best = unit, best_cost = INT64_MAX;
    for (int64_t rows = unit; rows <= 32 * static_cast<int64_t>(unit); rows += unit) {
        const int64_t ctas = (n + rows - 1) / rows * n_prob;
        const int64_t cost = (ctas + slots - 1) / slots * (std::min(rows, n) + 600);
        if (cost < best_cost) { best = rows; best_cost = cost; }
        if (rows >= n) break;
    }
    return static_cast<int>(best);
}

}  // namespace

int q4_score_scan(const Q4Rows& keys, int64_t prob_rows, int n_prob, int64_t n, int head_dim, int dtype, const void* q,
                  int q_mode, int group, uint32_t* scores, int64_t score_stride, uint32_t* minmax, cudaStream_t stream,
                  int kv_heads, int64_t q_stride_b, const int32_t* n_dev) {
    if (n_prob == 0 || n == 0) return DC_OK;
    const int rows = rows_per_cta(n, n_prob, scan_pass_rows(head_dim));
    const dim3 grid(static_cast<unsigned>((n + rows - 1) / rows), static_cast<unsigned>(n_prob));
#define CASE(DT, D)                                                                                                       \
    DC_CUDA_TRY(launch_chained(q4_scan_kernel<DT, D>, grid, dim3(kScanThreads), 0, stream, 0u, keys, prob_rows, n, n_dev, \
                               static_cast<const uint16_t*>(q), q_mode, group, kv_heads, q_stride_b, scores, score_stride, \
                               minmax, rows))
    if (dtype == DC_BF16) {
        if (head_dim == 64) CASE(DC_BF16, 64);
        else if (head_dim == 128) CASE(DC_BF16, 128);
        else CASE(DC_BF16, 256);
    } else {
        if (head_dim == 64) CASE(DC_FP16, 64);
        else if (head_dim == 128) CASE(DC_FP16, 128);
        else CASE(DC_FP16, 256);
    }
#undef CASE
    return DC_OK;
}

}  // namespace dc
