// Score scan over keys held in 4 bits: the ranking keys of score_scan (scan.cu; nsw.rs:601-607 with QKDist,
// nsw.rs:129-139) for stored keys s * c,  dist = 65536 - sum_g s_g * sum_{d in g} q_d c_d,  in fp32.
#include "q4.cuh"

namespace dc {
namespace {

constexpr int kScanThreads = 256;

// one thread per row
template <int DT, int D>
__global__ void __launch_bounds__(kScanThreads)
q4_scan_kernel(const Q4Rows keys, int64_t prob_rows, int64_t n, const int32_t* __restrict__ n_dev,
               const uint16_t* __restrict__ q, int q_mode, int group, int kv_heads, int64_t q_stride_b,
               uint32_t* __restrict__ scores, int64_t score_stride, uint32_t* __restrict__ minmax) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float s_q[D];
    __shared__ uint32_t s_lo, s_hi;
    const int64_t n_now = n_dev != nullptr ? min(n, static_cast<int64_t>(*n_dev)) : n;
    const int64_t prob = blockIdx.y;
    if (threadIdx.x == 0) { s_lo = 0xFFFFFFFFu; s_hi = 0u; }
    if (threadIdx.x < D / 8) {
        float f[8];
        load_query8<DT>(query_base(q, prob, D, q_mode, group, kv_heads, q_stride_b), D, q_mode, group, threadIdx.x * 8, f);
        for (int j = 0; j < 8; j++) s_q[threadIdx.x * 8 + j] = f[j];
    }
    __syncthreads();
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kScanThreads + threadIdx.x;
    uint32_t lo = 0xFFFFFFFFu, hi = 0u;
    if (i < n_now) {
        const int64_t row = prob * prob_rows + i;
        const uint32_t* cw = reinterpret_cast<const uint32_t*>(keys.codes + row * (D / 2));
        float acc[D / kQ4Group];
        for (int g = 0; g < D / kQ4Group; g++) acc[g] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int w = 0; w < D / 64; w++) {
                const uint32_t word = cw[j * (D / 64) + w];
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const int tile = 4 * w + (b == 1 ? 2 : b == 2 ? 1 : b);
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        acc[tile / 2] = fmaf(s_q[16 * tile + 2 * j + e],
                                             static_cast<float>(static_cast<int>((word >> (8 * b + 4 * e)) & 15u) - 8), acc[tile / 2]);
                }
            }
        float dot = 0.0f;
        for (int g = 0; g < D / kQ4Group; g++) dot = fmaf(elem_to_float<DT>(keys.scales[row * (D / kQ4Group) + g]), acc[g], dot);
        lo = hi = dist_bits(dot);
        scores[prob * score_stride + i] = lo;
    }
    if (minmax != nullptr) {
        lo = __reduce_min_sync(0xFFFFFFFFu, lo);
        hi = __reduce_max_sync(0xFFFFFFFFu, hi);
        if ((threadIdx.x & 31) == 0) { atomicMin(&s_lo, lo); atomicMax(&s_hi, hi); }
        __syncthreads();
        if (threadIdx.x == 0 && s_lo <= s_hi) { atomicMin(&minmax[2 * prob], s_lo); atomicMax(&minmax[2 * prob + 1], s_hi); }
    }
}

}  // namespace

int q4_score_scan(const Q4Rows& keys, int64_t prob_rows, int n_prob, int64_t n, int head_dim, int dtype, const void* q,
                  int q_mode, int group, uint32_t* scores, int64_t score_stride, uint32_t* minmax, cudaStream_t stream,
                  int kv_heads, int64_t q_stride_b, const int32_t* n_dev) {
    if (n_prob == 0 || n == 0) return DC_OK;
    const dim3 grid(static_cast<unsigned>((n + kScanThreads - 1) / kScanThreads), static_cast<unsigned>(n_prob));
#define CASE(DT, D)                                                                                                       \
    DC_CUDA_TRY(launch_chained(q4_scan_kernel<DT, D>, grid, dim3(kScanThreads), 0, stream, 0u, keys, prob_rows, n, n_dev, \
                               static_cast<const uint16_t*>(q), q_mode, group, kv_heads, q_stride_b, scores, score_stride, minmax))
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
