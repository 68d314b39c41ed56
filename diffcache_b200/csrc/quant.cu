// Rows into and out of a store held in 4 bits (format: q4.cuh).
//
// Counterpart of copy_rows / append / gather on the 16-bit store: DataLayer::prefill and insert
// (diffcache_cpu/src/lib.rs:329-369, nsw.rs:497-557) and the row gather of search_bruteforce (nsw.rs:621-629),
// which the reference does with plain copies.
//
// A thread holds one tile, 16 consecutive elements (32 bytes): the group maximum is one shuffle away, the codes move to their
// stored order with four more, and a row leaves as runs of 32 bytes.  Bound: HBM (2 * head_dim bytes in, 9/16 * head_dim out per row, or the other way round).
#include "q4.cuh"

namespace dc {
namespace {

constexpr int kRowThreads = 256;
// Rows a thread of the write kernel loads before it works on the first.  4 x 8 x 130496 rows of head_dim 128, keys and values:
// 522 us with one, 445 with two (6.16 TB/s), 443 with four; a single token 2.5, 2.8, 3.3 us.  Reading back does best with
// one row per thread (448 us, 6.12 TB/s; 452 with two, 524 with four).
constexpr int kWriteRows = 2;

struct WriteArgs {
    const uint16_t* keys;
    const uint16_t* vals;
    int64_t stride_b, stride_h, stride_s;
    int kv_heads;
    int64_t n, row0;
    Q4Store st;
    int32_t* len;
    int len_mode;
};

// (field by field: a reference into the kernel's parameters would copy them to local memory)
__device__ __forceinline__ Q4Rows pick(const Q4Store& st, int values) {
    return {values ? st.v.codes : st.k.codes, values ? st.v.scales : st.k.scales};
}

__device__ __forceinline__ void load_tile(const uint16_t* p, uint4 (&w)[2]) {   // 16-byte aligned
    w[0] = ld_stream16(p);
    w[1] = ld_stream16(p + 8);
}

template <int D>
__device__ __forceinline__ void q4_put(const Q4Rows& t, int64_t row, int v, const uint32_t (&word)[2], uint16_t scale) {
    uint32_t* c = reinterpret_cast<uint32_t*>(t.codes + row * (D / 2));
    c[q4_word_index<D>(v, 0)] = word[0];
    c[q4_word_index<D>(v, 1)] = word[1];
    if ((v & 1) == 0) t.scales[row * (D / kQ4Group) + (v >> 1)] = scale;
}

// grid = (row blocks, n_prob, 2 tensors)
template <int DT, int D>
__global__ void __launch_bounds__(kRowThreads)
q4_write_kernel(const WriteArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int LPR = D / 16, RPB = kRowThreads / LPR;
    const int64_t prob = blockIdx.y;
    const int v = threadIdx.x % LPR;
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * (RPB * kWriteRows) + threadIdx.x / LPR;
    const int64_t b = prob / a.kv_heads, h = prob % a.kv_heads;
    const uint16_t* src = (blockIdx.z ? a.vals : a.keys) + b * a.stride_b + h * a.stride_h + v * 16;
    uint4 w[kWriteRows][2];
#pragma unroll
    for (int r = 0; r < kWriteRows; r++) {
        const int64_t i = i0 + r * RPB;
        w[r][0] = w[r][1] = make_uint4(0, 0, 0, 0);
        if (i < a.n) load_tile(src + i * a.stride_s, w[r]);
    }
    const Q4Rows dst = pick(a.st, blockIdx.z);
#pragma unroll
    for (int r = 0; r < kWriteRows; r++) {
        const int64_t i = i0 + r * RPB;
        uint32_t word[2];
        uint16_t scale;
        q4_encode<DT>(w[r], v, word, scale);
        if (i < a.n) q4_put<D>(dst, prob * a.st.prob_rows + a.row0 + i, v, word, scale);
    }
    if (a.len_mode != kLenKeep && blockIdx.x == 0 && prob == 0 && blockIdx.z == 0 && threadIdx.x == 0) {
        const int32_t end = static_cast<int32_t>(a.row0 + a.n);
        a.len[0] = a.len_mode == kLenSet ? end : max(a.len[0], end);
    }
}

// Index::insert (diffcache_cpu/src/nsw.rs:544-557): row len[0] of every problem <- keys / vals (n_prob, D), then
// len[0] += 1.  One CTA, so that every thread sees the old length.
template <int DT, int D>
__global__ void __launch_bounds__(1024)
q4_append_kernel(const uint16_t* __restrict__ keys, const uint16_t* __restrict__ vals, int n_prob, const Q4Store st,
                 int64_t max_rows, int32_t* len, uint32_t* status) {
    constexpr int LPR = D / 16;
    const int64_t n = len[0];
    if (n >= max_rows) {   // full: nothing is written (the host-side call reports it when it can tell)
        if (threadIdx.x == 0 && status) atomicMax(status, 301u);
        return;
    }
    const int total = n_prob * 2 * LPR;
    for (int i0 = 0; i0 < total; i0 += blockDim.x) {   // all lanes of a warp stay in the loop: the encoder shuffles
        const int i = i0 + threadIdx.x;
        const bool ok = i < total;
        const int p = i / (2 * LPR), which = (i / LPR) & 1, v = i % LPR;
        uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (ok) load_tile((which ? vals : keys) + static_cast<int64_t>(p) * D + v * 16, w);
        uint32_t word[2];
        uint16_t scale;
        q4_encode<DT>(w, v, word, scale);
        if (ok) q4_put<D>(pick(st, which), p * st.prob_rows + n, v, word, scale);
    }
    __syncthreads();
    if (threadIdx.x == 0) len[0] = static_cast<int32_t>(n + 1);
}

// The window ring of the resident buffer (see window_push_kernel in engine.cu: same state words, same statuses) with the
// spilled token quantised on its way into the store.
template <int DT, int D>
__global__ void __launch_bounds__(1024)
q4_window_push_kernel(const uint16_t* __restrict__ k_new, const uint16_t* __restrict__ v_new, int64_t new_stride_b,
                      uint16_t* __restrict__ res_k, uint16_t* __restrict__ res_v, int64_t res_stride_b,
                      int64_t res_stride_h, int n_prob, int kv_heads, const Q4Store st, int64_t max_rows, int32_t* len,
                      int32_t* win, uint32_t* status) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int LPR = D / 16;
    const int suffix_len = win[0], head = win[1], prefix_len = win[2], cap = win[3];
    const int64_t n = len[0];
    const bool full = suffix_len >= cap;
    const bool spill = full && n < max_rows;
    const int slot = full ? head : suffix_len;
    if (full && !spill && threadIdx.x == 0 && status) atomicMax(status, 302u);  // store full: the oldest token is dropped
    const int total = n_prob * 2 * LPR;
    for (int i0 = 0; i0 < total; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        const bool ok = i < total;
        const int p = i / (2 * LPR), which = (i / LPR) & 1, v = i % LPR;
        const int b = p / kv_heads, h = p % kv_heads;
        uint16_t* row = (which ? res_v : res_k) + b * res_stride_b + h * res_stride_h +
                        static_cast<int64_t>(prefix_len + slot) * D + v * 16;
        if (spill) {
            uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
            if (ok) {
                w[0] = reinterpret_cast<const uint4*>(row)[0];
                w[1] = reinterpret_cast<const uint4*>(row)[1];
            }
            uint32_t word[2];
            uint16_t scale;
            q4_encode<DT>(w, v, word, scale);
            if (ok) q4_put<D>(pick(st, which), p * st.prob_rows + n, v, word, scale);
        }
        const int64_t off = new_stride_b ? b * new_stride_b + static_cast<int64_t>(h) * D : static_cast<int64_t>(p) * D;
        if (ok) {
            const uint4* fresh = reinterpret_cast<const uint4*>((which ? v_new : k_new) + off + v * 16);
            reinterpret_cast<uint4*>(row)[0] = fresh[0];
            reinterpret_cast<uint4*>(row)[1] = fresh[1];
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        if (spill) len[0] = static_cast<int32_t>(n + 1);
        win[4] = prefix_len + min(suffix_len + 1, cap);
    }
}

struct ReadArgs {
    Q4Store st;
    int64_t n_rows;
    const int32_t* n_dev;
    const uint32_t* ids;        // (n_prob, ids_stride) or NULL: rows row0, row0 + 1, ...
    int64_t ids_stride, row0, n;
    void* out_k;                // either may be NULL
    void* out_v;
};

// grid = (row blocks, n_prob, outputs)
template <int DT, int D, bool F32>
__global__ void __launch_bounds__(kRowThreads)
q4_read_kernel(const ReadArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int LPR = D / 16, RPB = kRowThreads / LPR;
    const int64_t prob = blockIdx.y;
    const int v = threadIdx.x % LPR;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / LPR;
    const int which = a.out_k == nullptr ? 1 : blockIdx.z;
    void* out = which ? a.out_v : a.out_k;
    const int64_t n_rows = a.n_dev != nullptr ? static_cast<int64_t>(*a.n_dev) : a.n_rows;
    const Q4Rows t = pick(a.st, which);
    uint32_t word[2] = {0x88888888u, 0x88888888u};
    uint16_t scale = 0;
    if (i < a.n) {
        const int64_t row = a.ids != nullptr ? static_cast<int64_t>(a.ids[prob * a.ids_stride + i]) : a.row0 + i;
        if (row < n_rows) {   // a pad (0xFFFFFFFF) or any id beyond the stored rows reads as zeros
            const int64_t at = prob * a.st.prob_rows + row;
            const uint32_t* c = reinterpret_cast<const uint32_t*>(t.codes + at * (D / 2));
            word[0] = __ldcs(c + q4_word_index<D>(v, 0));
            word[1] = __ldcs(c + q4_word_index<D>(v, 1));
            scale = t.scales[at * (D / kQ4Group) + (v >> 1)];
        }
    }
    const int64_t at = (prob * a.n + i) * D + v * 16;
    if (F32) {
        const float s = elem_to_float<DT>(scale);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t w = q4_transpose_in(word[h], v);
            if (i < a.n)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    static_cast<float*>(out)[at + 8 * h + e] = static_cast<float>(static_cast<int>((w >> (4 * e)) & 15u) - 8) * s;
        }
    } else {
        uint4 o[2];
        q4_decode<DT>(word, scale, v, o);
        if (i < a.n) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at);
            __stcs(dst, o[0]);
            __stcs(dst + 1, o[1]);
        }
    }
}

}  // namespace

#define DC_Q4_DISPATCH(dtype, head_dim, CASE)                 \
    if ((dtype) == DC_BF16) {                                 \
        if ((head_dim) == 64) { CASE(DC_BF16, 64); }          \
        else if ((head_dim) == 128) { CASE(DC_BF16, 128); }   \
        else { CASE(DC_BF16, 256); }                          \
    } else {                                                  \
        if ((head_dim) == 64) { CASE(DC_FP16, 64); }          \
        else if ((head_dim) == 128) { CASE(DC_FP16, 128); }   \
        else { CASE(DC_FP16, 256); }                          \
    }

int q4_write_rows(const void* keys, const void* vals, int64_t stride_b, int64_t stride_h, int64_t stride_s, int n_prob,
                  int kv_heads, int64_t n, int head_dim, int dtype, const Q4Store& st, int64_t row0, int32_t* len,
                  int len_mode, cudaStream_t stream) {
    if (n_prob == 0 || (n == 0 && len_mode == kLenKeep)) return DC_OK;
    WriteArgs a;
    a.keys = static_cast<const uint16_t*>(keys);
    a.vals = static_cast<const uint16_t*>(vals);
    a.stride_b = stride_b; a.stride_h = stride_h; a.stride_s = stride_s;
    a.kv_heads = kv_heads;
    a.n = n; a.row0 = row0;
    a.st = st;
    a.len = len; a.len_mode = len_mode;
    const int64_t rpb = kRowThreads / (head_dim / 16) * kWriteRows;
    const dim3 grid(static_cast<unsigned>(n > 0 ? (n + rpb - 1) / rpb : 1), static_cast<unsigned>(n_prob), 2u);
#define CASE(DT, D) DC_CUDA_TRY(launch_chained(q4_write_kernel<DT, D>, grid, dim3(kRowThreads), 0, stream, 0u, a))
    DC_Q4_DISPATCH(dtype, head_dim, CASE)
#undef CASE
    return DC_OK;
}

int q4_append_rows(const void* keys, const void* vals, int n_prob, int head_dim, int dtype, const Q4Store& st,
                   int64_t max_rows, int32_t* len, uint32_t* status, cudaStream_t stream) {
    const uint16_t* k = static_cast<const uint16_t*>(keys);
    const uint16_t* v = static_cast<const uint16_t*>(vals);
#define CASE(DT, D) q4_append_kernel<DT, D><<<1, 1024, 0, stream>>>(k, v, n_prob, st, max_rows, len, status)
    DC_Q4_DISPATCH(dtype, head_dim, CASE)
#undef CASE
    DC_CUDA_TRY(cudaGetLastError());
    return DC_OK;
}

int q4_window_push(const void* k_new, const void* v_new, int64_t new_stride_b, void* res_k, void* res_v,
                   int64_t res_stride_b, int64_t res_stride_h, int n_prob, int kv_heads, int head_dim, int dtype,
                   const Q4Store& st, int64_t max_rows, int32_t* len, int32_t* win, uint32_t* status, cudaStream_t stream) {
#define CASE(DT, D)                                                                                                     \
    DC_CUDA_TRY(launch_chained(q4_window_push_kernel<DT, D>, dim3(1), dim3(1024), 0, stream, 0u,                        \
                               static_cast<const uint16_t*>(k_new), static_cast<const uint16_t*>(v_new), new_stride_b, \
                               static_cast<uint16_t*>(res_k), static_cast<uint16_t*>(res_v), res_stride_b, res_stride_h, \
                               n_prob, kv_heads, st, max_rows, len, win, status))
    DC_Q4_DISPATCH(dtype, head_dim, CASE)
#undef CASE
    return DC_OK;
}

int q4_read_rows(const Q4Store& st, int64_t n_rows, const int32_t* n_dev, int n_prob, int head_dim, int dtype, int64_t row0,
                 const uint32_t* ids, int64_t ids_stride, int64_t n, void* out_k, void* out_v, bool f32, cudaStream_t stream) {
    if (n_prob == 0 || n == 0 || (out_k == nullptr && out_v == nullptr)) return DC_OK;
    ReadArgs a;
    a.st = st;
    a.n_rows = n_rows; a.n_dev = n_dev;
    a.ids = ids; a.ids_stride = ids_stride;
    a.row0 = row0; a.n = n;
    a.out_k = out_k; a.out_v = out_v;
    const int64_t rpb = kRowThreads / (head_dim / 16);
    const dim3 grid(static_cast<unsigned>((n + rpb - 1) / rpb), static_cast<unsigned>(n_prob), out_k && out_v ? 2u : 1u);
#define CASE(DT, D)                                                                                             \
    if (f32) DC_CUDA_TRY(launch_chained(q4_read_kernel<DT, D, true>, grid, dim3(kRowThreads), 0, stream, 0u, a)); \
    else DC_CUDA_TRY(launch_chained(q4_read_kernel<DT, D, false>, grid, dim3(kRowThreads), 0, stream, 0u, a))
    DC_Q4_DISPATCH(dtype, head_dim, CASE)
#undef CASE
    return DC_OK;
}

}  // namespace dc
