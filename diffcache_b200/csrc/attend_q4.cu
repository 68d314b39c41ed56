// Attention over a store held in 4 bits (format: q4.cuh), the resident 16-bit rows and the new token, with split-K
// and log-sum-exp merge: the 4-bit counterpart of attend.cu (flash_attn_with_kvcache over the gathered buffer,
// src/diffcache/base.py:134-142), over the rows of an id list or over every stored row of a sequence.
#include <algorithm>
#include <cmath>

#include "exchange.cuh"
#include "q4.cuh"

namespace dc {

int lse_combine(const float* acc, int64_t acc_ps, int64_t acc_rs, const float* ml, int64_t ml_ps, int64_t ml_rs,
                int n_part, int64_t rows, int head_dim, int dtype, void* out, float* out_lse, float* out_acc,
                float* out_ml, cudaStream_t stream, const XchgLL* ll, const XchgOut* xout, const XchgFinal* fin, bool keep_nan);

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kHeads = 8;            // query heads of one kv head handled by one CTA
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
    Q4Store st;
    int64_t n_rows;
    const int32_t* n_rows_dev;
    int kv_heads, group;
    const uint16_t* q;
    int64_t q_stride_b, new_stride_b;
    const uint32_t* sel;
    int64_t sel_stride;
    int n_sel;
    int64_t sel_base;
    const int32_t* sel_count;
    const int32_t* lens;
    const uint16_t* k_new;
    const uint16_t* v_new;
    uint16_t* res_k;
    uint16_t* res_v;
    int64_t res_stride_b, res_stride_h;
    int res_len;
    const int32_t* res_len_dev;
    float scale_log2;
    int n_split;
    float* part_acc;                 // (n_prob, group, n_split, D)
    float* part_ml;                  // (n_prob, group, n_split, 2)
};

// grid = (n_split, n_prob, ceil(group / 8)).  A warp takes one row at a time, a lane eight elements of it (one code
// word), every head's score is a butterfly sum and the softmax runs online per warp; the warps merge at the end.
template <int DT, int D>
__global__ void __launch_bounds__(kThreads)
q4_attend_kernel(const Args a) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int WORDS = D / 8;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t prob = blockIdx.y;
    const int split = blockIdx.x;
    const int g0 = blockIdx.z * kHeads;
    const int n_heads = min(kHeads, a.group - g0);
    const int b = static_cast<int>(prob / a.kv_heads), h = static_cast<int>(prob % a.kv_heads);
    const int64_t n_rows = a.n_rows_dev != nullptr ? min(a.n_rows, static_cast<int64_t>(*a.n_rows_dev)) : a.n_rows;
    const int res_len = a.res_len_dev != nullptr ? *a.res_len_dev : a.res_len;
    const int has_new = a.k_new != nullptr ? 1 : 0;
    const int64_t new_off = a.new_stride_b ? b * a.new_stride_b + static_cast<int64_t>(h) * D : prob * D;
    const bool all_rows = a.n_sel < 0;
    const uint32_t* sel = a.sel ? a.sel + prob * a.sel_stride : nullptr;
    const uint16_t* rk = a.res_k ? a.res_k + b * a.res_stride_b + h * a.res_stride_h : nullptr;
    const uint16_t* rv = a.res_v ? a.res_v + b * a.res_stride_b + h * a.res_stride_h : nullptr;
    // rows of the store: the first sel_count ids of the list, or rows 0 .. lens[b] - 1
    int64_t n_store = all_rows ? n_rows : a.n_sel;
    if (!all_rows && a.sel_count) n_store = max(0, min(a.n_sel, a.sel_count[prob]));
    if (all_rows && a.lens) n_store = max(static_cast<int64_t>(0), min(n_rows, static_cast<int64_t>(a.lens[b])));
    const int64_t total = n_store + res_len + has_new;
    const int64_t per = (total + a.n_split - 1) / a.n_split;
    const int64_t j0 = min(total, split * per), j1 = min(total, j0 + per);

    if (has_new && split == 0 && blockIdx.z == 0 && rk != nullptr && tid < D / 8) {   // in-place append of the new token
        const int64_t o = b * a.res_stride_b + h * a.res_stride_h + static_cast<int64_t>(res_len) * D;
        reinterpret_cast<uint4*>(a.res_k + o)[tid] = reinterpret_cast<const uint4*>(a.k_new + new_off)[tid];
        reinterpret_cast<uint4*>(a.res_v + o)[tid] = reinterpret_cast<const uint4*>(a.v_new + new_off)[tid];
    }

    __shared__ float s_q[kHeads][D];
    __shared__ float s_o[kWarps][kHeads][D];
    __shared__ float s_ml[kWarps][kHeads][2];
    const uint16_t* qb = a.q_stride_b ? a.q + b * a.q_stride_b + (static_cast<int64_t>(h) * a.group + g0) * D
                                      : a.q + (prob * a.group + g0) * D;
    for (int i = tid; i < kHeads * D; i += kThreads) s_q[i / D][i % D] = i / D < n_heads ? elem_to_float<DT>(qb[i]) : 0.0f;
    __syncthreads();

    // element of the row behind nibble i of this lane's word
    const int chunk = (lane % WORDS) / (D / 64), w = (lane % WORDS) % (D / 64);
    auto elem = [&](int i) { const int bt = i >> 1; return 16 * (4 * w + (bt == 1 ? 2 : bt == 2 ? 1 : bt)) + 2 * chunk + (i & 1); };
    float m[kHeads], l[kHeads], o[kHeads][8];
#pragma unroll
    for (int g = 0; g < kHeads; g++) {
        m[g] = -INFINITY; l[g] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) o[g][i] = 0.0f;
    }
    for (int64_t j = j0 + warp; j < j1; j += kWarps) {
        float kf[8], vf[8];
#pragma unroll
        for (int i = 0; i < 8; i++) { kf[i] = 0.0f; vf[i] = 0.0f; }
        if (j < n_store) {
            const int64_t row = all_rows ? j : static_cast<int64_t>(sel[j]) - a.sel_base;
            if (row < 0 || row >= n_rows) continue;   // pads and ids of other shards
            const int64_t r = prob * a.st.prob_rows + row;
            if (lane < WORDS) {
                const uint32_t kw = reinterpret_cast<const uint32_t*>(a.st.k.codes + r * (D / 2))[lane];
                const uint32_t vw = reinterpret_cast<const uint32_t*>(a.st.v.codes + r * (D / 2))[lane];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int grp = elem(i) / kQ4Group;
                    kf[i] = static_cast<float>(static_cast<int>((kw >> (4 * i)) & 15u) - 8) *
                            elem_to_float<DT>(a.st.k.scales[r * (D / kQ4Group) + grp]);
                    vf[i] = static_cast<float>(static_cast<int>((vw >> (4 * i)) & 15u) - 8) *
                            elem_to_float<DT>(a.st.v.scales[r * (D / kQ4Group) + grp]);
                }
            }
        } else {
            const bool is_res = j < n_store + res_len;
            const uint16_t* kp = is_res ? rk + (j - n_store) * D : a.k_new + new_off;
            const uint16_t* vp = is_res ? rv + (j - n_store) * D : a.v_new + new_off;
            if (lane < WORDS)
#pragma unroll
                for (int i = 0; i < 8; i++) { kf[i] = elem_to_float<DT>(kp[elem(i)]); vf[i] = elem_to_float<DT>(vp[elem(i)]); }
        }
#pragma unroll
        for (int g = 0; g < kHeads; g++) {
            if (g >= n_heads) continue;
            float x = 0.0f;
            if (lane < WORDS)
#pragma unroll
                for (int i = 0; i < 8; i++) x = fmaf(s_q[g][elem(i)], kf[i], x);
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, off);
            x *= a.scale_log2;
            const float mn = fmaxf(m[g], x);
            const float alpha = m[g] == -INFINITY ? 0.0f : exp2f(m[g] - mn);
            const float p = x == -INFINITY ? 0.0f : exp2f(x - mn);
            l[g] = l[g] * alpha + p;
            m[g] = mn;
#pragma unroll
            for (int i = 0; i < 8; i++) o[g][i] = o[g][i] * alpha + p * vf[i];
        }
    }
#pragma unroll
    for (int g = 0; g < kHeads; g++) {
        if (lane < WORDS)
#pragma unroll
            for (int i = 0; i < 8; i++) s_o[warp][g][elem(i)] = o[g][i];
        if (lane == 0) { s_ml[warp][g][0] = m[g]; s_ml[warp][g][1] = l[g]; }
    }
    __syncthreads();
    for (int e = tid; e < n_heads * D; e += kThreads) {
        const int g = e / D, d = e % D;
        float mx = -INFINITY;
        for (int i = 0; i < kWarps; i++) mx = fmaxf(mx, s_ml[i][g][0]);
        float acc = 0.0f, sum = 0.0f;
        for (int i = 0; i < kWarps; i++) {
            if (s_ml[i][g][0] == -INFINITY && s_ml[i][g][1] == 0.0f) continue;
            const float f = exp2f(s_ml[i][g][0] - mx);
            acc += s_o[i][g][d] * f;
            sum += s_ml[i][g][1] * f;
        }
        const int64_t slot = (prob * a.group + g0 + g) * a.n_split + split;
        a.part_acc[slot * D + d] = acc;
        if (d == 0) { a.part_ml[2 * slot] = mx; a.part_ml[2 * slot + 1] = sum; }
    }
}

int splits(int n_prob, int64_t total_rows) {
    const int64_t target = std::max(1, 2 * sm_count() / std::max(1, n_prob));
    const int64_t by_rows = std::max<int64_t>(1, (total_rows + 31) / 32);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(std::min(target, by_rows), 256)));
}

}  // namespace

int64_t q4_attend_scratch_bytes(int n_prob, int group, int head_dim) {
    const int64_t ctas = std::min<int64_t>(static_cast<int64_t>(n_prob) * 256, 2ll * sm_count() + n_prob);
    return ctas * group * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
}

int q4_attend(const Q4Attend& in, cudaStream_t stream) {
    DC_REQUIRE(in.q != nullptr && in.scratch != nullptr, "q4_attend: null q/scratch");
    DC_REQUIRE(in.n_prob >= 0 && in.n_prob <= 65535 && in.kv_heads >= 1 && in.n_prob % in.kv_heads == 0,
               "q4_attend: n_prob=%d must be a multiple of kv_heads=%d", in.n_prob, in.kv_heads);
    DC_REQUIRE(in.group >= 1 && in.group <= 64, "q4_attend: group=%d", in.group);
    DC_REQUIRE(in.res_len >= 0, "q4_attend: negative length");
    DC_REQUIRE(in.n_sel <= 0 || (in.sel != nullptr && in.sel_stride >= in.n_sel), "q4_attend: n_sel=%d without ids, or sel_stride=%lld",
               in.n_sel, static_cast<long long>(in.sel_stride));
    DC_REQUIRE((in.k_new == nullptr) == (in.v_new == nullptr), "q4_attend: k_new and v_new must both be set or both be NULL");
    DC_REQUIRE((in.res_k == nullptr) == (in.res_v == nullptr), "q4_attend: res_k and res_v must both be set or both be NULL");
    DC_REQUIRE(in.res_len == 0 || in.res_k != nullptr, "q4_attend: res_len > 0 needs resident buffers");
    DC_REQUIRE((in.out != nullptr) != (in.out_acc != nullptr && in.out_ml != nullptr),
               "q4_attend: give either out or (out_acc, out_ml)");
    DC_REQUIRE(in.res_stride_b % 8 == 0 && in.res_stride_h % 8 == 0 && in.q_stride_b % 8 == 0 && in.new_stride_b % 8 == 0,
               "q4_attend: strides must be multiples of 8 elements");
    DC_REQUIRE(((reinterpret_cast<uintptr_t>(in.q) | reinterpret_cast<uintptr_t>(in.k_new) |
                 reinterpret_cast<uintptr_t>(in.v_new) | reinterpret_cast<uintptr_t>(in.res_k) |
                 reinterpret_cast<uintptr_t>(in.res_v) | reinterpret_cast<uintptr_t>(in.scratch)) & 15) == 0,
               "q4_attend: every row pointer must be 16-byte aligned");
    if (in.n_prob == 0) return DC_OK;
    Args a;
    a.st = in.st;
    a.n_rows = in.n_rows; a.n_rows_dev = in.n_rows_dev;
    a.kv_heads = in.kv_heads; a.group = in.group;
    a.q = static_cast<const uint16_t*>(in.q);
    a.q_stride_b = in.q_stride_b; a.new_stride_b = in.new_stride_b;
    a.sel = in.sel; a.sel_stride = in.sel_stride; a.n_sel = in.n_sel; a.sel_base = in.sel_base; a.sel_count = in.sel_count;
    a.lens = in.lens;
    a.k_new = static_cast<const uint16_t*>(in.k_new); a.v_new = static_cast<const uint16_t*>(in.v_new);
    a.res_k = static_cast<uint16_t*>(in.res_k); a.res_v = static_cast<uint16_t*>(in.res_v);
    a.res_stride_b = in.res_stride_b; a.res_stride_h = in.res_stride_h;
    a.res_len = in.res_len; a.res_len_dev = in.res_len_dev;
    a.scale_log2 = (in.scale > 0.0f ? in.scale : 1.0f / std::sqrt(static_cast<float>(in.head_dim))) * kLog2e;
    const int64_t total = (in.n_sel < 0 ? in.n_rows : in.n_sel) + in.res_len + (in.k_new ? 1 : 0);
    a.n_split = splits(in.n_prob, total);
    a.part_acc = static_cast<float*>(in.scratch);
    a.part_ml = a.part_acc + static_cast<int64_t>(in.n_prob) * a.n_split * in.group * in.head_dim;
    const dim3 grid(static_cast<unsigned>(a.n_split), static_cast<unsigned>(in.n_prob),
                    static_cast<unsigned>((in.group + kHeads - 1) / kHeads));
#define CASE(DT, D) DC_CUDA_TRY(launch_chained(q4_attend_kernel<DT, D>, grid, dim3(kThreads), 0, stream, 0u, a))
    if (in.dtype == DC_BF16) {
        if (in.head_dim == 64) CASE(DC_BF16, 64);
        else if (in.head_dim == 128) CASE(DC_BF16, 128);
        else CASE(DC_BF16, 256);
    } else {
        if (in.head_dim == 64) CASE(DC_FP16, 64);
        else if (in.head_dim == 128) CASE(DC_FP16, 128);
        else CASE(DC_FP16, 256);
    }
#undef CASE
    return lse_combine(a.part_acc, in.head_dim, static_cast<int64_t>(a.n_split) * in.head_dim, a.part_ml, 2,
                       static_cast<int64_t>(a.n_split) * 2, a.n_split, static_cast<int64_t>(in.n_prob) * in.group, in.head_dim,
                       in.dtype, in.out, in.out_lse, in.out_acc, in.out_ml, stream, nullptr, in.xout, in.fin, true);
}

}  // namespace dc
