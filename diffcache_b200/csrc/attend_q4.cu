// Attention over a store held in 4 bits (format: q4.cuh), the resident 16-bit rows and the new token, with split-K
// and log-sum-exp merge: the 4-bit counterpart of attend.cu (flash_attn_with_kvcache over the gathered buffer,
// src/diffcache/base.py:134-142), over the rows of an id list or over every stored row of a sequence.
//
// Bound, at head_dim 128 and four query heads: 144 bytes a row against 387 instructions per 16 rows, most of them turning
// nibbles into fragment values.  64 problems x 32768 consecutive rows: 76 us = 4.0 TB/s of codes and scales, 2.7 instructions
// per clock (operands loaded to registers without the ring: 116; keys as the columns of B instead of the rows of A: 110;
// weights scaled and split in fp32, keys as fp16 integers with their offset subtracted: 83).  16384 random rows each: 63 us, 4.8 TB/s of DRAM traffic, twice the bytes used.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "exchange.cuh"
#include "q4_mma.cuh"

namespace dc {

namespace cg = cooperative_groups;

int lse_combine(const float* acc, int64_t acc_ps, int64_t acc_rs, const float* ml, int64_t ml_ps, int64_t ml_rs,
                int n_part, int64_t rows, int head_dim, int dtype, void* out, float* out_lse, float* out_acc,
                float* out_ml, cudaStream_t stream, const XchgLL* ll, const XchgOut* xout, const XchgFinal* fin, bool keep_nan);

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kHeads = 8;            // query heads of one kv head handled by one CTA (columns of the second product)
constexpr int kTile = 16;            // rows a warp takes at a time
constexpr int kMaxCluster = 8;        // CTAs of a problem that finish its output together (the portable cluster size)
constexpr float kLog2e = 1.4426950408889634f;
__host__ __device__ constexpr int ctas_per_sm(int head_dim) { return head_dim <= 128 ? 4 : 2; }

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
    int n_store_split;               // CTAs (per problem and head chunk) that take store rows; the others take 16-bit rows
    int n_split;
    int64_t run;                     // rows of the store a CTA takes; 0: an equal share of the problem's rows
    int cluster;                     // that many consecutive CTAs of a problem are one cluster and merge their results
    uint16_t* out;                   // set where one cluster is all there is: (n_prob, group, D), and optional (n_prob, group)
    float* out_lse;
    float* part_acc;                 // otherwise: (n_prob, group, n_split / cluster, D)
    float* part_ml;                  // (n_prob, group, n_split / cluster, 2)
};

// ---- a tile of 16 store rows in shared memory, private to one warp ----
// Asynchronous copies of 16 (codes) and 4 / 8 / 16 bytes (a row's scales); with `ok` false zeros are written instead.
template <int BYTES>
__device__ __forceinline__ void copy_async(unsigned dst, const void* src) {
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_async(unsigned dst, const void* src, bool ok) {
    const int n = ok ? BYTES : 0;
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&r)[N], unsigned addr) {
    if (N == 1) asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(r[0]) : "r"(addr));
    else if (N == 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];\n" : "=r"(r[0]), "=r"(r[N > 1 ? 1 : 0]) : "r"(addr));
    else
#pragma unroll
        for (int i = 0; i + 3 < N; i += 4)
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n"
                         : "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]) : "r"(addr + 4 * i));
}

template <int D>
struct Ring {
    static constexpr int CODES = kTile * (D / 2);        // one tensor's codes of a tile
    static constexpr int SCALES = kTile * (D / 16);
    static constexpr int STAGE = 2 * CODES + 2 * SCALES; // [K codes | V codes | K scales | V scales]
    static constexpr int STAGES = 4;
    // Byte of 16-byte chunk c of row r among a tile's codes.  Rows and chunks are permuted so that neither the keys (eight
    // rows, a quarter row per lane) nor the values (rows 4t + i, an eighth per lane) make a warp's lanes share banks.
    __device__ static __forceinline__ int chunk(int r, int c) {
        if (D == 64) return ((r & ~3) | ((r & 3) ^ (r >> 2))) * 32 + c * 16;
        if (D == 128) return (r ^ ((r >> 2) & 1)) * 64 + ((c ^ (r >> 2)) & 3) * 16;
        return r * 128 + ((c ^ (2 * (r >> 2)) ^ (r & 1)) & 7) * 16;
    }
};
template <int D>
constexpr size_t attend_smem_bytes() {
    const size_t ring = static_cast<size_t>(kWarps) * Ring<D>::STAGES * Ring<D>::STAGE;
    const size_t merge = static_cast<size_t>(kWarps) * kHeads * (D + 4) * sizeof(float);
    return ring > merge ? ring : merge;
}

// The pair of weights (x, y) as B operand of a head's two column groups: hi = rounded to 16 bits, rest = rounded remainder.
// With few heads (FEW) the lanes of rows g < 4 need hi, the others rest: `keep_lo` / `keep_hi` are byte selectors that read
// the rounded halves as floats there, and zeros in the lanes g < 4, so that one expression serves both.
template <bool BF16, bool FEW>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t keep_lo, uint32_t keep_hi, uint32_t& hi, uint32_t& rest) {
    const uint32_t r = pack2<BF16>(x, y);
    if (BF16) {
        hi = r;
        rest = pack2<true>(x - __uint_as_float(__byte_perm(r, 0u, keep_lo)), y - __uint_as_float(__byte_perm(r, 0u, keep_hi)));
        if (FEW) hi = rest;
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
        rest = pack2<false>(x - f.x, y - f.y);
        hi = FEW && keep_lo != 0x4444u ? rest : r;
    }
}
// Weights times bf16 scales, again as a bf16 value and its remainder, in packed bf16: with the weight as h + x,
//   hi = round(h s),  lo = round(x s + (h s - hi)),
// where h s - hi is exact (16 significant bits less the 8 kept).  hi + lo is the product to 2^-15: the remainder of a
// weight is kept to 2^-16 of it, and lo, at most 2^-7 of the product, is rounded once.  With few heads the lanes that hold
// the value pass h = 0 and the value as x, so that lo is round(h s) there and the remainder in the others.
template <bool FEW>
__device__ __forceinline__ void scale_pair(uint32_t h, uint32_t x, uint32_t s, uint32_t& hi, uint32_t& lo) {
    uint32_t v, e;
    asm("mul.rn.bf16x2 %0, %1, %2;\n" : "=r"(v) : "r"(h), "r"(s));
    asm("{\n .reg .b32 n;\n neg.bf16x2 n, %3;\n fma.rn.bf16x2 %0, %1, %2, n;\n}\n" : "=r"(e) : "r"(h), "r"(s), "r"(v));
    asm("fma.rn.bf16x2 %0, %1, %2, %3;\n" : "=r"(lo) : "r"(x), "r"(s), "r"(e));
    hi = FEW ? lo : v;
}

__device__ __forceinline__ float exp2_fast(float x) {   // 2^x to 2 ulp, 0 below 2^-126 and for -inf
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
    return r;
}

// Running softmax of the rows one warp has seen.  Lane (g, t) = (lane / 4, lane % 4) holds the scores x[2 * blk + e] of two
// rows (blk) of the tile for heads 2t + e, in log2 units, -inf where there is no row.  The reference value `m` the
// weights are relative to follows the maximum only when a score exceeds it by more than 8 (weights up to 2^8 cost
// nothing in fp32), so that a tile normally needs one vote and no reduction; the same columns of o are heads 2t + e.
// On return x holds the weights.
template <int NT>
__device__ __forceinline__ void softmax_step(float (&x)[4], float (&m)[2], float (&l)[2], float (&o)[NT][4]) {
    const float top[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
    if (__any_sync(0xFFFFFFFFu, top[0] > m[0] + 8.0f || top[1] > m[1] + 8.0f)) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float mx = fmaxf(top[e], m[e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16));
            const float alpha = mx == m[e] ? 1.0f : exp2_fast(m[e] - mx);   // 0 where nothing was seen before
            m[e] = mx;
            l[e] *= alpha;
#pragma unroll
            for (int i = 0; i < NT; i++) { o[i][e] *= alpha; o[i][2 + e] *= alpha; }
        }
    }
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const float ref = m[e] == -INFINITY ? 0.0f : m[e];   // nothing seen yet: every weight is 2^-inf = 0
        x[e] = exp2_fast(x[e] - ref);
        x[2 + e] = exp2_fast(x[2 + e] - ref);
        l[e] += x[e] + x[2 + e];
    }
}

// Weights (rows of the first product's output by heads) to the layout of the second product's B operand: lane (g, t) gets
// y[2 * blk + e] = the weight of row 4t + 2 blk + e for head g.  Row r of a block lives in the lanes of g = r.
__device__ __forceinline__ void transpose_weights(const float (&x)[4], float (&y)[4], int g, int t) {
#pragma unroll
    for (int blk = 0; blk < 2; blk++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int from = 4 * (2 * t + e) + (g >> 1);
            const float even = __shfl_sync(0xFFFFFFFFu, x[2 * blk], from), odd = __shfl_sync(0xFFFFFFFFu, x[2 * blk + 1], from);
            y[2 * blk + e] = g & 1 ? odd : even;
        }
}

// grid = (n_split, n_prob, ceil(group / 8)).
//
// Store rows.  S^T = K Q^T with m16n8k16 MMAs: 16 store rows are the rows of A, up to 8 query heads the columns of B.  The
// codes enter as small integers (fp16 subnormals, exact: codes_subnormal), so a group's partial product is exact up to fp32
// accumulation and its scale is applied once, in fp32.  The query of a head is normalised by a power of two so that a bf16 query is exact in fp16 too.
// O^T = V^T P^T: the value codes are A (16 elements of a tile x 16 rows, bf16 integers), the weights are B; a value's scale
// depends on (row, group) only, so it multiplies the weight, which enters as a bf16 value and its remainder
// (scale_pair for bf16 scales, split_pair for the 11 bits of fp16 ones).  With at most four heads value and remainder are two column groups of ONE MMA (columns h and h + 4),
// otherwise two MMAs.  The rows of a tile are numbered so that a lane's rows in both fragments are 4t .. 4t + 3.
// Every warp streams its tiles through a ring of its own in shared memory, three tiles ahead of the arithmetic; the stored
// order of the codes makes each lane's share of a row one load.  Warps are independent until the end.
//
// 16-bit rows (resident rows, new token): the same two products on the element type, by CTAs of their own.
template <int DT, int D, bool FEW, bool IDS>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(D))
q4_attend_kernel(const Args a) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int NT = D / 16;       // 16-element tiles of a row
    constexpr int NG = D / kQ4Group;
    constexpr bool BF16 = DT == DC_BF16;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int64_t prob = blockIdx.y;
    const int split = blockIdx.x;
    const int g0 = blockIdx.z * kHeads;
    const int n_heads = min(kHeads, a.group - g0);
    const int b = static_cast<int>(prob / a.kv_heads), h = static_cast<int>(prob % a.kv_heads);

    __shared__ __align__(16) uint16_t s_q[kHeads][D];
    extern __shared__ __align__(128) unsigned char s_ring[];   // the warps' rings; at the end their partial outputs
    __shared__ uint32_t s_ok[kWarps][Ring<D>::STAGES];         // rows of a tile that exist (id lists)
    __shared__ float s_ml[kWarps][kHeads][2];
    __shared__ float s_sum[kHeads][2];                         // the CTA's (reference, sum), for the cluster
    {
        const uint16_t* qb = a.q_stride_b ? a.q + b * a.q_stride_b + (static_cast<int64_t>(h) * a.group + g0) * D
                                          : a.q + (prob * a.group + g0) * D;
        for (int i = tid; i < kHeads * D / 8; i += kThreads) {
            const int head = i / (D / 8);
            reinterpret_cast<uint4*>(&s_q[0][0])[i] =
                head < n_heads ? reinterpret_cast<const uint4*>(qb)[i] : make_uint4(0, 0, 0, 0);
        }
    }
    const int res_len = a.res_len_dev != nullptr ? *a.res_len_dev : a.res_len;
    const int has_new = a.k_new != nullptr ? 1 : 0;
    const int64_t new_off = a.new_stride_b ? b * a.new_stride_b + static_cast<int64_t>(h) * D : prob * D;
    const int64_t res_off = b * a.res_stride_b + h * a.res_stride_h;
    const uint16_t* qrow = s_q[FEW ? g & 3 : g];   // few heads: rows 4..7 repeat heads 0..3

    const uint32_t keep_lo = FEW && g < 4 ? 0x4444u : 0x1044u, keep_hi = FEW && g < 4 ? 0x4444u : 0x3244u;

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float o[NT][4];
#pragma unroll
    for (int i = 0; i < NT; i++) { o[i][0] = 0.0f; o[i][1] = 0.0f; o[i][2] = 0.0f; o[i][3] = 0.0f; }

    if (split < a.n_store_split) {
        const int64_t n_rows = a.n_rows_dev != nullptr ? min(a.n_rows, static_cast<int64_t>(*a.n_rows_dev)) : a.n_rows;
        // rows of the store: the first sel_count ids of the list, or rows 0 .. lens[b] - 1
        int64_t n_store = IDS ? a.n_sel : n_rows;
        if (IDS && a.sel_count) n_store = max(static_cast<int64_t>(0), min(n_store, static_cast<int64_t>(a.sel_count[prob])));
        if (!IDS && a.lens) n_store = max(static_cast<int64_t>(0), min(n_rows, static_cast<int64_t>(a.lens[b])));
        int64_t per = a.run;
        if (per == 0) per = ((n_store + a.n_store_split - 1) / a.n_store_split + kTile - 1) / kTile * kTile;
        const int64_t j0 = min(n_store, split * per), j1 = min(n_store, j0 + per);
        if (a.run != 0 && j0 >= j1) {   // a run behind the end of this sequence: an empty partial, whose sums are not read
            if (tid < n_heads) {
                float* ml = a.part_ml + 2 * ((prob * a.group + g0 + tid) * a.n_split + split);
                ml[0] = -INFINITY;
                ml[1] = 0.0f;
            }
            return;
        }
        const uint8_t* kc = a.st.k.codes + prob * a.st.prob_rows * (D / 2);
        const uint8_t* vc = a.st.v.codes + prob * a.st.prob_rows * (D / 2);
        const uint8_t* sc_base = reinterpret_cast<const uint8_t*>((lane < 16 ? a.st.k.scales : a.st.v.scales) + prob * a.st.prob_rows * NG);

        // ---- the ring: lane copies chunks lane + 32 j of both tensors' codes and one row's scales of one tensor ----
        using R = Ring<D>;
        constexpr int CPR = D / 32;                    // chunks per row
        constexpr int NC = kTile * CPR / 32;           // chunks per lane and tensor
        const unsigned ring = smem_u32(s_ring) + warp * R::STAGES * R::STAGE;
        int dst[NC];
#pragma unroll
        for (int j = 0; j < NC; j++) dst[j] = R::chunk((lane + 32 * j) / CPR, (lane + 32 * j) % CPR);
        const int dst_scale = 2 * R::CODES + lane * (D / 16);
        // This lane's id of a tile's 16 (lane and lane + 16 hold the same), as listed, and as a row: -1 where there is none.
        // sel_base + n_rows < 2^32 (checked on the host), so pads and ids of other shards end up beyond n_rows.
        auto listed_id = [&](int i) -> uint32_t {
            const int64_t j = j0 + (warp + static_cast<int64_t>(i) * kWarps) * kTile + (lane & 15);
            return j < j1 ? a.sel[prob * a.sel_stride + j] - static_cast<uint32_t>(a.sel_base) : 0xFFFFFFFFu;
        };
        auto row_of = [&](uint32_t id) -> int32_t { return id < n_rows ? static_cast<int32_t>(id) : -1; };
        // Consecutive rows: 16 of them are one run of bytes per array, so the addresses just advance from tile to tile.
        // (ids: this lane's chunk of any row is a multiple of the row length away.)
        const uint8_t* kp = kc + (IDS ? lane % CPR * 16 : (j0 + warp * kTile) * (D / 2) + lane * 16);
        const uint8_t* vp = vc + (IDS ? lane % CPR * 16 : (j0 + warp * kTile) * (D / 2) + lane * 16);
        const uint8_t* sp = sc_base + (j0 + warp * kTile + (lane & 15)) * (D / 16);
        const int n_mine = static_cast<int>((max(j1 - j0 - warp * kTile, static_cast<int64_t>(0)) + kWarps * kTile - 1) / (kWarps * kTile));
        const int last_rows = static_cast<int>(j1 - j0) - (warp + (n_mine - 1) * kWarps) * kTile;   // of this warp's last tile; > 16: whole
        auto issue = [&](unsigned st, int i, int32_t id) {   // this warp's tile i into the stage at st
            if (!IDS) {
                if (i < n_mine - 1 || (i == n_mine - 1 && last_rows >= kTile)) {
#pragma unroll
                    for (int j = 0; j < NC; j++) {
                        copy_async<16>(st + dst[j], kp + 512 * j);
                        copy_async<16>(st + R::CODES + dst[j], vp + 512 * j);
                    }
                    copy_async<D / 16>(st + dst_scale, sp);
                } else if (i < n_mine) {               // the last rows; zeros behind them
#pragma unroll
                    for (int j = 0; j < NC; j++) {
                        const bool ok = (lane + 32 * j) / CPR < last_rows;
                        copy_async<16>(st + dst[j], ok ? kp + 512 * j : kc, ok);
                        copy_async<16>(st + R::CODES + dst[j], ok ? vp + 512 * j : vc, ok);
                    }
                    const bool ok = (lane & 15) < last_rows;
                    copy_async<D / 16>(st + dst_scale, ok ? sp : sc_base, ok);
                }
                kp += kWarps * kTile * (D / 2);
                vp += kWarps * kTile * (D / 2);
                sp += kWarps * kTile * (D / 16);
            } else {
                const uint32_t ok = __ballot_sync(0xFFFFFFFFu, id >= 0);
                const uint32_t safe = max(id, 0);      // (nothing is read where there is no row)
                const uint8_t* sc_at = sc_base + static_cast<uint64_t>(safe) * (D / 16);
#pragma unroll
                for (int j = 0; j < NC; j++) {
                    const uint64_t off = static_cast<uint64_t>(__shfl_sync(0xFFFFFFFFu, safe, (lane + 32 * j) / CPR)) * (D / 2);
                    if (ok == 0xFFFFFFFFu) {
                        copy_async<16>(st + dst[j], kp + off);
                        copy_async<16>(st + R::CODES + dst[j], vp + off);
                    } else {
                        const bool there = (ok >> ((lane + 32 * j) / CPR)) & 1u;
                        copy_async<16>(st + dst[j], kp + off, there);
                        copy_async<16>(st + R::CODES + dst[j], vp + off, there);
                    }
                }
                if (ok == 0xFFFFFFFFu) copy_async<D / 16>(st + dst_scale, sc_at);
                else copy_async<D / 16>(st + dst_scale, sc_at, id >= 0);
                if (lane == 0) s_ok[warp][i % R::STAGES] = ok & 0xFFFFu;
            }
            copy_commit();
        };
        // where this lane reads: keys of rows 4 (g / 2) + 2 blk + g % 2, values and scales of rows 4t + i
        unsigned k_at[2], v_at[4];
        const unsigned ks_at = 2 * R::CODES + (4 * (g >> 1) + (g & 1)) * (D / 16);
#pragma unroll
        for (int blk = 0; blk < 2; blk++) {
            const int r = 4 * (g >> 1) + 2 * blk + (g & 1);
            k_at[blk] = D == 64 ? R::chunk(r, t >> 1) + (t & 1) * 8 : R::chunk(r, D == 128 ? t : 2 * t);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            v_at[i] = R::CODES + R::chunk(4 * t + i, g * (D / 16) / 16) + g * (D / 16) % 16;
        uint32_t id[R::STAGES] = {};                   // of the first tiles; then id[0] runs one tile ahead of the copies
        if (IDS) {
#pragma unroll
            for (int i = 0; i < R::STAGES; i++) id[i] = listed_id(i);
        }
        if (n_mine > 0) {
#pragma unroll
            for (int i = 0; i < R::STAGES - 1; i++) issue(ring + i * R::STAGE, i, IDS ? row_of(id[i]) : 0);   // beyond the last: nothing
        }
        id[0] = id[R::STAGES - 1];
        __syncthreads();                               // the query is in shared memory
        // query fragments, normalised to [2^14, 2^15) by a power of two
        uint32_t top = 0;                              // magnitude bits order like magnitudes
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            const uint4 w = *reinterpret_cast<const uint4*>(qrow + 32 * i + 8 * t);
            top = __vmaxu2(top, __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu)));
        }
        top = __vmaxu2(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = __vmaxu2(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        float down, up_g;
        q4_normalise(elem_to_float<DT>(static_cast<uint16_t>(max(top & 0xFFFFu, top >> 16))), down, up_g);
        up_g *= a.scale_log2;
        const float up[2] = {__shfl_sync(0xFFFFFFFFu, up_g, 8 * t), __shfl_sync(0xFFFFFFFFu, up_g, 8 * t + 4)};   // heads 2t, 2t + 1
        uint32_t qa[NT][2];
        float start[NG][2];                            // where the sums of a group start: heads 2t, 2t + 1
#pragma unroll
        for (int w = 0; w < D / 64; w++)
#pragma unroll
            for (int gp = 0; gp < 2; gp++) {
                float sum = 0.0f;                      // of head g over this lane's part of the group
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int d = 16 * (4 * w + 2 * gp) + 2 * (2 * t + c);   // a tile's element; + 16 is the group's other tile
                    const uint32_t w0 = *reinterpret_cast<const uint32_t*>(qrow + d), w1 = *reinterpret_cast<const uint32_t*>(qrow + d + 16);
                    uint32_t (&q)[2] = qa[4 * w + 2 * gp + c];
                    q[0] = pack2<false>(low_elem<DT>(w0) * down, low_elem<DT>(w1) * down);
                    q[1] = pack2<false>(high_elem<DT>(w0) * down * 0.0625f, high_elem<DT>(w1) * down * 0.0625f);
                    const float2 r0 = __half22float2(*reinterpret_cast<const __half2*>(&q[0]));
                    const float2 r1 = __half22float2(*reinterpret_cast<const __half2*>(&q[1]));
                    sum += (r0.x + r0.y) + 16.0f * (r1.x + r1.y);
                }
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
                start[2 * w + gp][0] = -0x1p-21f * __shfl_sync(0xFFFFFFFFu, sum, 8 * t);
                start[2 * w + gp][1] = -0x1p-21f * __shfl_sync(0xFFFFFFFFu, sum, 8 * t + 4);
            }

        const CodeConst cc(static_cast<uint32_t>(a.kv_heads) >> 31);
        auto compute = [&](unsigned st, uint32_t ok) {
            float sc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            {
                uint32_t kw[2][D / 32], ks[2][D / 64];
#pragma unroll
                for (int blk = 0; blk < 2; blk++) {
                    if (D == 256) {                    // chunks 2t and 2t + 1: the permutation flips bit 0 or not
                        uint32_t half[4];
                        lds_words<4>(half, st + k_at[blk]);
#pragma unroll
                        for (int i = 0; i < 4; i++) kw[blk][i] = half[i];
                        lds_words<4>(half, st + (k_at[blk] ^ 16u));
#pragma unroll
                        for (int i = 0; i < 4; i++) kw[blk][(D / 64 + i) % (D / 32)] = half[i];
                    } else {
                        lds_words<D / 32>(kw[blk], st + k_at[blk]);
                    }
                    lds_words<D / 64>(ks[blk], st + ks_at + 2 * blk * (D / 16));
                }
#pragma unroll
                for (int w = 0; w < D / 64; w++) {
                    float acc[2][4];
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t p[4], r[4];
                        codes_subnormal(kw[0][c * (D / 64) + w], p);
                        codes_subnormal(kw[1][c * (D / 64) + w], r);
#pragma unroll
                        for (int gp = 0; gp < 2; gp++) {
                            const uint32_t (&q)[2] = qa[4 * w + 2 * gp + c];
                            if (c == 0) {
                                const float s4[4] = {start[2 * w + gp][0], start[2 * w + gp][1], start[2 * w + gp][0], start[2 * w + gp][1]};
                                mma_from(acc[gp], s4, p[2 * gp], r[2 * gp], p[2 * gp + 1], r[2 * gp + 1], q[0], q[1]);
                            }
                            else mma<false>(acc[gp], p[2 * gp], r[2 * gp], p[2 * gp + 1], r[2 * gp + 1], q[0], q[1]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        sc[i] = fmaf(low_elem<DT>(ks[i >> 1][w]), acc[0][i], sc[i]);
                        sc[i] = fmaf(high_elem<DT>(ks[i >> 1][w]), acc[1][i], sc[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++) sc[i] = sc[i] * up[i & 1] * 0x1p24f;   // up * 2^24 may overflow
            }
            if (ok != 0xFFFFu) {   // rows that are not there: no weight (their scales and codes are zeros)
                const int r = 4 * (g >> 1) + (g & 1);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (((ok >> (r + 2 * (i >> 1))) & 1u) == 0) sc[i] = -INFINITY;
            }
            softmax_step<NT>(sc, m, l, o);
            float wt[4];
            transpose_weights(sc, wt, g, t);
            uint32_t ph[2], px[2];                     // the weights as value and remainder (scale_pair)
            if (BF16)
#pragma unroll
                for (int blk = 0; blk < 2; blk++) {
                    const uint32_t r = pack2<true>(wt[2 * blk], wt[2 * blk + 1]);
                    const uint32_t rest = pack2<true>(wt[2 * blk] - low_elem<DC_BF16>(r), wt[2 * blk + 1] - high_elem<DC_BF16>(r));
                    ph[blk] = FEW && g < 4 ? 0u : r;
                    px[blk] = FEW && g < 4 ? r : rest;
                }
            constexpr int WV = D == 64 ? 1 : 2;        // words of a row's values and scales read at a time
            uint32_t vw[4][WV], vs[4][WV];
#pragma unroll
            for (int w = 0; w < D / 64; w++) {
                if (w % WV == 0) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        lds_words<WV>(vw[i], st + v_at[i] + 4 * w);
                        lds_words<WV>(vs[i], st + 2 * R::CODES + R::SCALES + (4 * t + i) * (D / 16) + 4 * w);
                    }
                }
                uint32_t hi[2][2], lo[2][2];   // [group of the word][row block]
#pragma unroll
                for (int gp = 0; gp < 2; gp++)
#pragma unroll
                    for (int blk = 0; blk < 2; blk++) {
                        if (BF16) {   // both rows' scales as a pair
                            scale_pair<FEW>(ph[blk], px[blk], __byte_perm(vs[2 * blk][w % WV], vs[2 * blk + 1][w % WV], gp ? 0x7632 : 0x5410),
                                            hi[gp][blk], lo[gp][blk]);
                        } else {
                            const float p0 = wt[2 * blk] * (gp ? high_elem<DT>(vs[2 * blk][w % WV]) : low_elem<DT>(vs[2 * blk][w % WV]));
                            const float p1 = wt[2 * blk + 1] *
                                             (gp ? high_elem<DT>(vs[2 * blk + 1][w % WV]) : low_elem<DT>(vs[2 * blk + 1][w % WV]));
                            split_pair<true, FEW>(p0, p1, keep_lo, keep_hi, hi[gp][blk], lo[gp][blk]);
                        }
                    }
                // value codes of rows (4t, 4t + 1) and (4t + 2, 4t + 3): nibble pairs of the same element
                uint32_t va[2][2][4];
#pragma unroll
                for (int blk = 0; blk < 2; blk++) {
                    codes_bf16(cc, __byte_perm(vw[2 * blk][w % WV], vw[2 * blk + 1][w % WV], 0x5410), va[blk][0]);   // tiles 4w, 4w + 2
                    codes_bf16(cc, __byte_perm(vw[2 * blk][w % WV], vw[2 * blk + 1][w % WV], 0x7632), va[blk][1]);   // tiles 4w + 1, 4w + 3
                }
#pragma unroll
                for (int tile = 0; tile < 4; tile++) {
                    const int half = tile & 1, pos = (tile >> 1) * 2, gp = tile >> 1;
                    mma<true>(o[4 * w + tile], va[0][half][pos], va[0][half][pos + 1], va[1][half][pos], va[1][half][pos + 1],
                              hi[gp][0], hi[gp][1]);
                }
                if (!FEW)
#pragma unroll
                    for (int tile = 0; tile < 4; tile++) {
                        const int half = tile & 1, pos = (tile >> 1) * 2, gp = tile >> 1;
                        mma<true>(o[4 * w + tile], va[0][half][pos], va[0][half][pos + 1], va[1][half][pos], va[1][half][pos + 1],
                                  lo[gp][0], lo[gp][1]);
                    }
            }
        };
        unsigned now = ring, next = ring + (R::STAGES - 1) * R::STAGE;
        for (int i = 0; i < n_mine; i++) {
            copy_wait<R::STAGES - 2>();
            __syncwarp();   // every lane's copies of this tile have landed, and nobody reads the tile before any more
            issue(next, i + R::STAGES - 1, IDS ? row_of(id[0]) : 0);
            if (IDS) id[0] = listed_id(i + R::STAGES);
            compute(now, IDS ? s_ok[warp][i % R::STAGES] : i < n_mine - 1 || last_rows >= kTile ? 0xFFFFu : (1u << last_rows) - 1u);
            next = now;
            now = now == ring + (R::STAGES - 1) * R::STAGE ? ring : now + R::STAGE;
        }
        copy_wait<0>();
    } else {
        // flash-attn's in-place append of the new token (base.py:134-142): one CTA per problem
        if (has_new && split == a.n_store_split && blockIdx.z == 0 && a.res_k != nullptr && tid < D / 8) {
            const int64_t off = res_off + static_cast<int64_t>(res_len) * D;
            reinterpret_cast<uint4*>(a.res_k + off)[tid] = reinterpret_cast<const uint4*>(a.k_new + new_off)[tid];
            reinterpret_cast<uint4*>(a.res_v + off)[tid] = reinterpret_cast<const uint4*>(a.v_new + new_off)[tid];
        }
        const int parts = a.n_split - a.n_store_split, part = split - a.n_store_split;
        const int total = res_len + has_new;
        int per = (total + parts - 1) / parts;
        per = (per + kTile - 1) / kTile * kTile;
        const int j0 = min(total, part * per), j1 = min(total, j0 + per);
        __syncthreads();                     // the query is in shared memory
        uint32_t qa[NT][2];
#pragma unroll
        for (int i = 0; i < D / 32; i++) {   // lane t: elements 32 i + 8 t .. + 7 are two k-steps
            const uint4 w = *reinterpret_cast<const uint4*>(qrow + 32 * i + 8 * t);
            qa[2 * i][0] = w.x; qa[2 * i][1] = w.y; qa[2 * i + 1][0] = w.z; qa[2 * i + 1][1] = w.w;
        }
        auto row_ptr = [&](const uint16_t* res, const uint16_t* fresh, int j) {
            return j < res_len ? res + res_off + static_cast<int64_t>(j) * D : fresh + new_off;
        };
        for (int base = j0 + warp * kTile; base < j1; base += kWarps * kTile) {
            uint4 kw[2][D / 32];
            int row[2];
#pragma unroll
            for (int blk = 0; blk < 2; blk++) {
                row[blk] = base + 4 * (g >> 1) + 2 * blk + (g & 1);
#pragma unroll
                for (int i = 0; i < D / 32; i++) kw[blk][i] = make_uint4(0, 0, 0, 0);
                if (row[blk] < j1) {
                    const uint16_t* kp = row_ptr(a.res_k, a.k_new, row[blk]) + 8 * t;
#pragma unroll
                    for (int i = 0; i < D / 32; i++) kw[blk][i] = *reinterpret_cast<const uint4*>(kp + 32 * i);
                }
            }
            uint32_t vw[4][NT];              // rows 4t .. 4t + 3, elements g * D / 8 .. + D / 8
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int j = base + 4 * t + i;
#pragma unroll
                for (int n = 0; n < NT; n++) vw[i][n] = 0;
                if (j < j1) {
                    const uint16_t* vp = row_ptr(a.res_v, a.v_new, j) + g * (D / 8);
#pragma unroll
                    for (int n = 0; n < NT; n += 4) {
                        const uint4 w = *reinterpret_cast<const uint4*>(vp + 2 * n);
                        vw[i][n] = w.x; vw[i][n + 1] = w.y; vw[i][n + 2] = w.z; vw[i][n + 3] = w.w;
                    }
                }
            }
            float acc[2][4];
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                if (i == 0) {
                    mma_first<BF16>(acc[0], kw[0][i].x, kw[1][i].x, kw[0][i].y, kw[1][i].y, qa[2 * i][0], qa[2 * i][1]);
                    mma_first<BF16>(acc[1], kw[0][i].z, kw[1][i].z, kw[0][i].w, kw[1][i].w, qa[2 * i + 1][0], qa[2 * i + 1][1]);
                } else {
                    mma<BF16>(acc[0], kw[0][i].x, kw[1][i].x, kw[0][i].y, kw[1][i].y, qa[2 * i][0], qa[2 * i][1]);
                    mma<BF16>(acc[1], kw[0][i].z, kw[1][i].z, kw[0][i].w, kw[1][i].w, qa[2 * i + 1][0], qa[2 * i + 1][1]);
                }
            }
            float sc[4], wt[4];
#pragma unroll
            for (int i = 0; i < 4; i++) sc[i] = row[i >> 1] < j1 ? (acc[0][i] + acc[1][i]) * a.scale_log2 : -INFINITY;
            softmax_step<NT>(sc, m, l, o);
            transpose_weights(sc, wt, g, t);
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int blk = 0; blk < 2; blk++) {
                split_pair<BF16, FEW>(wt[2 * blk], wt[2 * blk + 1], keep_lo, keep_hi, hi[blk], lo[blk]);
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint32_t a0 = __byte_perm(vw[0][n], vw[1][n], 0x5410), a1 = __byte_perm(vw[0][n], vw[1][n], 0x7632);
                const uint32_t a2 = __byte_perm(vw[2][n], vw[3][n], 0x5410), a3 = __byte_perm(vw[2][n], vw[3][n], 0x7632);
                mma<BF16>(o[n], a0, a1, a2, a3, hi[0], hi[1]);
                if (!FEW) mma<BF16>(o[n], a0, a1, a2, a3, lo[0], lo[1]);
            }
        }
    }

    // ---- merge the warps (log-sum-exp) and write this split's partial ----
    __syncthreads();   // the rings are idle: they hold the warps' outputs now
    float (*s_o)[kHeads][D + 4] = reinterpret_cast<float (*)[kHeads][D + 4]>(s_ring);
#pragma unroll
    for (int e = 0; e < 2; e++) {
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) l[e] += __shfl_xor_sync(0xFFFFFFFFu, l[e], off);
        if (g == 0) { s_ml[warp][2 * t + e][0] = m[e]; s_ml[warp][2 * t + e][1] = l[e]; }
    }
#pragma unroll
    for (int i = 0; i < NT; i++) {
        if (FEW)   // columns h and h + 4 are the two halves of head h's weights
#pragma unroll
            for (int e = 0; e < 4; e++) o[i][e] += __shfl_xor_sync(0xFFFFFFFFu, o[i][e], 2);
        // this lane's elements (d, d + 1) of the tile, for heads 2t and 2t + 1
        const int d = split < a.n_store_split ? 16 * i + 2 * g : g * (D / 8) + 2 * i;
        *reinterpret_cast<float2*>(&s_o[warp][2 * t][d]) = make_float2(o[i][0], o[i][2]);
        *reinterpret_cast<float2*>(&s_o[warp][2 * t + 1][d]) = make_float2(o[i][1], o[i][3]);
    }
    __syncthreads();
    for (int e = tid; e < n_heads * D; e += kThreads) {
        const int head = e / D, d = e % D;
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < kWarps; i++) mx = fmaxf(mx, s_ml[i][head][0]);
        float acc = 0.0f, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kWarps; i++) {
            const float mi = s_ml[i][head][0], li = s_ml[i][head][1];
            if (mi == -INFINITY && li == 0.0f) continue;   // a warp without rows
            const float f = exp2f(mi - mx);
            acc += s_o[i][head][d] * f;
            sum += li * f;
        }
        if (a.out == nullptr && a.cluster == 1) {
            const int64_t slot = (prob * a.group + g0 + head) * a.n_split + split;
            a.part_acc[slot * D + d] = acc;
            if (d == 0) { a.part_ml[2 * slot] = mx; a.part_ml[2 * slot + 1] = sum; }
        } else {
            s_o[0][head][d] = acc;           // the element this thread has just read is free
            if (d == 0) { s_sum[head][0] = mx; s_sum[head][1] = sum; }
        }
    }
    if (a.out == nullptr && a.cluster == 1) return;

    // ---- merge the CTAs of the cluster through distributed shared memory, each a share of the elements ----
    cg::cluster_group cluster = cg::this_cluster();
    if (a.cluster > 1) cluster.sync();
    else __syncthreads();
    const int n_part = a.n_split / a.cluster, part = split / a.cluster;
    for (int e = (split % a.cluster) * kThreads + tid; e < n_heads * D; e += a.cluster * kThreads) {
        const int head = e / D, d = e % D;
        // everything the other CTAs hold is requested before any of it is used; a CTA without rows has zeros
        float mr[kMaxCluster], lr[kMaxCluster], ar[kMaxCluster];
#pragma unroll
        for (int r = 0; r < kMaxCluster; r++) {
            if (r < a.cluster) {
                const float* ml = cluster.map_shared_rank(&s_sum[0][0], r);
                mr[r] = ml[2 * head];
                lr[r] = ml[2 * head + 1];
                ar[r] = cluster.map_shared_rank(&s_o[0][0][0], r)[head * (D + 4) + d];
            } else {
                mr[r] = -INFINITY; lr[r] = 0.0f; ar[r] = 0.0f;
            }
        }
        float mx = mr[0];
#pragma unroll
        for (int r = 1; r < kMaxCluster; r++) mx = fmaxf(mx, mr[r]);
        float acc = 0.0f, sum = 0.0f;
#pragma unroll
        for (int r = 0; r < kMaxCluster; r++) {
            const float f = mr[r] == -INFINITY && lr[r] == 0.0f ? 0.0f : exp2f(mr[r] - mx);
            acc = fmaf(ar[r], f, acc);
            sum = fmaf(lr[r], f, sum);
        }
        const int64_t row = prob * a.group + g0 + head;
        if (a.out != nullptr) {
            const bool some = !(sum <= 0.0f);   // a NaN stays a NaN; nothing to attend over gives 0
            a.out[row * D + d] = float_to_elem<DT>(some ? acc / sum : 0.0f);
            if (d == 0 && a.out_lse != nullptr) a.out_lse[row] = some ? (mx + log2f(sum)) * 0.6931471805599453f : -INFINITY;
        } else {
            const int64_t slot = row * n_part + part;
            a.part_acc[slot * D + d] = acc;
            if (d == 0) { a.part_ml[2 * slot] = mx; a.part_ml[2 * slot + 1] = sum; }
        }
    }
    if (a.cluster > 1) cluster.sync();   // nobody leaves while its shared memory is being read
}

constexpr int kMaxSplits = 256;

// Merge of n_part partials per row into the output: grid = (rows, D / 64), a CTA has 64 elements of a row, 16 lanes of four
// elements by 16 groups of parts.
constexpr int kMergeThreads = 256;

template <int DT>
__global__ void __launch_bounds__(kMergeThreads)
q4_merge_kernel(const float* __restrict__ part_acc, const float* __restrict__ part_ml, int n_part, int dim,
                uint16_t* __restrict__ out, float* __restrict__ out_lse) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float s_w[kMaxSplits];
    __shared__ float s_red[2][kMergeThreads / 32];
    __shared__ __align__(16) float4 s_acc[16][16];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = tid & 15, grp = tid >> 4;
    // thread i has part i: its (reference, sum)
    const float2 ml = tid < n_part ? reinterpret_cast<const float2*>(part_ml)[row * n_part + tid] : make_float2(-INFINITY, 0.0f);
    const bool has = !(ml.x == -INFINITY && ml.y == 0.0f);
    float mx = ml.x;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, off));
    if (lane == 0) s_red[0][warp] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMergeThreads / 32; i++) mx = fmaxf(mx, s_red[0][i]);
    const float w = has ? exp2f(ml.x - mx) : 0.0f;
    if (tid < n_part) s_w[tid] = w;
    float sum = has ? ml.y * w : 0.0f;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
    if (lane == 0) s_red[1][warp] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kMergeThreads / 32; i++) sum += s_red[1][i];
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float* src = part_acc + (row * n_part) * dim + blockIdx.y * 64 + 4 * c;
#pragma unroll 4
    for (int i = grp; i < n_part; i += 16) {
        const float4 v = *reinterpret_cast<const float4*>(src + static_cast<int64_t>(i) * dim);
        const float f = s_w[i];
        if (f == 0.0f) continue;   // an empty partial, or one that does not count
        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
    }
    s_acc[grp][c] = acc;
    __syncthreads();
    if (tid < 64) {
        const float* col = reinterpret_cast<const float*>(s_acc) + tid;
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) v += col[64 * i];
        const bool some = !(sum <= 0.0f);   // a NaN stays a NaN; nothing to attend over gives 0
        out[row * dim + blockIdx.y * 64 + tid] = float_to_elem<DT>(some ? v / sum : 0.0f);
        if (tid == 0 && blockIdx.y == 0 && out_lse != nullptr)
            out_lse[row] = some ? (mx + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    }
}

template <int DT, int D, bool FEW, bool IDS>
int launch_one(const Args& a, dim3 grid, cudaStream_t stream) {
    static PerDeviceOnce once;   // > 48 KB of dynamic shared memory needs an opt-in per kernel and device
    int rc = once.run([](int) {
        DC_CUDA_TRY(cudaFuncSetAttribute(q4_attend_kernel<DT, D, FEW, IDS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(attend_smem_bytes<D>())));
        return DC_OK;
    });
    if (rc != DC_OK) return rc;
    DC_CUDA_TRY(launch_chained(q4_attend_kernel<DT, D, FEW, IDS>, grid, dim3(kThreads), attend_smem_bytes<D>(), stream,
                               a.cluster > 1 ? static_cast<unsigned>(a.cluster) : 0u, a));
    return DC_OK;
}

template <int DT, int D>
int launch(const Args& a, bool few, bool ids, dim3 grid, cudaStream_t stream) {
    if (few) return ids ? launch_one<DT, D, true, true>(a, grid, stream) : launch_one<DT, D, true, false>(a, grid, stream);
    return ids ? launch_one<DT, D, false, true>(a, grid, stream) : launch_one<DT, D, false, false>(a, grid, stream);
}

// CTAs per problem (and chunk of 8 heads).  A 16-bit row costs as much as 2.7 consecutive store rows or 1.6 gathered ones
// (115, 42 and 70 ps measured at head_dim 128); every kind of row that occurs gets at least one CTA.
//
// Up to 8 CTAs of a problem are a cluster that merges its results on chip and finishes the output, in one launch; that is
// taken when 8 CTAs per problem fill the SMs, or when the rows are so few that more CTAs would save less than the second
// launch costs (4096 rows of 8 problems: 10.7 us in one launch, 12.4 in two; 8192 rows 14.0 either way).  Otherwise every
// CTA writes a partial for a merge kernel: one wave of the CTAs that fit.  With sequences of unequal length a CTA takes a
// run of the same length whatever its sequence (shares of each sequence took 66 us instead of 52 on 64 problems of 0 to
// 32768 rows), runs behind a sequence's end exit at once, and there are two waves of them (one: 65 us), up to eight as long
// as a run keeps 2048 rows (128 problems of 0 to 131072 rows: 405 us with two, 336 with eight).  Clusters
// of 8 in those launches as well would merge on chip first, but do not fill every SM: 4 x 65536 rows of head_dim 256 took
// 54 us with them, 36 without.
struct Split { int store, total, cluster; int64_t run; };
constexpr int kFewUnits = 12;     // per CTA of a cluster: 768 rows
constexpr int kMaxWaves = 8;
constexpr int kWaveUnits = 32;    // 2048 rows

Split splits(int n_prob, int chunks, int head_dim, bool ids, bool ragged, int64_t store_rows, int64_t res_rows) {
    const int64_t problems = std::max<int64_t>(1, static_cast<int64_t>(n_prob) * chunks);
    int64_t target = std::max<int64_t>(1, static_cast<int64_t>(ctas_per_sm(head_dim)) * sm_count() / problems);
    const int64_t w_store = (store_rows + 63) / 64, w_res = ((ids ? 16 : 27) * res_rows + 639) / 640;   // units of 64 store rows
    const int64_t units = std::max<int64_t>(1, w_store + w_res);
    const bool one = (target <= kMaxCluster && !ragged) || units <= kMaxCluster * kFewUnits;
    if (ragged && !one) {
        const int64_t waves = std::max<int64_t>(2, std::min<int64_t>(kMaxWaves, units / target / kWaveUnits));
        target = std::min(waves * target, (units + 3) / 4);
    }
    int64_t total = std::min(std::min(target, units), static_cast<int64_t>(one ? kMaxCluster : kMaxSplits));
    if (w_store > 0 && w_res > 0) total = std::max<int64_t>(total, 2);
    total = std::max<int64_t>(total, 1);
    int64_t store = total;
    if (w_store + w_res > 0) store = (total * w_store + (w_store + w_res) / 2) / (w_store + w_res);
    if (w_store > 0) store = std::max<int64_t>(store, 1);
    if (w_res > 0) store = std::min(store, total - 1);
    return {static_cast<int>(store), static_cast<int>(total), total <= kMaxCluster ? static_cast<int>(total) : 1,
            ragged && total > kMaxCluster ? ((store_rows + store - 1) / store + kTile - 1) / kTile * kTile : 0};
}

}  // namespace

int64_t q4_attend_scratch_bytes(int n_prob, int group, int head_dim) {
    // at most kMaxWaves waves of CTAs, one cluster per problem where a wave has fewer, kMaxSplits per problem
    const int64_t parts = std::min<int64_t>(static_cast<int64_t>(n_prob) * kMaxSplits,
                                            static_cast<int64_t>(kMaxWaves) * ctas_per_sm(head_dim) * sm_count() + n_prob);
    return parts * group * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
}

int q4_attend(const Q4Attend& in, cudaStream_t stream) {
    DC_REQUIRE(in.q != nullptr && in.scratch != nullptr, "q4_attend: null q/scratch");
    DC_REQUIRE(in.n_prob >= 0 && in.n_prob <= 65535 && in.kv_heads >= 1 && in.n_prob % in.kv_heads == 0,
               "q4_attend: n_prob=%d must be a multiple of kv_heads=%d", in.n_prob, in.kv_heads);
    DC_REQUIRE(in.group >= 1 && in.group <= 64, "q4_attend: group=%d", in.group);
    DC_REQUIRE(in.res_len >= 0, "q4_attend: negative length");
    DC_REQUIRE(in.n_sel <= 0 || (in.sel != nullptr && in.sel_stride >= in.n_sel), "q4_attend: n_sel=%d without ids, or sel_stride=%lld",
               in.n_sel, static_cast<long long>(in.sel_stride));
    DC_REQUIRE(in.sel_base >= 0 && in.sel_base + in.n_rows < (1ll << 32), "q4_attend: sel_base=%lld: ids are 32 bits",
               static_cast<long long>(in.sel_base));
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
    const int chunks = (in.group + kHeads - 1) / kHeads;
    // the exchanges and callers of partials take the merge of attend.cu, which reads every partial: no empty runs there
    const bool own_merge = in.out != nullptr && in.xout == nullptr && in.fin == nullptr;
    const Split sp = splits(in.n_prob, chunks, in.head_dim, in.n_sel >= 0, own_merge && in.n_sel < 0 && in.lens != nullptr,
                            in.n_sel < 0 ? in.n_rows : in.n_sel, in.res_len + (in.k_new ? 1 : 0));
    const int n_part = sp.total / sp.cluster;
    const bool finish = n_part == 1 && own_merge;
    a.n_store_split = sp.store;
    a.n_split = sp.total;
    a.cluster = sp.cluster;
    a.run = sp.run;
    a.out = finish ? static_cast<uint16_t*>(in.out) : nullptr;
    a.out_lse = in.out_lse;
    DC_REQUIRE(finish || static_cast<int64_t>(in.n_prob) * n_part * in.group * (in.head_dim + 2) * 4 <=
                             q4_attend_scratch_bytes(in.n_prob, in.group, in.head_dim),
               "q4_attend: %d partials per problem exceed the scratch buffer", n_part);
    a.part_acc = static_cast<float*>(in.scratch);
    a.part_ml = a.part_acc + static_cast<int64_t>(in.n_prob) * n_part * in.group * in.head_dim;
    const dim3 grid(static_cast<unsigned>(a.n_split), static_cast<unsigned>(in.n_prob),
                    static_cast<unsigned>(chunks));
#define CASE(DT, D) rc = launch<DT, D>(a, in.group <= 4, in.n_sel >= 0, grid, stream)
    int rc = DC_OK;
    if (in.dtype == DC_BF16) {
        if (in.head_dim == 64) { CASE(DC_BF16, 64); }
        else if (in.head_dim == 128) { CASE(DC_BF16, 128); }
        else { CASE(DC_BF16, 256); }
    } else {
        if (in.head_dim == 64) { CASE(DC_FP16, 64); }
        else if (in.head_dim == 128) { CASE(DC_FP16, 128); }
        else { CASE(DC_FP16, 256); }
    }
#undef CASE
    if (rc != DC_OK || finish) return rc;
    if (own_merge) {
        const dim3 merge(static_cast<unsigned>(in.n_prob * in.group), static_cast<unsigned>(in.head_dim / 64));
        if (in.dtype == DC_BF16)
            DC_CUDA_TRY(launch_chained(q4_merge_kernel<DC_BF16>, merge, dim3(kMergeThreads), 0, stream, 0u, a.part_acc, a.part_ml,
                                       n_part, in.head_dim, static_cast<uint16_t*>(in.out), in.out_lse));
        else
            DC_CUDA_TRY(launch_chained(q4_merge_kernel<DC_FP16>, merge, dim3(kMergeThreads), 0, stream, 0u, a.part_acc, a.part_ml,
                                       n_part, in.head_dim, static_cast<uint16_t*>(in.out), in.out_lse));
        return DC_OK;
    }
    return lse_combine(a.part_acc, in.head_dim, static_cast<int64_t>(n_part) * in.head_dim, a.part_ml, 2,
                       static_cast<int64_t>(n_part) * 2, n_part, static_cast<int64_t>(in.n_prob) * in.group, in.head_dim,
                       in.dtype, in.out, in.out_lse, in.out_acc, in.out_ml, stream, nullptr, in.xout, in.fin, true);
}

}  // namespace dc
