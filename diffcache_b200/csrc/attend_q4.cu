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
constexpr int kHeads = 8;            // query heads of one kv head handled by one CTA (columns of the second product)
constexpr int kTile = 16;            // rows a warp takes at a time
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
    int n_store_split;               // CTAs (per problem and head chunk) that take store rows; the others take 16-bit rows
    int n_split;
    float* part_acc;                 // (n_prob, group, n_split, D)
    float* part_ml;                  // (n_prob, group, n_split, 2)
};

template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// N 32-bit words from a naturally aligned address, streamed past L1.
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&r)[N], const void* p) {
    if (N == 1) {
        asm volatile("ld.global.nc.L1::no_allocate.b32 %0, [%1];\n" : "=r"(r[0]) : "l"(p));
    } else if (N == 2) {
        asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0,%1}, [%2];\n" : "=r"(r[0]), "=r"(r[N > 1 ? 1 : 0]) : "l"(p));
    } else {
#pragma unroll
        for (int i = 0; i + 3 < N; i += 4)
            asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];\n"
                         : "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]) : "l"(static_cast<const char*>(p) + 4 * i));
    }
}

// Four pairs of codes of a word: pair j = (nibble j, nibble j + 4).  Inserting a nibble into the mantissa of 1024 (fp16) or
// 128 (bf16) makes it that number plus the nibble, exactly; the offset and the 8 of the encoding go with one operation.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t (&p)[4]) {
    const uint32_t hi = w >> 8;
    uint32_t t[4] = {(w & 0x000F000Fu) | 0x64006400u, (w & 0x00F000F0u) | 0x64006400u,
                     (hi & 0x000F000Fu) | 0x64006400u, (hi & 0x00F000F0u) | 0x64006400u};
    asm("sub.f16x2 %0, %1, %2;\n" : "=r"(p[0]) : "r"(t[0]), "r"(0x64086408u));                       // - 1032
    asm("fma.rn.f16x2 %0, %1, %2, %3;\n" : "=r"(p[1]) : "r"(t[1]), "r"(0x2C002C00u), "r"(0xD480D480u));   // / 16 - 72
    asm("sub.f16x2 %0, %1, %2;\n" : "=r"(p[2]) : "r"(t[2]), "r"(0x64086408u));
    asm("fma.rn.f16x2 %0, %1, %2, %3;\n" : "=r"(p[3]) : "r"(t[3]), "r"(0x2C002C00u), "r"(0xD480D480u));
}
__device__ __forceinline__ void codes_bf16(uint32_t w, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t t = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
        asm("sub.bf16x2 %0, %1, %2;\n" : "=r"(p[i]) : "r"(t), "r"(0x43084308u));                      // - 136
    }
}

// (x, y) rounded to a pair of 16-bit values, x in the low half; what is lost goes to a second pair.
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    uint32_t r;
    if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(y), "f"(x));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(y), "f"(x));
    return r;
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
template <int DT>
__device__ __forceinline__ float low_elem(uint32_t w) { return elem_to_float<DT>(static_cast<uint16_t>(w & 0xFFFFu)); }
template <int DT>
__device__ __forceinline__ float high_elem(uint32_t w) {
    return DT == DC_BF16 ? __uint_as_float(w & 0xFFFF0000u) : elem_to_float<DT>(static_cast<uint16_t>(w >> 16));
}

__device__ __forceinline__ float exp2_fast(float x) {   // 2^x to 2 ulp, 0 below 2^-126 and for -inf
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
    return r;
}

// Running softmax of the rows one warp has seen.  Lane (g, t) = (lane / 4, lane % 4) works for head g: x[2 * blk + e] is the
// score of row 4t + 2 blk + e of the tile (log2 units, -inf where there is no row).  On return x holds the weights
// relative to the new maximum; the return value is the factor the sums so far take.
__device__ __forceinline__ float softmax_step(float (&x)[4], float& m, float& l) {
    float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
    mx = fmaxf(fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2)), m);
    const float ref = mx == -INFINITY ? 0.0f : mx;       // nothing seen yet: every weight is 2^-inf = 0
    const float alpha = exp2_fast(m - ref);
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = exp2_fast(x[i] - ref);
    l = fmaf(l, alpha, (x[0] + x[1]) + (x[2] + x[3]));
    m = mx;
    return alpha;
}

// o columns are heads 2t, 2t + 1; their factors live in the lanes of rows g = 2t, 2t + 1.
template <int NT>
__device__ __forceinline__ void rescale(float (&o)[NT][4], float alpha, int t) {
    if (!__any_sync(0xFFFFFFFFu, alpha != 1.0f)) return;   // the maximum rarely moves after the first tiles
    const float a0 = __shfl_sync(0xFFFFFFFFu, alpha, 8 * t), a1 = __shfl_sync(0xFFFFFFFFu, alpha, 8 * t + 4);
#pragma unroll
    for (int i = 0; i < NT; i++) { o[i][0] *= a0; o[i][1] *= a1; o[i][2] *= a0; o[i][3] *= a1; }
}

// One warp's share of a tile of store rows, as loaded: lane (g, t) holds its part of the keys of rows
// 4 (g / 2) + 2 blk + g % 2 (blk = 0, 1) and of the values and scales of rows 4t .. 4t + 3.
template <int D>
struct StoreTile {
    uint32_t k[2][D / 32], v[4][D / 64], ks[4][D / 64], vs[4][D / 64];
    uint32_t ok;                     // bit i: row 4t + i is attended (tiles that may lack rows only)
};

// grid = (n_split, n_prob, ceil(group / 8)).
//
// Store rows.  S = Q K^T with m16n8k16 MMAs: the query heads are the rows of A, 8 store rows the columns of B.  The codes
// enter as small integers (fp16, exact), so a group's partial product is exact up to fp32 accumulation and its scale is
// applied once, in fp32.  The query of a head is normalised by a power of two so that a bf16 query is exact in fp16 too.
// O^T = V^T P^T: the value codes are A (16 elements of a tile x 16 rows, bf16 integers), the weights are B; a value's scale
// depends on (row, group) only, so it multiplies the weight, which then enters as a bf16 value and its remainder
// (16 bits).  With at most four heads value and remainder are two column groups of ONE MMA (columns h and h + 4),
// otherwise two MMAs.  The rows of a tile are numbered so that a lane's rows in both fragments are 4t .. 4t + 3.
// All operands go from global memory straight to registers (the stored order of the codes makes every lane's share
// contiguous), one tile ahead of the arithmetic; warps are independent until the end.
//
// 16-bit rows (resident rows, new token): the same two products on the element type, by CTAs of their own.
template <int DT, int D, bool FEW, bool IDS>
__global__ void __launch_bounds__(kThreads, D <= 128 ? 3 : 2)
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
    __shared__ __align__(16) float s_o[kWarps][kHeads][D + 4];
    __shared__ float s_ml[kWarps][kHeads][2];
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

    float m = -INFINITY, l = 0.0f;
    float o[NT][4];
#pragma unroll
    for (int i = 0; i < NT; i++) { o[i][0] = 0.0f; o[i][1] = 0.0f; o[i][2] = 0.0f; o[i][3] = 0.0f; }
    __syncthreads();

    if (split < a.n_store_split) {
        const int64_t n_rows = a.n_rows_dev != nullptr ? min(a.n_rows, static_cast<int64_t>(*a.n_rows_dev)) : a.n_rows;
        const uint32_t* sel = IDS ? a.sel + prob * a.sel_stride : nullptr;
        // rows of the store: the first sel_count ids of the list, or rows 0 .. lens[b] - 1
        int64_t n_store = IDS ? (n_rows > 0 ? a.n_sel : 0) : n_rows;
        if (IDS && a.sel_count) n_store = max(static_cast<int64_t>(0), min(n_store, static_cast<int64_t>(a.sel_count[prob])));
        if (!IDS && a.lens) n_store = max(static_cast<int64_t>(0), min(n_rows, static_cast<int64_t>(a.lens[b])));
        int64_t per = (n_store + a.n_store_split - 1) / a.n_store_split;
        per = (per + kTile - 1) / kTile * kTile;
        const int64_t j0 = min(n_store, split * per), j1 = min(n_store, j0 + per);
        const uint8_t* kc = a.st.k.codes + prob * a.st.prob_rows * (D / 2) + t * (D / 8);
        const uint8_t* vc = a.st.v.codes + prob * a.st.prob_rows * (D / 2) + g * (D / 16);
        const uint16_t* ks = a.st.k.scales + prob * a.st.prob_rows * NG;
        const uint16_t* vs = a.st.v.scales + prob * a.st.prob_rows * NG;

        // query fragments, normalised to [2^14, 2^15) by a power of two
        float top = 0.0f;
        for (int d = t; d < D; d += 4) top = fmaxf(top, fabsf(elem_to_float<DT>(qrow[d])));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        int ex = static_cast<int>((__float_as_uint(top) >> 23) & 255u);   // 0: zero or subnormal, 255: infinite
        ex = ex == 255 ? 127 + 14 : max(ex, 28);
        const float down = __uint_as_float(static_cast<uint32_t>(127 + 14 - ex + 127) << 23);   // 2^(14 - e)
        const float up = __uint_as_float(static_cast<uint32_t>(ex - 14) << 23) * a.scale_log2;    // 2^(e - 14)
        uint32_t qa[NT][2];
#pragma unroll
        for (int w = 0; w < D / 64; w++)
#pragma unroll
            for (int gp = 0; gp < 2; gp++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int d = 16 * (4 * w + 2 * gp) + 2 * (2 * t + c);   // a tile's element; + 16 is the group's other tile
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        qa[4 * w + 2 * gp + c][e] = pack2<false>(elem_to_float<DT>(qrow[d + e]) * down,
                                                                 elem_to_float<DT>(qrow[d + 16 + e]) * down);
                }

        // A whole tile of consecutive rows: every address is a lane constant plus the first row.
        auto load_run = [&](StoreTile<D>& x, int64_t row0) {
            const uint8_t* kp = kc + (row0 + 4 * (g >> 1) + (g & 1)) * (D / 2);
            const uint8_t* vp = vc + (row0 + 4 * t) * (D / 2);
            const uint16_t* ksp = ks + (row0 + 4 * t) * NG;
            const uint16_t* vsp = vs + (row0 + 4 * t) * NG;
            load_words<D / 32>(x.k[0], kp);
            load_words<D / 32>(x.k[1], kp + D);
#pragma unroll
            for (int i = 0; i < 4; i++) load_words<D / 64>(x.ks[i], ksp + i * NG);
#pragma unroll
            for (int i = 0; i < 4; i++) load_words<D / 64>(x.v[i], vp + i * (D / 2));
#pragma unroll
            for (int i = 0; i < 4; i++) load_words<D / 64>(x.vs[i], vsp + i * NG);
        };
        // This lane's row of a tile's 16 (lane and lane + 16 hold the same); -1 where there is none.
        auto fetch_id = [&](int64_t base) -> int32_t {
            const int64_t j = base + (lane & 15);
            if (j >= j1) return -1;
            if (!IDS) return static_cast<int32_t>(j);
            const int64_t row = static_cast<int64_t>(sel[j]) - a.sel_base;
            return row >= 0 && row < n_rows ? static_cast<int32_t>(row) : -1;   // pads and ids of other shards
        };
        // Any 16 rows; where there is none, row 0 (which exists) is loaded and not used.
        auto load_any = [&](StoreTile<D>& x, int32_t id) {
            const int32_t safe = max(id, 0);
            x.ok = (__ballot_sync(0xFFFFFFFFu, id >= 0) >> (4 * t)) & 15u;
#pragma unroll
            for (int blk = 0; blk < 2; blk++) {
                const int64_t row = __shfl_sync(0xFFFFFFFFu, safe, 4 * (g >> 1) + 2 * blk + (g & 1));
                load_words<D / 32>(x.k[blk], kc + row * (D / 2));
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int64_t row = __shfl_sync(0xFFFFFFFFu, safe, 4 * t + i);
                load_words<D / 64>(x.ks[i], ks + row * NG);
                load_words<D / 64>(x.v[i], vc + row * (D / 2));
                load_words<D / 64>(x.vs[i], vs + row * NG);
            }
        };
        auto compute = [&](StoreTile<D>& x, bool whole) {
            float sc[4];
#pragma unroll
            for (int blk = 0; blk < 2; blk++) {
                float acc[NG][4];
#pragma unroll
                for (int i = 0; i < NG; i++) { acc[i][0] = 0.0f; acc[i][1] = 0.0f; acc[i][2] = 0.0f; acc[i][3] = 0.0f; }
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int w = 0; w < D / 64; w++) {
                        uint32_t p[4];
                        codes_f16(x.k[blk][c * (D / 64) + w], p);
                        mma<false>(acc[2 * w], qa[4 * w + c][0], 0u, qa[4 * w + c][1], 0u, p[0], p[1]);
                        mma<false>(acc[2 * w + 1], qa[4 * w + 2 + c][0], 0u, qa[4 * w + 2 + c][1], 0u, p[2], p[3]);
                    }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float s = 0.0f;
#pragma unroll
                    for (int w = 0; w < D / 64; w++) {
                        s = fmaf(low_elem<DT>(x.ks[2 * blk + e][w]), acc[2 * w][e], s);
                        s = fmaf(high_elem<DT>(x.ks[2 * blk + e][w]), acc[2 * w + 1][e], s);
                    }
                    sc[2 * blk + e] = s * up;
                }
            }
            if (!whole) {   // rows that are not there: no weight, and a scale of 0 in place of whatever was loaded
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (((x.ok >> i) & 1u) == 0) {
                        sc[i] = -INFINITY;
#pragma unroll
                        for (int w = 0; w < D / 64; w++) x.vs[i][w] = 0;
                    }
            }
            rescale<NT>(o, softmax_step(sc, m, l), t);
#pragma unroll
            for (int w = 0; w < D / 64; w++) {
                uint32_t hi[2][2], lo[2][2];   // [group of the word][row block]
#pragma unroll
                for (int gp = 0; gp < 2; gp++)
#pragma unroll
                    for (int blk = 0; blk < 2; blk++) {
                        const float p0 = sc[2 * blk] * (gp ? high_elem<DT>(x.vs[2 * blk][w]) : low_elem<DT>(x.vs[2 * blk][w]));
                        const float p1 = sc[2 * blk + 1] *
                                         (gp ? high_elem<DT>(x.vs[2 * blk + 1][w]) : low_elem<DT>(x.vs[2 * blk + 1][w]));
                        split_pair<true, FEW>(p0, p1, keep_lo, keep_hi, hi[gp][blk], lo[gp][blk]);
                    }
                // value codes of rows (4t, 4t + 1) and (4t + 2, 4t + 3): nibble pairs of the same element
                uint32_t va[2][2][4];
#pragma unroll
                for (int blk = 0; blk < 2; blk++) {
                    codes_bf16(__byte_perm(x.v[2 * blk][w], x.v[2 * blk + 1][w], 0x5410), va[blk][0]);   // tiles 4w, 4w + 2
                    codes_bf16(__byte_perm(x.v[2 * blk][w], x.v[2 * blk + 1][w], 0x7632), va[blk][1]);   // tiles 4w + 1, 4w + 3
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
        const int64_t step = kWarps * kTile;
        int64_t base = j0 + warp * kTile;
        if (!IDS) {
            if (D <= 128 && base + kTile <= j1) {      // one tile ahead, in two sets of registers
                StoreTile<D> x, y;
                load_run(x, base);
                while (true) {
                    if (base + step + kTile > j1) { compute(x, true); base += step; break; }
                    load_run(y, base + step);
                    compute(x, true);
                    base += step;
                    if (base + step + kTile > j1) { compute(y, true); base += step; break; }
                    load_run(x, base + step);
                    compute(y, true);
                    base += step;
                }
            }
            StoreTile<D> x;
            for (; base < j1; base += step) {          // the last tile; every tile where registers do not hold two
                const bool whole = base + kTile <= j1;
                if (whole) load_run(x, base);
                else load_any(x, fetch_id(base));
                compute(x, whole);
            }
        } else if (base < j1) {
            StoreTile<D> x, y;
            load_any(x, fetch_id(base));
            int32_t id = fetch_id(base + step);
            while (true) {
                bool more = base + step < j1;
                if (D <= 128 && more) { load_any(y, id); id = fetch_id(base + 2 * step); }
                compute(x, __all_sync(0xFFFFFFFFu, x.ok == 15u));
                if (!more) break;
                base += step;
                more = base + step < j1;
                if (D > 128) { load_any(y, id); id = fetch_id(base + step); }
                else if (more) { load_any(x, id); id = fetch_id(base + 2 * step); }
                compute(y, __all_sync(0xFFFFFFFFu, y.ok == 15u));
                if (!more) break;
                base += step;
                if (D > 128) { load_any(x, id); id = fetch_id(base + step); }
            }
        }
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
            float sc[4];
#pragma unroll
            for (int blk = 0; blk < 2; blk++) {
                const int j = base + 4 * (g >> 1) + 2 * blk + (g & 1);
                uint4 kw[D / 32];
#pragma unroll
                for (int i = 0; i < D / 32; i++) kw[i] = make_uint4(0, 0, 0, 0);
                if (j < j1) {
                    const uint16_t* kp = row_ptr(a.res_k, a.k_new, j) + 8 * t;
#pragma unroll
                    for (int i = 0; i < D / 32; i++) kw[i] = *reinterpret_cast<const uint4*>(kp + 32 * i);
                }
                float acc[2][4] = {};
#pragma unroll
                for (int i = 0; i < D / 32; i++) {
                    mma<BF16>(acc[0], qa[2 * i][0], 0u, qa[2 * i][1], 0u, kw[i].x, kw[i].y);
                    mma<BF16>(acc[1], qa[2 * i + 1][0], 0u, qa[2 * i + 1][1], 0u, kw[i].z, kw[i].w);
                }
#pragma unroll
                for (int e = 0; e < 2; e++)
                    sc[2 * blk + e] = base + 4 * t + 2 * blk + e < j1 ? (acc[0][e] + acc[1][e]) * a.scale_log2 : -INFINITY;
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
            rescale<NT>(o, softmax_step(sc, m, l), t);
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int blk = 0; blk < 2; blk++) {
                split_pair<BF16, FEW>(sc[2 * blk], sc[2 * blk + 1], keep_lo, keep_hi, hi[blk], lo[blk]);
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
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
    if (t == 0) { s_ml[warp][g][0] = m; s_ml[warp][g][1] = l; }
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
        const int64_t slot = (prob * a.group + g0 + head) * a.n_split + split;
        a.part_acc[slot * D + d] = acc;
        if (d == 0) { a.part_ml[2 * slot] = mx; a.part_ml[2 * slot + 1] = sum; }
    }
}

// CTAs per problem (and chunk of 8 heads).  One wave of three CTAs per SM; a 16-bit row counts as three store rows (its
// 512 bytes at head_dim 128 against 144); every kind of row that occurs gets at least one CTA.
constexpr int kCtasPerSm = 3;
constexpr int kMaxSplits = 256;

struct Split { int store, total; };

Split splits(int n_prob, int64_t store_rows, int64_t res_rows) {
    const int64_t target = std::max(1, kCtasPerSm * sm_count() / std::max(1, n_prob));
    const int64_t w_store = (store_rows + 63) / 64, w_res = (3 * res_rows + 63) / 64;   // units of 64 store rows
    const int64_t total = std::max<int64_t>(1, std::min<int64_t>(std::min(target, w_store + w_res), kMaxSplits - 1));
    int64_t store = 0, res = 0;
    if (w_store + w_res > 0) {
        store = w_store > 0 ? std::max<int64_t>(1, (total * w_store + (w_store + w_res) / 2) / (w_store + w_res)) : 0;
        res = w_res > 0 ? std::max<int64_t>(1, total - store) : 0;
    }
    if (store + res == 0) store = 1;
    return {static_cast<int>(store), static_cast<int>(store + res)};
}

}  // namespace

int64_t q4_attend_scratch_bytes(int n_prob, int group, int head_dim) {
    // splits() makes at most kCtasPerSm * SMs / n_prob + 1 per problem (2 where that is 0 or 1), and at most kMaxSplits
    const int64_t ctas = std::min<int64_t>(static_cast<int64_t>(n_prob) * kMaxSplits,
                                           static_cast<int64_t>(kCtasPerSm) * sm_count() + 2ll * n_prob);
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
    const Split sp = splits(in.n_prob, in.n_sel < 0 ? in.n_rows : in.n_sel, in.res_len + (in.k_new ? 1 : 0));
    a.n_store_split = sp.store;
    a.n_split = sp.total;
    a.part_acc = static_cast<float*>(in.scratch);
    a.part_ml = a.part_acc + static_cast<int64_t>(in.n_prob) * a.n_split * in.group * in.head_dim;
    const dim3 grid(static_cast<unsigned>(a.n_split), static_cast<unsigned>(in.n_prob),
                    static_cast<unsigned>((in.group + kHeads - 1) / kHeads));
#define LAUNCH(DT, D, FEW, IDS) DC_CUDA_TRY(launch_chained(q4_attend_kernel<DT, D, FEW, IDS>, grid, dim3(kThreads), 0, stream, 0u, a))
#define CASE(DT, D)                                                                                   \
    if (in.group <= 4) { if (in.n_sel < 0) LAUNCH(DT, D, true, false); else LAUNCH(DT, D, true, true); } \
    else { if (in.n_sel < 0) LAUNCH(DT, D, false, false); else LAUNCH(DT, D, false, true); }
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
#undef LAUNCH
    return lse_combine(a.part_acc, in.head_dim, static_cast<int64_t>(a.n_split) * in.head_dim, a.part_ml, 2,
                       static_cast<int64_t>(a.n_split) * 2, a.n_split, static_cast<int64_t>(in.n_prob) * in.group, in.head_dim,
                       in.dtype, in.out, in.out_lse, in.out_acc, in.out_ml, stream, nullptr, in.xout, in.fin, true);
}

}  // namespace dc
