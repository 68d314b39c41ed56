// A store held in 4 bits: row format and device helpers (kernels in quant.cu, scan_q4.cu, attend_q4.cu).
//
// Every 32 consecutive elements of a row form a group with one scale s of the element type:
//   s = min(round_to_type(max|x| / 7), largest s whose 7-fold is finite); s < 2^-126 is stored as 0;
//   a group that holds a NaN or an infinity gets s = NaN;
//   c = clamp(round_half_even(x / s), -7, 7), 0 where s is 0 or NaN;  x is read back as s * c.
// codes:  head_dim / 2 bytes per row, two codes to a byte, each as the nibble c + 8 (1..15);
// scales: head_dim / 32 elements per row.  Both arrays are dense over (problem, row).
//
// Order of the codes inside a row, chosen so that a lane's share of a row is contiguous in BOTH roles of a
// tensor-core fragment and one mask yields the pairs the fragment wants.  A tile is 16 elements (half a group).
// The row is 8 chunks of head_dim / 16 bytes: chunk j holds elements (2j, 2j + 1) of every tile, one byte per
// tile, the lower element in the low nibble; inside each 32-bit word of a chunk the bytes are tiles
// 4w + {0, 2, 1, 3}, so that nibbles i and i + 4 of a word are the same element position of the two tiles of ONE
// group.  Keys: lane t of the four that share a row reads chunks 2t, 2t + 1.  Values: lane g of eight reads chunk g.
#pragma once

#include "common.cuh"

namespace dc {

constexpr int kQ4Group = 32;

struct Q4Rows {             // one tensor (keys or values) of a store
    uint8_t* codes;
    uint16_t* scales;
};
struct Q4Store {
    Q4Rows k, v;
    int64_t prob_rows;      // rows between two problems
};

inline int64_t q4_code_bytes(int head_dim) { return head_dim / 2; }
inline int64_t q4_scale_bytes(int head_dim) { return head_dim / kQ4Group * 2; }

// Largest scale whose 7-fold still rounds to a finite number of the type: 145 * 2^118 (bf16), 9352 (fp16).
template <int DT>
__device__ __forceinline__ float q4_scale_max() { return DT == DC_BF16 ? 145.0f * 332306998946228968225951765070086144.0f : 9352.0f; }

// A thread works on one tile (16 elements, 32 bytes) of a row: tile v of head_dim / 16, the threads of a row being
// consecutive lanes.  Four threads (v = 4w + x) exchange bytes so that thread x ends up with word w of chunks x and 4 + x
// (q4_word_index of both), i.e. a row leaves as full 32-byte runs.
template <int D>
__device__ __forceinline__ int q4_word_index(int v, int half) { return (4 * half + (v & 3)) * (D / 64) + (v >> 2); }

// Byte k of `word` = the pair of this thread's tile that belongs to chunk 4 * half + k; afterwards thread x holds chunk
// 4 * half + x of the four tiles, in the stored byte order.  Two exchanges.  All lanes of a warp take part.
__device__ __forceinline__ uint32_t q4_transpose_out(uint32_t word, int v) {
    uint32_t r = __shfl_xor_sync(0xFFFFFFFFu, word, 1);
    word = __byte_perm(word, r, (v & 1) ? 0x3715 : 0x6240);
    r = __shfl_xor_sync(0xFFFFFFFFu, word, 2);
    return __byte_perm(word, r, (v & 2) ? 0x3726 : 0x5140);
}
__device__ __forceinline__ uint32_t q4_transpose_in(uint32_t word, int v) {
    word = __byte_perm(word, 0u, 0x3120);
    uint32_t r = __shfl_xor_sync(0xFFFFFFFFu, word, 2);
    word = __byte_perm(word, r, (v & 2) ? 0x3276 : 0x5410);
    r = __shfl_xor_sync(0xFFFFFFFFu, word, 1);
    return __byte_perm(word, r, (v & 1) ? 0x3715 : 0x6240);
}

// The scale of a group from its largest magnitude bits (of the element type); `inv` is about 1 / scale, 0 where the codes
// are all zero.  max|x| / 7 is never nearer than 2^-15 (relative) to a midpoint between two numbers of the type, so one
// fp32 product rounds to the same scale as the exact quotient.
template <int DT>
__device__ __forceinline__ uint16_t q4_scale(uint32_t top_bits, float& inv) {
    inv = 0.0f;
    if (top_bits >= (DT == DC_BF16 ? 0x7F80u : 0x7C00u)) return 0x7FFF;   // a NaN or an infinity in the group
    const float top = elem_to_float<DT>(static_cast<uint16_t>(top_bits));
    const uint16_t sb = float_to_elem<DT>(fminf(top * (1.0f / 7.0f), q4_scale_max<DT>()));
    const float s = elem_to_float<DT>(sb);
    if (s < 1.17549435e-38f) return 0;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(inv) : "f"(s));
    return sb;
}

// Eight elements -> their eight nibbles (c + 8), element i in bits 4i.
//
// The quotient is rounded exactly as defined without a division per element: x / s is either exactly a half-integer
// or at least 2^-12 away from one (x and s have at most 11 significant bits), x * inv is off by less than 2^-19,
// and fma(x, inv, 1536) rounds to a multiple of 2^-13: a tie lands exactly on the half-integer, nothing else does.
// The second addition then rounds half to even (1.5 * 2^23 + 8 is even), leaving c + 8 in the low bits.
template <int DT>
__device__ __forceinline__ uint32_t q4_codes8(const uint4& w, float inv) {
    float f[8];
    unpack8<DT>(w, f);
    uint32_t word = 0, bias = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float t = fmaf(f[i], inv, 1536.0f);
        if (DT == DC_FP16) t = fminf(fmaxf(t, 1529.0f), 1543.0f);   // a subnormal scale can be off by up to a half
        word += __float_as_uint(t + (12582920.0f - 1536.0f)) << (4 * i);
        bias += 0x4B400000u << (4 * i);                             // the bits of 1.5 * 2^23, in every term
    }
    return word - bias;
}

// One tile -> the two code words this thread stores (chunks x and 4 + x) and its group's scale.  All lanes take part.
template <int DT>
__device__ __forceinline__ void q4_encode(const uint4 (&w)[2], int v, uint32_t (&word)[2], uint16_t& scale) {
    const uint32_t kAbs = 0x7FFF7FFFu;
    uint32_t m = __vmaxu2(__vmaxu2(__vmaxu2(w[0].x & kAbs, w[0].y & kAbs), __vmaxu2(w[0].z & kAbs, w[0].w & kAbs)),
                          __vmaxu2(__vmaxu2(w[1].x & kAbs, w[1].y & kAbs), __vmaxu2(w[1].z & kAbs, w[1].w & kAbs)));
    m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));   // magnitude bits order like magnitudes; NaN and inf on top
    m = max(m & 0xFFFFu, m >> 16);
    float inv;
    scale = q4_scale<DT>(m, inv);
    // a group whose codes are all zero must not multiply (0 * inf): its elements are replaced by zeros
    const bool live = inv != 0.0f;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t c = q4_codes8<DT>(w[h], inv);
        word[h] = q4_transpose_out(live ? c : 0x88888888u, v);
    }
}

// The inverse: the two code words and the group's scale -> the tile, s * c rounded once (a packed 16-bit product of exact
// operands rounds the exact result).
template <int DT>
__device__ __forceinline__ void q4_decode(const uint32_t (&word)[2], uint16_t scale, int v, uint4 (&out)[2]) {
    const uint32_t s2 = scale * 0x10001u;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t w = q4_transpose_in(word[h], v);   // byte k: elements (2k, 2k + 1) of this half tile
        const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t pair = __byte_perm(lo, hi, k * 0x0011 + (4 + k) * 0x1100) & 0x000F000Fu;
            if (DT == DC_BF16) {
                uint32_t c;
                asm("sub.bf16x2 %0, %1, %2;\n" : "=r"(c) : "r"(pair | 0x43004300u), "r"(0x43084308u));
                asm("mul.rn.bf16x2 %0, %1, %2;\n" : "=r"(o[k]) : "r"(c), "r"(s2));
            } else {
                uint32_t c;
                asm("sub.f16x2 %0, %1, %2;\n" : "=r"(c) : "r"(pair | 0x64006400u), "r"(0x64086408u));
                asm("mul.rn.f16x2 %0, %1, %2;\n" : "=r"(o[k]) : "r"(c), "r"(s2));
            }
        }
        out[h] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// ---- host side (quant.cu, scan_q4.cu, attend_q4.cu) ----
struct XchgOut;
struct XchgFinal;

// what happens to the device word that counts the valid rows, once rows [row0, row0 + n) are written
enum { kLenKeep = 0, kLenSet = 1, kLenMax = 2 };

int q4_write_rows(const void* keys, const void* vals, int64_t stride_b, int64_t stride_h, int64_t stride_s, int n_prob,
                  int kv_heads, int64_t n, int head_dim, int dtype, const Q4Store& st, int64_t row0, int32_t* len,
                  int len_mode, cudaStream_t stream);
int q4_append_rows(const void* keys, const void* vals, int n_prob, int head_dim, int dtype, const Q4Store& st,
                   int64_t max_rows, int32_t* len, uint32_t* status, cudaStream_t stream);
int q4_window_push(const void* k_new, const void* v_new, int64_t new_stride_b, void* res_k, void* res_v,
                   int64_t res_stride_b, int64_t res_stride_h, int n_prob, int kv_heads, int head_dim, int dtype,
                   const Q4Store& st, int64_t max_rows, int32_t* len, int32_t* win, uint32_t* status, cudaStream_t stream);
// out[p][i] = row ids[p][i] (ids given) or row row0 + i; rows outside [0, *n_dev or n_rows) are zeros.  Either output
// may be NULL.  f32: fp32 outputs instead of the element type.
int q4_read_rows(const Q4Store& st, int64_t n_rows, const int32_t* n_dev, int n_prob, int head_dim, int dtype, int64_t row0,
                 const uint32_t* ids, int64_t ids_stride, int64_t n, void* out_k, void* out_v, bool f32, cudaStream_t stream);
int q4_score_scan(const Q4Rows& keys, int64_t prob_rows, int n_prob, int64_t n, int head_dim, int dtype, const void* q,
                  int q_mode, int group, uint32_t* scores, int64_t score_stride, uint32_t* minmax, cudaStream_t stream,
                  int kv_heads = 1, int64_t q_stride_b = 0, const int32_t* n_dev = nullptr);
struct Q4Attend {
    Q4Store st;
    int64_t n_rows;             // rows the launch is sized for; n_rows_dev overrides it when the kernel runs
    const int32_t* n_rows_dev;
    int n_prob, kv_heads, group, head_dim, dtype;
    const void* q;
    int64_t q_stride_b;
    const uint32_t* sel;        // NULL: every stored row
    int64_t sel_stride;
    int n_sel;
    int64_t sel_base;
    const int32_t* sel_count;
    const int32_t* lens;        // per batch, with sel == NULL: only the first lens[b] rows (may be NULL)
    const void* k_new;
    const void* v_new;
    int64_t new_stride_b;
    void* res_k;
    void* res_v;
    int64_t res_stride_b, res_stride_h;
    int res_len;
    const int32_t* res_len_dev;
    float scale;
    void* out;
    float* out_lse;
    float* out_acc;
    float* out_ml;
    void* scratch;
    const XchgOut* xout;
    const XchgFinal* fin;
};
int q4_attend(const Q4Attend& a, cudaStream_t stream);
int64_t q4_attend_scratch_bytes(int n_prob, int group, int head_dim);

}  // namespace dc
