// jk_attention.hpp -- attention of a step's queries over the paged 8-bit cache: what its two kernels (jk_attention.hip,
// jk_attention_prompt.hip) share.
//
// Notation: a column is one (query token, query head) pair of a kv head's group; the columns of a request
// and kv head are numbered token-major, c = token * group + head of the group.
//
// One pass over the keys with a running maximum m and sum l per column:
//   s_j = scale q.k_j,  p_j = exp(s_j - m),  l = sum p_j,  o = sum p_j v_j / l
// with k_j = ks * codes and v_j = vs * codes, ks and vs one number per page and head. The products run on f16
// matrix instructions: codes are exact in f16, ks multiplies the finished score, and vs joins the
// probability: w_j = p_j vs / r with r the largest vs so far of the pages that the column sees, so that w_j stays in f16's range
// whatever the values' size, and no page that is hidden from a column costs its weights their bits; o is rescaled by r like by m. Scores are computed transposed (rows = tokens), so a lane that holds a column's
// scores of four consecutive tokens holds them just as the second product's operand wants them: the order
// of the tokens inside a matrix instruction is free as long as both of its operands agree on it.
#pragma once

#include "jk_device.hpp"

namespace jk {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_inff();
constexpr int kCodeShift = 9;  // a code becomes code / 2^9 in f16 (code_pair)
constexpr float kCodeScale = 1 << kCodeShift;
constexpr float kLog2e = 1.44269504088896340736f;
// Queries are held in f16 with their row's largest value near 2^14, so that what is 2^-28 of it is still a normal number and
// the low parts of f32 ones keep their bits.
// The maximum that weights are taken against is a reference that moves only when a tile's scores pass it by kSlack powers of
// two, and so is the largest value scale, by a factor of kSlackV: almost no tile has to rescale the outputs, or to find
// its maximum across lanes. Weights are p_j vs / r times kWeight: at most 16 * 2^8 * 8 = 2^15, which f16 holds, and what is
// 2^-18 of the reference is still a normal number.
constexpr float kSlack = 8.0f, kSlackV = 8.0f, kWeight = 16.0f;
// The value scale that weights are taken against is at least this, so that kWeight / r is finite: the smallest scale that
// the append stores is above 2^-126 and still gives weights of 2^-2 p.
constexpr float kLeastV = 0x1p-120f;

struct AttnDev {
    const void *q;
    void *out;
    size_t qt, qh, ot, oh;  // strides in elements
    bool q_vec, out_vec;
    int n_tokens, n_heads, n_kv, grp, hd, page_shift, n_pages, max_pages, n_requests, max_new;
    const int32_t *q_start, *lens, *table;
    const int8_t *k, *v;
    const float *ks, *vs;
    float scale_log2;  // scale * log2(e)
    int window;        // INT_MAX: none
    int tile_cols, tiles;  // columns a workgroup takes, column tiles of a request
    int splits, chunk;     // workgroups that share a tile's keys, and how many keys each takes
    // requests of at most few_cols columns are the rows kernel's, the others the prompt kernel's (each launch sees all requests);
    // the joining launch needs both kernels' tiles and splits
    int few_cols, few_splits, few_chunk, many_cols, many_splits, many_chunk;
    int pitch;       // splits that the parts of a row have room for
    float *part_o;   // [n_tokens * n_heads][pitch][hd]: sums over a split, not yet divided by l
    float2 *part_ml;  // [n_tokens * n_heads][pitch]: m (in powers of two) and l
};

// The tokens of a request in the step, [first, last) of q, and the length of its cache, as far as the arrays go.
struct Req {
    int first, count, len;
};
__device__ __forceinline__ Req request_of(const AttnDev &a, int r) {
    Req q;
    q.first = min(max(a.q_start[r], 0), a.n_tokens);
    q.count = min(max(a.q_start[r + 1], q.first), a.n_tokens) - q.first;
    q.len = (int)min((long)max(a.lens[r], 0), (long)a.max_pages << a.page_shift);
    return q;
}

// The keys that columns [c0, c1) of a request can see, [lo, hi) with lo a multiple of 64, cut into pieces of
// `chunk` (a multiple of 128): the plan's, or longer ones where more than `splits` pieces would be needed.
constexpr int kMaxSplits = 256;
// Tokens of a request end so far below 2^31 that what is added to their numbers (tiles ahead, roundings) stays an int.
constexpr size_t kMaxTokens = ((size_t)1 << 31) - 4096;
struct Span {
    int lo, hi, chunk, active;
};
__device__ __forceinline__ Span span_of(const AttnDev &a, const Req &q, int c0, int c1) {
    Span s;
    const int p0 = q.len - q.count + c0 / a.grp, p1 = q.len - q.count + (c1 - 1) / a.grp;
    s.lo = max(p0 < a.window ? 0 : p0 - a.window + 1, 0) & ~63;
    s.hi = max(min(q.len, p1 + 1), s.lo);
    const int n = s.hi - s.lo;
    s.chunk = max(a.chunk, ((n + a.splits - 1) / a.splits + 127) & ~127);
    s.active = max(1, (int)(((unsigned)n + s.chunk - 1) / s.chunk));
    return s;
}
// The end of the piece that begins at `begin`.
__device__ __forceinline__ int piece_end(const Span &s, int begin) { return s.hi - begin > s.chunk ? begin + s.chunk : s.hi; }

// Two biased codes (code + 128 in the low byte of each half) as f16 pair code / 512: a half 0x00bb is the
// subnormal bb * 2^-24, and bb * 2^-24 * 2^15 - 128 / 512 = code / 512 exactly.
__device__ __forceinline__ f16x2 code_pair(uint32_t halves) {
    const f16x2 x = __builtin_bit_cast(f16x2, halves);
    const f16x2 up = {(_Float16)32768.0f, (_Float16)32768.0f}, bias = {(_Float16)-0.25f, (_Float16)-0.25f};
    return __builtin_elementwise_fma(x, up, bias);
}
__device__ __forceinline__ f16x8 codes8(uint32_t w0, uint32_t w1) {
    union {
        f16x2 p[4];
        f16x8 v;
    } u;
    w0 ^= 0x80808080u;
    w1 ^= 0x80808080u;
    u.p[0] = code_pair(__builtin_amdgcn_perm(0u, w0, 0x0c010c00u));
    u.p[1] = code_pair(__builtin_amdgcn_perm(0u, w0, 0x0c030c02u));
    u.p[2] = code_pair(__builtin_amdgcn_perm(0u, w1, 0x0c010c00u));
    u.p[3] = code_pair(__builtin_amdgcn_perm(0u, w1, 0x0c030c02u));
    return u.v;
}
// Byte b of eight dwords (biased already): the codes of one channel of eight tokens.
__device__ __forceinline__ f16x8 codes_across(const uint32_t *w, int b) {
    union {
        f16x2 p[4];
        f16x8 v;
    } u;
    const uint32_t sel = 0x0c000c00u | (uint32_t)((4 + b) << 16) | (uint32_t)b;
#pragma unroll
    for (int i = 0; i < 4; ++i) u.p[i] = code_pair(__builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], sel));
    return u.v;
}

// Maximum over the four lanes of a column (lanes 16 apart).
__device__ __forceinline__ float max_rows(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Eight f32 values as f16 (PARTS 1), or as two f16 that add up to 22 bits of them. One part for 16-bit types: a weight is then off
// by up to 2^-11 of itself, as much as an f16 output by its own rounding (an eighth of a bf16 one's), and a second part would double the
// matrix instructions of the second product. The low part is taken from the very
// number that the high part became: the empty asm keeps the compiler from converting y a second time with another
// instruction, which was seen to round some values to the other neighbour.
template <int PARTS>
__device__ __forceinline__ void split_f16(const float *y, f16x8 *out) {
    union {
        f16x8 v;
        uint32_t w[4];
    } hi;
#pragma unroll
    for (int i = 0; i < 8; ++i) hi.v[i] = (_Float16)y[i];
    if constexpr (PARTS == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("" : "+v"(hi.w[i]));
#pragma unroll
        for (int i = 0; i < 8; ++i) out[1][i] = (_Float16)(y[i] - (float)hi.v[i]);
    }
    out[0] = hi.v;
}

// Maximum and sum over the two lanes of a column (lanes 32 apart).
__device__ __forceinline__ float max_halves(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Byte offsets of the 16-byte pieces in a row of the LDS tiles, swizzled so that the lanes that read (or write) one piece
// each of neighbouring rows meet different banks: keys by the token, values by the channel and the channel / 8 (their
// writers hold every fourth channel).
template <int HDP>
__device__ __forceinline__ int swz_k(int piece, int token) {
    return (piece ^ (token & (HDP / 8 - 1))) * 16;
}
__device__ __forceinline__ int swz_v(int piece, int channel) { return (piece ^ ((channel ^ (channel >> 3)) & 7)) * 16; }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Power of two that brings a row whose largest |value| is m to [2^13, 2^14) (zeros, infinities and NaN: any).
__device__ __forceinline__ int range_shift(float m) { return 140 - (int)((__float_as_uint(m) >> 23) & 255u); }

// The launch of the prompt kernel for the plan that d holds (dtype: jk_dtype; tile_cols 128, or 256 for up to 128 channels).
jk_status launch_attn_prompt(hipStream_t s, int dtype, const AttnDev &d);

}  // namespace jk
