// jk_attention.hip -- attention of a step's queries over the paged 8-bit cache.
//
// Notation: a column is one (query token, query head) pair of a kv head's group; the columns of a request
// and kv head are numbered token-major, c = token * group + head of the group.
//
// One pass over the keys with a running maximum m and sum l per column:
//   s_j = scale q.k_j,  p_j = exp(s_j - m),  l = sum p_j,  o = sum p_j v_j / l
// with k_j = ks * codes and v_j = vs * codes, ks and vs one number per page and head. The products run on f16
// matrix instructions: codes are exact in f16, ks multiplies the finished score, and vs joins the
// probability: w_j = p_j vs / r with r the largest vs so far, so that w_j <= 1 whatever the values' size (held times 2^14); o is
// rescaled by r like by m. Scores are computed transposed (rows = tokens), so a lane that holds a column's
// scores of four consecutive tokens holds them just as the second product's operand wants them: the order
// of the tokens inside a matrix instruction is free as long as both of its operands agree on it.
#include <algorithm>
#include <cmath>

#include "jk_device.hpp"

namespace jk {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_inff();
constexpr float kCodeScale = 512.0f;  // a code becomes code / 512 in f16 (code_pair)
// Queries and weights are held in f16 with their largest values near 2^14, so that what is 2^-28 of those is still a
// normal number, and the low parts of f32 ones keep their bits: weights are p_j vs / r times this.
constexpr float kWeightScale = 16384.0f;

struct AttnDev {
    const void *q;
    void *out;
    size_t qt, qh, ot, oh;  // strides in elements
    bool q_vec, out_vec;
    int n_tokens, n_heads, n_kv, grp, hd, page_shift, n_pages, max_pages, n_requests, max_new;
    const int32_t *q_start, *lens, *table;
    const int8_t *k, *v;
    const float *ks, *vs;
    float scale_log2;  // scale * log2(e) * kCodeScale
    int window;        // INT_MAX: none
    int tiles, splits;
    float *part_o;   // [n_tokens * n_heads][splits][hd]: sums over a split, not yet divided by l
    float2 *part_ml;  // [n_tokens * n_heads][splits]: m (in powers of two) and l
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

// The keys that columns [c0, c1) of a request can see, [lo, hi) with lo a multiple of 32, cut into pieces of
// `chunk` (a multiple of 128) over at most `splits` workgroups.
constexpr int kMinChunk = 256;
struct Span {
    int lo, hi, chunk, active;
};
__device__ __forceinline__ Span span_of(const AttnDev &a, const Req &q, int c0, int c1) {
    Span s;
    const int p0 = q.len - q.count + c0 / a.grp, p1 = q.len - q.count + (c1 - 1) / a.grp;
    s.lo = max(p0 < a.window ? 0 : p0 - a.window + 1, 0) & ~31;
    s.hi = max(min(q.len, p1 + 1), s.lo);
    const int n = s.hi - s.lo;
    s.chunk = max(kMinChunk, ((n + a.splits - 1) / a.splits + 127) & ~127);
    s.active = max(1, (n + s.chunk - 1) / s.chunk);
    return s;
}

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

// Eight f32 values as f16 (PARTS 1), or as two f16 that add up to 22 bits of them. The low part is taken from the very
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

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Power of two that brings a row whose largest |value| is m to [2^13, 2^14) (zeros, infinities and NaN: any).
__device__ __forceinline__ int range_shift(float m) { return 140 - (int)((__float_as_uint(m) >> 23) & 255u); }

// Up to 16 columns of one request and kv head over one split of its keys, by four waves that take 32 tokens in
// turn; their sums are joined in LDS. A lane (n = lane % 16, g = lane / 16) holds of column n: the query's
// channels 64 j + 16 g + .. as the first product's operand, the scores of tokens 4 g + i and 16 + 4 g + i, and
// of its output the channels (HDP / 16) (4 g + i) + t. Of the keys it loads row n (16 bytes at a time), of the values
// channels (HDP / 16) n + t of the eight tokens whose scores it holds, so that the loads of a wave cover whole rows
// and nothing goes through LDS.
// PARTS: f16 parts that f32 queries and probabilities are split into.
template <typename T, int HDP, int PARTS>
__global__ __launch_bounds__(256) void attn_q8_rows_kernel(AttnDev a) {
    constexpr int KJ = HDP / 64, NT = HDP / 16, VW = HDP / 64;  // VW: dwords of a value row that a lane loads
    __shared__ float s_ml[4][16][3];
    __shared__ float s_o[4][16][HDP + 4];
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = l & 15, g = l >> 4;
    unsigned id = blockIdx.x;
    const int split = id % a.splits;
    id /= a.splits;
    const int h = id % a.n_kv;
    id /= a.n_kv;
    const int ct = id % a.tiles, r = id / a.tiles;

    const Req rq = request_of(a, r);
    const int cols = min(rq.count, a.max_new) * a.grp, c0 = ct * 16;
    if (c0 >= cols) return;
    const Span sp = span_of(a, rq, c0, min(c0 + 16, cols));
    if (split >= sp.active) return;
    const int begin = sp.lo + split * sp.chunk, end = min(sp.hi, begin + sp.chunk);

    // this lane's column
    const int c = min(c0 + n, cols - 1), token = rq.first + c / a.grp, head = h * a.grp + c % a.grp;
    const int pos = rq.len - rq.count + c / a.grp;  // sees tokens (pos - window, pos]
    f16x8 qf[PARTS][2 * KJ];
    float to_score;
    {
        const typename T::raw *q = static_cast<const typename T::raw *>(a.q) + (size_t)token * a.qt + (size_t)head * a.qh;
        float x[KJ][16], top = 0.0f;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
            const int d = 64 * j + 16 * g;
            if (d < a.hd) load_up<T, 16>(q + d, a.q_vec, x[j]);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                if (d >= a.hd) x[j][e] = 0.0f;
                top = fmaxf(top, fabsf(x[j][e]));
            }
        }
        top = max_rows(top);
        const int e2 = range_shift(top);
        to_score = ldexpf(a.scale_log2, -e2);
#pragma unroll
        for (int j = 0; j < 2 * KJ; ++j) {
            float y[8];
            f16x8 part[PARTS];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = ldexpf(x[j / 2][8 * (j % 2) + e], e2);
            split_f16<PARTS>(y, part);
#pragma unroll
            for (int p = 0; p < PARTS; ++p) qf[p][j] = part[p];
        }
    }

    f32x4 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = f32x4{0, 0, 0, 0};
    float m = kNegInf, lsum = 0.0f, vref = 0.0f;

    // Byte offsets of this lane's loads inside 16 tokens' rows. Channels past the head dimension are read
    // from the row's start: queries are 0 there, and outputs are not stored.
    const unsigned hd = (unsigned)a.hd;
    unsigned koff[KJ], voff[4];
#pragma unroll
    for (int j = 0; j < KJ; ++j) koff[j] = n * hd + (64u * j + 16u * g < hd ? 64u * j + 16u * g : 0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) voff[i] = (4u * g + i) * hd + ((unsigned)(NT * n) < hd ? (unsigned)(NT * n) : 0u);

    const int page_mask = (1 << a.page_shift) - 1;
    const int32_t *table = a.table + (size_t)r * a.max_pages;
    // 2 x 16 tokens, each 16 in one page; the next tile's are loaded while this one's are used
    struct Tile {
        float ks[2], vs[2];
        bool there[2];
        u32x4 kw[2][KJ];
        uint32_t vw[VW][8];
    };
    // (the page ids of a tile are fetched while the tile before it is loaded; past the end the last
    // tokens are loaded again, so that every tile has the same loads in flight behind it)
    const int t_last = max(end - 1, begin) & ~15;
    int page0, page1;
    auto fetch = [&](int t0) {
        page0 = table[min(t0, t_last) >> a.page_shift];
        page1 = table[min(t0 + 16, t_last) >> a.page_shift];
    };
    auto load = [&](int t0, Tile &x) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int t = min(t0 + 16 * s, t_last), page = s ? page1 : page0;
            x.there[s] = page_ok(page, a.n_pages);
            const size_t ph = (size_t)(x.there[s] ? page : 0) * a.n_kv + h;
            x.ks[s] = a.ks[ph];
            x.vs[s] = a.vs[ph];
            const size_t row = ((ph << a.page_shift) + (t & page_mask)) * hd;
            const int8_t *kp = a.k + row, *vp = a.v + row;
#pragma unroll
            for (int j = 0; j < KJ; ++j) x.kw[s][j] = *reinterpret_cast<const u32x4 *>(kp + koff[j]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w[VW];
                __builtin_memcpy(w, __builtin_assume_aligned(vp + voff[i], 4 * VW), 4 * VW);
#pragma unroll
                for (int e = 0; e < VW; ++e) x.vw[e][4 * s + i] = w[e];
            }
        }
    };
    const int pos_lo = rq.len - rq.count + c0 / a.grp, pos_hi = rq.len - rq.count + (min(c0 + 16, cols) - 1) / a.grp;
    auto use = [&](int t0, Tile &x) {
        float s[8], top = kNegInf;
        // (tiles that every column sees whole need no comparisons)
        const bool whole = x.there[0] && x.there[1] && t0 + 31 <= pos_lo && pos_hi - t0 < a.window;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                const f16x8 k0 = codes8(x.kw[u][j].x, x.kw[u][j].y), k1 = codes8(x.kw[u][j].z, x.kw[u][j].w);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[p][2 * j], acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[p][2 * j + 1], acc, 0, 0, 0);
                }
            }
            const float f = x.ks[u] * to_score;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * u + i] = acc[i] * f;
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int t = t0 + 16 * (i / 4) + 4 * g + i % 4;
                if (!(x.there[i / 4] && t <= pos && pos - t < a.window)) s[i] = kNegInf;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, s[i]);
        const float m_new = fmaxf(m, max_rows(top)), m_use = m_new == kNegInf ? 0.0f : m_new;
        const float vs[2] = {x.there[0] ? x.vs[0] : 0.0f, x.there[1] ? x.vs[1] : 0.0f};
        const float vref_new = fmaxf(vref, fmaxf(vs[0], vs[1])), per = vref_new > 0.0f ? 1.0f / vref_new : 0.0f;
        const float fade = exp2_fast(m - m_use), fade_o = vref == vref_new ? fade : fade * (vref * per);
        const float vw[2] = {vs[0] * (per * kWeightScale), vs[1] * (per * kWeightScale)};
        lsum *= fade;
        f16x8 wf[PARTS];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = exp2_fast(s[i] - m_use);  // (unseen: 2^-inf = 0)
            lsum += p;
            s[i] = p * vw[i / 4];
        }
        split_f16<PARTS>(s, wf);
        m = m_new;
        vref = vref_new;
        if (__any(fade_o != 1.0f)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] *= fade_o;
        }
#pragma unroll
        for (int e = 0; e < VW; ++e)
#pragma unroll
            for (int i = 0; i < 8; ++i) x.vw[e][i] ^= 0x80808080u;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const f16x8 vf = codes_across(x.vw[t / 4], t % 4);
#pragma unroll
            for (int p = 0; p < PARTS; ++p) o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, wf[p], o[t], 0, 0, 0);
        }
    };
    int t0 = begin + 32 * w;
    if (t0 < end) {
        Tile tiles[2];
        fetch(t0);
        load(t0, tiles[0]);
        fetch(t0 + 128);
        while (true) {
            load(t0 + 128, tiles[1]);
            fetch(t0 + 256);
            use(t0, tiles[0]);
            t0 += 128;
            if (t0 >= end) break;
            load(t0 + 128, tiles[0]);
            fetch(t0 + 256);
            use(t0, tiles[1]);
            t0 += 128;
            if (t0 >= end) break;
        }
    }

    // the four waves' sums, joined per column
    lsum += __shfl_xor(lsum, 16, 64);
    lsum += __shfl_xor(lsum, 32, 64);
    if (g == 0) {
        s_ml[w][n][0] = m;
        s_ml[w][n][1] = lsum;
    }
    __syncthreads();
    float m_all = kNegInf;
#pragma unroll
    for (int i = 0; i < 4; ++i) m_all = fmaxf(m_all, s_ml[i][n][0]);
    const float m_use = m_all == kNegInf ? 0.0f : m_all;
    // (NaN scores leave m at -inf but make the sum NaN: it must not be multiplied away)
    const float mine = m == kNegInf ? (__builtin_isnan(lsum) ? lsum : 0.0f) : exp2_fast(m - m_use) * vref * (kCodeScale / kWeightScale);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_o[w][n][NT * (4 * g + i) + t] = o[t][i] * mine;
    float l_all = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float mi = s_ml[i][n][0], li = s_ml[i][n][1];
        l_all += mi == kNegInf ? (__builtin_isnan(li) ? li : 0.0f) : li * exp2_fast(mi - m_use);
    }
    __syncthreads();
    if (w == 0 && g == 0) s_ml[0][n][2] = l_all;
    if (w == 0 && g == 1) s_ml[1][n][2] = m_all;
    __syncthreads();
    // 8 channels a thread
    for (int i = threadIdx.x; i < 16 * (HDP / 8); i += 256) {
        const int col = i / (HDP / 8), d = i % (HDP / 8) * 8;
        if (c0 + col >= cols || d >= a.hd) continue;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = ((s_o[0][col][d + e] + s_o[1][col][d + e]) + s_o[2][col][d + e]) + s_o[3][col][d + e];
        const float lc = s_ml[0][col][2];
        const int tok = rq.first + (c0 + col) / a.grp, hq = h * a.grp + (c0 + col) % a.grp;
        if (sp.active == 1) {
            const float inv = lc == 0.0f ? 0.0f : 1.0f / lc;
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] *= inv;
            store_down<T, 8>(static_cast<typename T::raw *>(a.out) + (size_t)tok * a.ot + (size_t)hq * a.oh + d, a.out_vec, y);
        } else {
            const size_t at = ((size_t)tok * a.n_heads + hq) * a.splits + split;
            store_down<F32, 8>(a.part_o + at * a.hd + d, true, y);
            if (d == 0) a.part_ml[at] = make_float2(s_ml[1][col][2], lc);
        }
    }
}

// Joins the splits of one column a wave: out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
template <typename T>
__global__ __launch_bounds__(256) void attn_q8_join_kernel(AttnDev a) {
    const int l = threadIdx.x & 63;
    const long unit = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (long)a.n_tokens * a.n_heads) return;
    const int token = (int)(unit / a.n_heads), head = (int)(unit % a.n_heads), h = head / a.grp;
    // the request of the token
    if (token < a.q_start[0]) return;
    int lo = 0, hi = a.n_requests;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] <= token) lo = mid;
        else hi = mid;
    }
    const Req rq = request_of(a, lo);
    const int i = token - rq.first;
    const int cols = min(rq.count, a.max_new) * a.grp, c = i * a.grp + (head - h * a.grp), c0 = c & ~15;
    if (i < 0 || c >= cols) return;
    const Span sp = span_of(a, rq, c0, min(c0 + 16, cols));
    if (sp.active == 1) return;  // (written whole)
    const size_t at = (size_t)unit * a.splits;
    float m = kNegInf;
    for (int s = 0; s < sp.active; ++s) m = fmaxf(m, a.part_ml[at + s].x);
    const float m_use = m == kNegInf ? 0.0f : m;
    float y[4] = {0, 0, 0, 0}, lsum = 0.0f;
    for (int s = 0; s < sp.active; ++s) {
        const float2 ml = a.part_ml[at + s];
        const float f = exp2_fast(ml.x - m_use);
        lsum += ml.x == kNegInf ? ml.y : ml.y * f;  // (0, or NaN)
        if (4 * l < a.hd) {
            const float4 o = *reinterpret_cast<const float4 *>(a.part_o + (at + s) * a.hd + 4 * l);
            y[0] = fmaf(o.x, f, y[0]), y[1] = fmaf(o.y, f, y[1]), y[2] = fmaf(o.z, f, y[2]), y[3] = fmaf(o.w, f, y[3]);
        }
    }
    const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
    if (4 * l < a.hd) {
        typename T::raw *out = static_cast<typename T::raw *>(a.out) + (size_t)token * a.ot + (size_t)head * a.oh + 4 * l;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = T::down(y[e] * inv);
    }
}

static jk_status attn_check(const jk_kv_q8 *c, const jk_attn_q8_args *a) {
    JK_TRY(kv_check("attn_q8", c));
    if (!a) return fail(JK_TENSOR_BOUNDS, "attn_q8: null arguments");
    if (!dtype_ok(a->dtype)) return fail(JK_CAPABILITY_MISMATCH, "attn_q8: unknown element type %d", a->dtype);
    if (a->n_heads == 0 || a->n_heads % c->n_kv || a->n_heads > 65536)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: %zu query heads for %zu kv heads", a->n_heads, c->n_kv);
    if (a->n_requests == 0 || a->max_pages == 0 || a->n_requests > (size_t)INT32_MAX / 64 ||
        a->max_pages > (size_t)INT32_MAX / c->page)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: %zu requests of %zu pages", a->n_requests, a->max_pages);
    if (a->n_tokens > (size_t)INT32_MAX / a->n_heads)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: %zu tokens of %zu heads exceed the int32 range", a->n_tokens, a->n_heads);
    return JK_OK;
}

// How many workgroups share the keys of a column tile: enough to fill the GPU twice over, and no more than
// kMaxChunk keys each, so that a long request in a batch of short ones does not hold up the launch.
constexpr size_t kMaxChunk = 4096, kMaxSplits = 256;
static size_t attn_tiles(const jk_kv_q8 *c, const jk_attn_q8_args *a) {
    return (std::min(a->max_new, a->n_tokens) * (a->n_heads / c->n_kv) + 15) / 16;
}
static size_t attn_splits(const jk_kv_q8 *c, const jk_attn_q8_args *a) {
    const size_t units = std::max<size_t>(1, a->n_requests * attn_tiles(c, a) * c->n_kv);
    const size_t len = std::min(a->max_len, a->max_pages * c->page);
    const size_t most = std::max<size_t>(1, std::min<size_t>(kMaxSplits, (len + kMinChunk - 1) / kMinChunk));
    const size_t want = std::max((2 * (size_t)cu_count() + units - 1) / units, (len + kMaxChunk - 1) / kMaxChunk);
    return std::min(most, std::max<size_t>(1, want));
}
static size_t attn_ws_bytes(const jk_kv_q8 *c, const jk_attn_q8_args *a) {
    const size_t s = attn_splits(c, a);
    return s == 1 ? 0 : a->n_tokens * a->n_heads * s * (c->head_dim * 4 + 8);
}

template <typename T, int PARTS>
static jk_status launch_attn(hipStream_t s, const AttnDev &d, unsigned grid) {
    if (d.hd <= 64) hipLaunchKernelGGL((attn_q8_rows_kernel<T, 64, PARTS>), dim3(grid), dim3(256), 0, s, d);
    else if (d.hd <= 128) hipLaunchKernelGGL((attn_q8_rows_kernel<T, 128, PARTS>), dim3(grid), dim3(256), 0, s, d);
    else hipLaunchKernelGGL((attn_q8_rows_kernel<T, 256, PARTS>), dim3(grid), dim3(256), 0, s, d);
    JK_TRY(check_launch("attn_q8_rows_kernel"));
    if (d.splits == 1) return JK_OK;
    const unsigned blocks = (unsigned)(((size_t)d.n_tokens * d.n_heads + 3) / 4);
    hipLaunchKernelGGL(attn_q8_join_kernel<T>, dim3(blocks), dim3(256), 0, s, d);
    return check_launch("attn_q8_join_kernel");
}

}  // namespace jk

using namespace jk;

extern "C" {

size_t jk_attn_q8_workspace_bytes(const jk_kv_q8 *c, const jk_attn_q8_args *a) {
    return attn_check(c, a) == JK_OK ? attn_ws_bytes(c, a) : 0;
}

jk_status jk_attn_q8(jk_stream s, const jk_kv_q8 *c, const jk_attn_q8_args *a, void *ws, size_t ws_bytes) {
    JK_TRY(attn_check(c, a));
    if (a->n_tokens == 0 || a->max_new == 0) return JK_OK;
    if (!a->q || !a->out || !a->q_start || !a->lens || !a->table)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: null queries, output, q_start, lengths or table");
    const size_t es = dtype_bytes(a->dtype);
    if ((uintptr_t)a->q % es || (uintptr_t)a->out % es)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: queries and output must be aligned to their elements");
    if (!std::isfinite(a->scale)) return fail(JK_TENSOR_BOUNDS, "attn_q8: scale %g", (double)a->scale);
    AttnDev d{};
    d.q = a->q, d.out = a->out;
    d.qh = a->q_stride_head ? a->q_stride_head : c->head_dim, d.oh = a->out_stride_head ? a->out_stride_head : c->head_dim;
    d.qt = a->q_stride_token ? a->q_stride_token : a->n_heads * c->head_dim;
    d.ot = a->out_stride_token ? a->out_stride_token : a->n_heads * c->head_dim;
    d.q_vec = (uintptr_t)a->q % 16 == 0 && d.qt * es % 16 == 0 && d.qh * es % 16 == 0;
    d.out_vec = (uintptr_t)a->out % 16 == 0 && d.ot * es % 16 == 0 && d.oh * es % 16 == 0;
    d.n_tokens = (int)a->n_tokens, d.n_heads = (int)a->n_heads, d.n_kv = (int)c->n_kv;
    d.grp = (int)(a->n_heads / c->n_kv), d.hd = (int)c->head_dim;
    d.page_shift = 4;
    while (((size_t)1 << d.page_shift) < c->page) ++d.page_shift;
    d.n_pages = (int)c->n_pages, d.max_pages = (int)a->max_pages, d.n_requests = (int)a->n_requests;
    d.max_new = (int)std::min<size_t>(a->max_new, a->n_tokens);
    d.q_start = a->q_start, d.lens = a->lens, d.table = a->table;
    d.k = c->k, d.v = c->v, d.ks = c->k_scale, d.vs = c->v_scale;
    d.scale_log2 = a->scale * 1.44269504088896340736f * kCodeScale;
    d.window = a->window == 0 || a->window > (size_t)INT32_MAX ? INT32_MAX : (int)a->window;
    d.tiles = (int)attn_tiles(c, a), d.splits = (int)attn_splits(c, a);
    const size_t need = attn_ws_bytes(c, a);
    if (need && (!ws || (uintptr_t)ws % 16 || ws_bytes < need))
        return fail(JK_TENSOR_BOUNDS, "attn_q8: workspace of %zu bytes at %p: %zu needed, 16-byte aligned", ws_bytes, ws,
                    need);
    d.part_o = static_cast<float *>(ws);
    d.part_ml = reinterpret_cast<float2 *>(d.part_o + (need ? a->n_tokens * a->n_heads * d.splits * c->head_dim : 0));
    const size_t grid = a->n_requests * d.tiles * c->n_kv * d.splits;
    if (grid >= (size_t)1 << 24)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: %zu requests of up to %zu new tokens and %zu kv heads are too many for one call",
                    a->n_requests, a->max_new, c->n_kv);
    if (a->dtype == JK_F32) return launch_attn<F32, 2>((hipStream_t)s, d, (unsigned)grid);
    if (a->dtype == JK_F16) return launch_attn<F16, 1>((hipStream_t)s, d, (unsigned)grid);
    return launch_attn<BF16, 1>((hipStream_t)s, d, (unsigned)grid);
}

}  // extern "C"
