// jk_attention.hip -- attention over the paged 8-bit cache: the kernel for few columns (a decode step, drafted tokens), the
// joining of split keys, and the entry points.
#include <algorithm>
#include <cmath>

#include "jk_attention.hpp"

namespace jk {

// Up to 16 columns of one request and kv head over one split of its keys, by four waves that take 32 tokens in
// turn; their sums are joined in LDS. A lane (n = lane % 16, g = lane / 16) holds of column n: the query's
// channels 64 j + 16 g + .. as the first product's operand, the scores of tokens 4 g + i and 16 + 4 g + i, and
// of its output the channels (HDP / 16) (4 g + i) + t. Of the keys it loads row n (16 bytes at a time), of the values
// channels (HDP / 16) n + t of the eight tokens whose scores it holds, so that the loads of a wave cover whole rows
// and nothing goes through LDS.
// What bounds it: the cache's bytes, 2 a channel and token for all columns of the group, where requests are many (64 requests,
// 290 thousand tokens, 8 kv heads of 128, bf16: 117-119 us, 5.1 TB/s, as fast as a copy); where one long request is cut
// over the CUs, a tile's chain of loads, products and exponentials (32 thousand tokens 20-21 us, 3.3 TB/s, and 4 for the joining); and
// with hundreds of columns the matrix units, of which a tile of 16 columns uses a quarter of what the prompt kernel's does. Waves
// take tokens in turn and not columns because the few columns of a step are one tile, and its keys' loads need many
// waves in flight: three a SIMD.
// PARTS: f16 parts that f32 queries and probabilities are split into.
template <typename T, int HDP, int PARTS>
__global__ __launch_bounds__(256, HDP <= 128 ? 3 : 1) void attn_q8_rows_kernel(AttnDev a) {
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
    if (c0 >= cols || cols > a.few_cols) return;
    const Span sp = span_of(a, rq, c0, min(c0 + 16, cols));
    if (split >= sp.active) return;
    const int begin = sp.lo + split * sp.chunk, end = piece_end(sp, begin);

    f32x4 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = f32x4{0, 0, 0, 0};
    float m = kNegInf, lsum = 0.0f, vref = kLeastV, per = kWeight / kLeastV;  // per: kWeight / vref

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
    // (the first tile's loads go out before the queries are looked at)
    Tile tiles[2];
    int t0 = begin + 32 * w;
    if (t0 < end) {
        fetch(t0);
        load(t0, tiles[0]);
        fetch(t0 + 128);
    }

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
        to_score = ldexpf(fabsf(a.scale_log2), kCodeShift - e2);  // (its sign goes to the queries)
#pragma unroll
        for (int j = 0; j < 2 * KJ; ++j) {
            float y[8];
            f16x8 part[PARTS];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float q = x[j / 2][8 * (j % 2) + e];
                y[e] = ldexpf(a.scale_log2 < 0.0f ? -q : q, e2);
            }
            split_f16<PARTS>(y, part);
#pragma unroll
            for (int p = 0; p < PARTS; ++p) qf[p][j] = part[p];
        }
    }

    const int pos_lo = rq.len - rq.count + c0 / a.grp, pos_hi = rq.len - rq.count + (min(c0 + 16, cols) - 1) / a.grp;
    auto use = [&](int t0, Tile &x) {
        float s[8], f[2], vs[2], top = kNegInf;
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
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * u + i] = acc[i];
            vs[u] = x.vs[u];
            f[u] = x.ks[u];
        }
        if (!whole) {
            asm("" : "+v"(s[0]));  // (keeps the branch: few tiles need this, and selects would cost every tile)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int t = t0 + 16 * (i / 4) + 4 * g + i % 4;
                if (!(x.there[i / 4] && t <= pos && pos - t < a.window)) s[i] = kNegInf;
            }
            // (a page that the column sees nothing of has no say in its references: its scales, or those of what stands in
            // for a missing page, may be of any size, or no numbers)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int t = t0 + 16 * u;
                if (!(x.there[u] && t <= pos && pos - (t + 15) < a.window)) vs[u] = f[u] = 0.0f;
            }
        }
        // scores are s * f, f one number a page and positive (0 becomes next to nothing: an unseen -inf stays one)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f[u] *= to_score;
            f[u] = f[u] < 1e-37f ? 1e-37f : f[u];
            top = fmaxf(top, fmaxf(fmaxf(s[4 * u], s[4 * u + 1]), fmaxf(s[4 * u + 2], s[4 * u + 3])) * f[u]);
        }
        const bool vmove = fmaxf(vs[0], vs[1]) > vref * kSlackV;
        if (__any(vmove || top > m + kSlack)) {
            top = max_rows(top);
            const float m_new = top > m + kSlack ? top : m, vref_new = vmove ? fmaxf(vs[0], vs[1]) : vref;
            // (the first reference of a column comes from nothing: nothing is kept)
            const float fade = m_new == m ? 1.0f : exp2_fast(m - m_new), fade_o = vmove ? fade * (vref / vref_new) : fade;
            m = m_new;
            vref = vref_new;
            per = kWeight / vref;
            lsum *= fade;
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] *= fade_o;
        }
        const float m_use = m == kNegInf ? 0.0f : m;
        f16x8 wf[PARTS];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float vw = vs[u] * per;
#pragma unroll
            for (int i = 4 * u; i < 4 * u + 4; ++i) {
                const float p = exp2_fast(__builtin_fmaf(s[i], f[u], -m_use));  // (unseen: 2^-inf = 0)
                lsum += p;
                s[i] = p * vw;
            }
        }
        split_f16<PARTS>(s, wf);
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
    if (t0 < end) {
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
    const float mine = m == kNegInf ? (__builtin_isnan(lsum) ? lsum : 0.0f) : exp2_fast(m - m_use) * vref * (kCodeScale / kWeight);
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
            const size_t at = ((size_t)tok * a.n_heads + hq) * a.pitch + split;
            store_down<F32, 8>(a.part_o + at * a.hd + d, true, y);
            if (d == 0) a.part_ml[at] = make_float2(s_ml[1][col][2], lc);
        }
    }
}

// Joins the splits of one column a wave: out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i. The lanes first take a split each
// (their factors), then four channels each, with G groups of lanes on every G-th split; four splits' loads in flight. A second
// launch's latency: 4 us for 32 rows of 33 splits (0.6 MB).
// WPR: waves that share a column's splits.
template <typename T, int HDP, int WPR>
__global__ __launch_bounds__(256) void attn_q8_join_kernel(AttnDev a) {
    constexpr int LP = HDP / 4, G = 64 / LP;
    __shared__ float s_f[4][kMaxSplits];
    __shared__ float4 s_y[4][LP];
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long unit = (long)blockIdx.x * (4 / WPR) + w / WPR;
    if (unit >= (long)a.n_tokens * a.n_heads) return;
    const int token = (int)(unit / a.n_heads), head = (int)(unit % a.n_heads), h = head / a.grp;
    // the request of the token: the last of those that do not begin after it, 64 of them looked at together
    int lo = 0;
    for (int n = a.n_requests; n > 0;) {
        const int step = (n + 63) / 64, probes = (n + step - 1) / step;
        const unsigned long long before = __ballot(l < probes && a.q_start[lo + min(l * step, n - 1)] <= token);
        if (!(before & 1)) return;
        const int at = __builtin_popcountll(before) - 1;
        lo += at * step;
        n = step == 1 ? 0 : min(step, n - at * step);
    }
    const Req rq = request_of(a, lo);
    const int i = token - rq.first;
    const int cols = min(rq.count, a.max_new) * a.grp, c = i * a.grp + (head - h * a.grp);
    if (i < 0 || c >= cols) return;
    a.splits = cols <= a.few_cols ? a.few_splits : a.many_splits;
    a.chunk = cols <= a.few_cols ? a.few_chunk : a.many_chunk;
    const int tile = cols <= a.few_cols ? 16 : a.many_cols, c0 = c / tile * tile;
    const Span sp = span_of(a, rq, c0, min(c0 + tile, cols));
    if (sp.active == 1) return;  // (written whole)
    const size_t at = (size_t)unit * a.pitch;
    const float2 none = make_float2(kNegInf, 0.0f);
    float2 ml[kMaxSplits / 64];
    float m = kNegInf, lsum = 0.0f;
#pragma unroll
    for (int k = 0; k < kMaxSplits / 64; ++k) {
        ml[k] = none;
        if (64 * k < sp.active && l + 64 * k < sp.active) ml[k] = a.part_ml[at + l + 64 * k];
        m = fmaxf(m, ml[k].x);
    }
    m = wave_max64_dpp(m);
    const float m_use = m == kNegInf ? 0.0f : m;
#pragma unroll
    for (int k = 0; k < kMaxSplits / 64; ++k) {
        if (64 * k >= sp.active) break;
        const float f = exp2_fast(ml[k].x - m_use);
        s_f[w][l + 64 * k] = f;
        lsum += ml[k].x == kNegInf ? ml[k].y : ml[k].y * f;  // (0, or NaN)
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) lsum += __shfl_xor(lsum, o, 64);
    wave_lds_sync();
    const int d = 4 * (l % LP);
    float4 y = make_float4(0, 0, 0, 0);
    if (d < a.hd) {
#pragma unroll 4
        for (int s = w % WPR * G + l / LP; s < sp.active; s += WPR * G) {
            const float4 o = *reinterpret_cast<const float4 *>(a.part_o + (at + s) * a.hd + d);
            const float f = s_f[w][s];
            y.x = fmaf(o.x, f, y.x), y.y = fmaf(o.y, f, y.y), y.z = fmaf(o.z, f, y.z), y.w = fmaf(o.w, f, y.w);
        }
    }
#pragma unroll
    for (int o = LP; o < 64; o <<= 1) {
        y.x += __shfl_xor(y.x, o, 64), y.y += __shfl_xor(y.y, o, 64);
        y.z += __shfl_xor(y.z, o, 64), y.w += __shfl_xor(y.w, o, 64);
    }
    if constexpr (WPR > 1) {  // (a workgroup is one column: its waves have all come here)
        if (l < LP) s_y[w][l] = y;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int k = 1; k < WPR; ++k) {
            const float4 z = s_y[k][l % LP];
            y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
        }
    }
    if (l < LP && d < a.hd) {
        const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
        typename T::raw *out = static_cast<typename T::raw *>(a.out) + (size_t)token * a.ot + (size_t)head * a.oh + d;
        out[0] = T::down(y.x * inv), out[1] = T::down(y.y * inv), out[2] = T::down(y.z * inv), out[3] = T::down(y.w * inv);
    }
}

static jk_status attn_check(const jk_kv_q8 *c, const jk_attn_q8_args *a) {
    JK_TRY(kv_check("attn_q8", c));
    if (!a) return fail(JK_TENSOR_BOUNDS, "attn_q8: null arguments");
    if (!dtype_ok(a->dtype)) return fail(JK_CAPABILITY_MISMATCH, "attn_q8: unknown element type %d", a->dtype);
    if (a->n_heads == 0 || a->n_heads % c->n_kv || a->n_heads > 65536)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: %zu query heads for %zu kv heads", a->n_heads, c->n_kv);
    if (a->n_requests == 0 || a->max_pages == 0 || a->n_requests > (size_t)INT32_MAX / 64 ||
        a->max_pages > kMaxTokens / c->page)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: %zu requests of %zu pages", a->n_requests, a->max_pages);
    if (a->n_tokens > (size_t)INT32_MAX / a->n_heads)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: %zu tokens of %zu heads exceed the int32 range", a->n_tokens, a->n_heads);
    return JK_OK;
}

// How a call is cut up. Requests of up to kFewCols columns go to the rows kernel, sixteen columns a workgroup; longer ones to
// the prompt kernel. (One request, 32 query and 8 kv heads of 128, bf16, rows against prompt kernel: 128 new tokens after 2000 20 and
// 30 us; 512 after none 19 and 20 us, after 4000 105 and 70 us; 2048 after none 115 and 64 us. In f32, whose parts cost the prompt
// kernel's products twice as much: 256 new tokens after none 10.5 and 18 us, after 2000 34 and 50, after 8000 103 and 113; 512 after
// none 20 and 27, after 2000 64 and 64, after 8000 200 and 153; 1024 after none 45 and 46, after 2000 131 and 150.) A call that can hold both
// launches both (the counts are known on the device only), except that the prompt kernel takes a lone request
// whatever its length turns out to be.
// The prompt kernel takes 256 columns a workgroup (one a CU, 159 us for the 4096-token prompt, 175 with 128) where
// there are two tiles a CU to level out their lengths, else 128 (two a CU: 64 us for 2048 tokens against 96).
// Where there are fewer tiles than places, their keys are cut into chunks of one size for the whole call, a place's share of the work,
// so that the last ones are not left with a long request or with a prompt's last tiles, which see the most keys. Up to kWholeLen
// keys are not cut: the second launch costs more than it saves (decode step of three requests of up to 700 keys 9 us whole, 13
// in two; one of 1000 12.4 and 14; of 2000 17.5 and 14. A prompt of 1024 tokens 34 us whole and 50 in two; two of 700 after 300
// 39 and 75; 512 tokens after 500 33 and 38, but of 256 channels 64 and 56). Longer ones go down to kMinPromptChunk keys (512
// tokens after 2000 52 us, with 1024 keys at least 64; 1024 after 1000 83 and 73).
// Few rows are joined by four waves each, more by one (one step after 32 thousand tokens, 32 rows: 19.2 us with four, 20.1 with one; 8
// after 16 thousand, 256 rows: 46.3 and 50.2; 31 after 8 thousand, 992 rows: 121.7 and 118.5; 2048 rows: 40.1 and 37.3).
constexpr size_t kJoinByFour = 512;
constexpr size_t kFewCols = 1024, kFewColsF32 = 2048, kMixedCols = 64, kMinChunk = 256, kMinPromptChunk = 512, kWholeLen = 1024;
struct AttnPlan {
    size_t few_tiles, few_splits, few_chunk, many_cols, many_tiles, many_splits, many_chunk, few_cols, pitch;
};
static AttnPlan attn_plan(const jk_kv_q8 *c, const jk_attn_q8_args *a) {
    AttnPlan p{};
    const size_t new_tokens = std::min(a->max_new, a->n_tokens), cols = new_tokens * (a->n_heads / c->n_kv);
    const size_t heads = a->n_requests * c->n_kv, ncu = (size_t)cu_count();
    size_t len = std::min(a->max_len, a->max_pages * c->page);
    if (a->window) len = std::min(len, a->window + new_tokens);
    auto cut = [&](size_t share, size_t least, size_t *splits, size_t *chunk) {
        *chunk = std::max({share, len <= kWholeLen ? kWholeLen : least, (len + kMaxSplits - 1) / kMaxSplits});
        *chunk = (std::min(*chunk, std::max<size_t>(len, 1)) + 127) / 128 * 128;
        *splits = std::max<size_t>(1, (len + *chunk - 1) / *chunk);
    };
    const size_t few = a->dtype == JK_F32 ? kFewColsF32 : kFewCols;
    p.few_cols = cols <= few ? few : a->n_requests == 1 ? 0 : kMixedCols;
    p.few_splits = p.many_splits = p.few_chunk = p.many_chunk = 1;
    if (p.few_cols) {
        p.few_tiles = (std::min(cols, p.few_cols) + 15) / 16;
        cut(heads * p.few_tiles * len / ncu, kMinChunk, &p.few_splits, &p.few_chunk);
    }
    if (cols > p.few_cols) {
        p.many_cols = c->head_dim <= 128 && heads * ((cols + 255) / 256) >= 2 * ncu ? 256 : 128;
        p.many_tiles = (cols + p.many_cols - 1) / p.many_cols;
        const size_t tiles = heads * p.many_tiles, places = p.many_cols == 128 ? 2 * ncu : ncu;
        if (tiles < places)
            cut(tiles * (len - std::min(len, new_tokens) / 2) / places, kMinPromptChunk, &p.many_splits, &p.many_chunk);
    }
    p.pitch = std::max(p.few_splits, p.many_splits);
    return p;
}
static size_t attn_ws_bytes(const jk_kv_q8 *c, const jk_attn_q8_args *a, const AttnPlan &p) {
    return p.pitch == 1 ? 0 : a->n_tokens * a->n_heads * p.pitch * (c->head_dim * 4 + 8);
}

template <typename T, int HDP>
static void launch_join(hipStream_t s, const AttnDev &d) {
    const size_t rows = (size_t)d.n_tokens * d.n_heads;
    if (rows <= kJoinByFour)
        hipLaunchKernelGGL((attn_q8_join_kernel<T, HDP, 4>), dim3((unsigned)rows), dim3(256), 0, s, d);
    else
        hipLaunchKernelGGL((attn_q8_join_kernel<T, HDP, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, d);
}

template <typename T, int PARTS>
static jk_status launch_attn(hipStream_t s, int dtype, AttnDev d, const AttnPlan &p) {
    const size_t units = (size_t)d.n_requests * d.n_kv;
    if (p.few_tiles) {
        d.tile_cols = 16, d.tiles = (int)p.few_tiles, d.splits = d.few_splits, d.chunk = d.few_chunk;
        const dim3 grid((unsigned)(units * p.few_tiles * p.few_splits));
        if (d.hd <= 64) hipLaunchKernelGGL((attn_q8_rows_kernel<T, 64, PARTS>), grid, dim3(256), 0, s, d);
        else if (d.hd <= 128) hipLaunchKernelGGL((attn_q8_rows_kernel<T, 128, PARTS>), grid, dim3(256), 0, s, d);
        else hipLaunchKernelGGL((attn_q8_rows_kernel<T, 256, PARTS>), grid, dim3(256), 0, s, d);
        JK_TRY(check_launch("attn_q8_rows_kernel"));
    }
    if (p.many_tiles) {
        d.tile_cols = d.many_cols, d.tiles = (int)p.many_tiles, d.splits = d.many_splits, d.chunk = d.many_chunk;
        JK_TRY(launch_attn_prompt(s, dtype, d));
    }
    if (p.pitch == 1) return JK_OK;
    if (d.hd <= 64) launch_join<T, 64>(s, d);
    else if (d.hd <= 128) launch_join<T, 128>(s, d);
    else launch_join<T, 256>(s, d);
    return check_launch("attn_q8_join_kernel");
}

}  // namespace jk

using namespace jk;

extern "C" {

size_t jk_attn_q8_workspace_bytes(const jk_kv_q8 *c, const jk_attn_q8_args *a) {
    return attn_check(c, a) == JK_OK ? attn_ws_bytes(c, a, attn_plan(c, a)) : 0;
}

jk_status jk_attn_q8(jk_stream s, const jk_kv_q8 *c, const jk_attn_q8_args *a, void *ws, size_t ws_bytes) {
    JK_TRY(attn_check(c, a));
    if (a->n_tokens == 0 || a->max_new == 0) return JK_OK;
    if (!a->q || !a->out || !a->q_start || !a->lens || !a->table)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: null queries, output, q_start, lengths or table");
    const size_t es = dtype_bytes(a->dtype);
    if ((uintptr_t)a->q % es || (uintptr_t)a->out % es)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: queries and output must be aligned to their elements");
    if (!std::isfinite(a->scale * kLog2e)) return fail(JK_TENSOR_BOUNDS, "attn_q8: scale %g", (double)a->scale);
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
    d.scale_log2 = a->scale * kLog2e;
    d.window = a->window == 0 || a->window > (size_t)INT32_MAX ? INT32_MAX : (int)a->window;
    const AttnPlan plan = attn_plan(c, a);
    d.few_cols = (int)plan.few_cols, d.few_splits = (int)plan.few_splits, d.few_chunk = (int)plan.few_chunk;
    d.many_cols = (int)plan.many_cols, d.many_splits = (int)plan.many_splits, d.many_chunk = (int)plan.many_chunk;
    d.pitch = (int)plan.pitch;
    const size_t need = attn_ws_bytes(c, a, plan);
    if (need && (!ws || (uintptr_t)ws % 16 || ws_bytes < need))
        return fail(JK_TENSOR_BOUNDS, "attn_q8: workspace of %zu bytes at %p: %zu needed, 16-byte aligned", ws_bytes, ws,
                    need);
    d.part_o = static_cast<float *>(ws);
    d.part_ml = reinterpret_cast<float2 *>(d.part_o + (need ? a->n_tokens * a->n_heads * plan.pitch * c->head_dim : 0));
    const size_t units = a->n_requests * c->n_kv, most = (size_t)1 << 24;
    if (units * plan.few_tiles * plan.few_splits >= most || units * plan.many_tiles * plan.many_splits >= most)
        return fail(JK_TENSOR_BOUNDS, "attn_q8: %zu requests of up to %zu new tokens and %zu kv heads are too many for one call",
                    a->n_requests, a->max_new, c->n_kv);
    if (a->dtype == JK_F32) return launch_attn<F32, 2>((hipStream_t)s, a->dtype, d, plan);
    if (a->dtype == JK_F16) return launch_attn<F16, 1>((hipStream_t)s, a->dtype, d, plan);
    return launch_attn<BF16, 1>((hipStream_t)s, a->dtype, d, plan);
}

}  // extern "C"
