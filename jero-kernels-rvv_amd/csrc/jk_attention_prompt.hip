// jk_attention_prompt.hip -- attention over the paged 8-bit cache: the kernel for prompts.
#include "jk_attention.hpp"

#include <type_traits>

namespace jk {

// 32 NC NW columns of one request and kv head by NW waves of 32 NC columns each. 64 tokens at a time are widened to f16
// once for all waves, in LDS, two tiles in turn: codes are loaded a tile ahead of their widening, with one barrier a tile.
//   K: [token][HDP], 16-byte pieces swizzled by the token; a lane of the first product (32 x 32 x 16, rows = tokens) reads
//      8 channels of token lane % 32.
//   V: [channel][64 tokens], the tokens of each 16 ordered 0-3, 8-11, 4-7, 12-15: a lane of the second product (rows =
//      channels) reads the 8 tokens whose scores the first one left in that half of the wave.
// A prompt of 4096 tokens, 32 query and 8 kv heads of 128, bf16: 152 us, 900 TFLOP/s of the products under the diagonal, where a
// large matrix product reaches 1185. What bounds it: each 32 x 32 x 16 instruction needs 1 KB from LDS, which gives 64 to 67
// bytes a cycle to a CU however it is read; that is 4096 of the about 4700 cycles of a tile, and beside it run the matrix units
// (2048) and the exponentials, sums and conversions (about 2800 on each SIMD). 64 columns a wave would halve the reads, but need all
// registers of a SIMD for one wave, whose latencies then stand open (230 us). Keys kept as bytes in LDS save a quarter of the
// reads and cost as much in unpacking (164 us).
typedef float f32x16 __attribute__((ext_vector_type(16)));

// PG: pages that a tile can lie in: 1 (pages of 64 tokens or more), 2 or 4.
template <typename T, int HDP, int PARTS, int NC, int NW, int PG>
__global__ __launch_bounds__(64 * NW, HDP <= 128 ? 2 : 1) void attn_q8_prompt_kernel(AttnDev a) {
    constexpr int KS = HDP / 16, DT = HDP / 32, TH = 64 * NW;
    // 16-byte pieces of K and 8-token x 4-channel blocks of V, and how many a thread stages (the first waves, where they
    // are fewer than threads)
    constexpr int KB = 64 * (HDP / 16), KP = (KB + TH - 1) / TH;
    constexpr int VB = 8 * (HDP / 4), VP = (VB + TH - 1) / TH;
    constexpr int kRowK = HDP * 2, kRowV = 128;   // bytes of a row in LDS
    __shared__ __align__(16) uint8_t s_k[2][64 * kRowK];
    __shared__ __align__(16) uint8_t s_v[2][HDP * kRowV];
    const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), n = l & 31, hf = l >> 5;
    unsigned id = blockIdx.x;
    const int split = id % a.splits;
    id /= a.splits;
    const int h = id % a.n_kv;
    id /= a.n_kv;
    const int r = id % a.n_requests, ct = a.tiles - 1 - (int)(id / a.n_requests);  // (the longest first)

    const Req rq = request_of(a, r);
    const int cols = min(rq.count, a.max_new) * a.grp, c0 = ct * a.tile_cols;
    if (cols <= a.few_cols || c0 >= cols) return;
    const Span sp = span_of(a, rq, c0, min(c0 + a.tile_cols, cols));
    if (split >= sp.active) return;
    const int begin = sp.lo + split * sp.chunk, end = piece_end(sp, begin);

    // this lane's columns
    const int w0 = c0 + w * (32 * NC);  // the wave's first
    int pos[NC];
    f16x8 qf[PARTS][NC][KS];
    float to_score[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int col = min(w0 + 32 * c + n, cols - 1), token = rq.first + col / a.grp, head = h * a.grp + col % a.grp;
        pos[c] = rq.len - rq.count + col / a.grp;
        const typename T::raw *q = static_cast<const typename T::raw *>(a.q) + (size_t)token * a.qt + (size_t)head * a.qh;
        float x[KS][8], top = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (16 * s < a.hd) load_up<T, 8>(q + 16 * s + 8 * hf, a.q_vec, x[s]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (16 * s >= a.hd) x[s][e] = 0.0f;
                top = fmaxf(top, fabsf(x[s][e]));
            }
        }
        top = max_halves(top);
        const int e2 = range_shift(top);
        to_score[c] = ldexpf(fabsf(a.scale_log2), kCodeShift - e2);  // (its sign goes to the queries)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            f16x8 part[PARTS];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[s][e] = ldexpf(a.scale_log2 < 0.0f ? -x[s][e] : x[s][e], e2);
            split_f16<PARTS>(x[s], part);
#pragma unroll
            for (int p = 0; p < PARTS; ++p) qf[p][c][s] = part[p];
        }
    }
    const int pos_lo = rq.len - rq.count + w0 / a.grp;  // the wave's first and last positions
    const int pos_hi = w0 < cols ? rq.len - rq.count + (min(w0 + 32 * NC, cols) - 1) / a.grp : -1;

    f32x16 o[NC][DT];
    float m[NC], lsum[NC], vref[NC], per[NC];  // per: kWeight / vref
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        m[c] = kNegInf, lsum[c] = 0.0f, vref[c] = kLeastV, per[c] = kWeight / kLeastV;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[c][t][e] = 0.0f;
    }

    const unsigned hd = (unsigned)a.hd;
    const int page_mask = (1 << a.page_shift) - 1, t_last = max(end - 1, begin) & ~15;
    const int32_t *table = a.table + (size_t)r * a.max_pages;
    // A tile's pages and scales come as scalars, ahead of their use: page ids (as head index page * n_kv + h, -1 where the table
    // holds none) before the loads, scales with them. Past the end the last tokens are loaded again, so that every
    // tile has the same loads in flight behind it.
    constexpr int kSpan = 64 / PG;  // tokens of a page in a tile
    struct Pages {
        int head[PG];
        float ks[PG], vs[PG];
    };
    auto fetch = [&](int t0, Pages &p) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PG; ++i) p.head[i] = table[min(t0 + kSpan * i, t_last) >> a.page_shift];
    };
    const unsigned page_bytes = hd << a.page_shift;
    u32x4 kraw[KP];
    uint32_t vraw[VP][8];
    auto load = [&](int t0, Pages &p) __attribute__((always_inline)) {
        size_t place[PG];  // of the tile's tokens in each page, keys and values alike
#pragma unroll
        for (int i = 0; i < PG; ++i) {
            p.head[i] = page_ok(p.head[i], a.n_pages) ? p.head[i] * a.n_kv + h : -1;
            const unsigned ph = max(p.head[i], 0);
            p.ks[i] = a.ks[ph];
            p.vs[i] = a.vs[ph];
            place[i] = (size_t)ph * page_bytes + (min(t0 + kSpan * i, t_last) & page_mask & ~(kSpan - 1)) * hd;
        }
        // (a wave's lanes stage tokens of one page, but for values where a page has 16 tokens in a tile or a row 64 channels)
        auto pick = [&](int token) __attribute__((always_inline)) {
            size_t at = place[0];
#pragma unroll
            for (int i = 1; i < PG; ++i) {
                size_t other = place[i];
                // (kept a value: a choice among an array's elements puts the array into scratch memory; 2048 tokens in pages of 16
                // took 110 us so, and 83 now, in pages of 64 60)
                asm("" : "+s"(other));
                at = token >= kSpan * i ? other : at;
            }
            return at;
        };
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int piece = tid + i * TH, t = piece / (HDP / 16), c = piece % (HDP / 16);
            if (w * 64 + i * TH >= KB) break;
            const unsigned off = (t % kSpan) * hd + (16u * c < hd ? 16u * c : 0u);
            kraw[i] = *reinterpret_cast<const u32x4 *>(a.k + pick((w * 64 + i * TH) / (HDP / 16)) + off);
        }
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            const int block = tid + i * TH, tg = block / (HDP / 4), c = block % (HDP / 4) * 4;
            if (w * 64 + i * TH >= VB) break;
            const int t = 16 * (tg / 2) + 4 * (tg & 1);
            const int8_t *at = a.v + pick(PG == 4 && HDP == 64 ? t : 16 * ((w * 64 + i * TH) / (HDP / 4) / 2));
            const unsigned off = (t % kSpan) * hd + ((unsigned)c < hd ? (unsigned)c : 0u);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                vraw[i][e] = *reinterpret_cast<const uint32_t *>(at + off + (e < 4 ? e : e + 4) * hd);
        }
    };
    auto stage_k = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int piece = tid + i * TH, t = piece / (HDP / 16), c = piece % (HDP / 16);
            if (w * 64 + i * TH >= KB) break;
            const f16x8 lo = codes8(kraw[i].x, kraw[i].y), hi = codes8(kraw[i].z, kraw[i].w);
            *reinterpret_cast<f16x8 *>(&s_k[buf][t * kRowK + swz_k<HDP>(2 * c, t)]) = lo;
            *reinterpret_cast<f16x8 *>(&s_k[buf][t * kRowK + swz_k<HDP>(2 * c + 1, t)]) = hi;
        }
    };
    auto stage_v = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            const int block = tid + i * TH, tg = block / (HDP / 4), c = block % (HDP / 4) * 4;
            if (w * 64 + i * TH >= VB) break;
#pragma unroll
            for (int e = 0; e < 8; ++e) vraw[i][e] ^= 0x80808080u;
#pragma unroll
            for (int b = 0; b < 4; ++b)
                *reinterpret_cast<f16x8 *>(&s_v[buf][(c + b) * kRowV + swz_v(tg, c + b)]) = codes_across(vraw[i], b);
        }
    };

    union Scores {
        f32x16 m;
        float v[16];
    };
    // The LDS reads of both products run kAhead matrix instructions ahead of their use (left alone, the compiler puts each read
    // right before its use and the wave waits out the LDS latency every time).
    constexpr int kAhead = PARTS == 2 ? 3 : 6;
    auto scores = [&](int buf, Scores (&s)[2][NC]) __attribute__((always_inline)) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int c = 0; c < NC; ++c) s[tt][c].m = f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                const int t = 32 * tt + n;
                const f16x8 kf = *reinterpret_cast<const f16x8 *>(&s_k[buf][t * kRowK + swz_k<HDP>(2 * k + hf, t)]);
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int p = 0; p < PARTS; ++p)
                        s[tt][c].m = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[p][c][k], s[tt][c].m, 0, 0, 0);
            }
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int i = 0; i < 2 * KS - kAhead; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, NC * PARTS, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, NC * PARTS * kAhead, 0);
    };
    auto use = [&](int t0, int buf, const Pages &pages) __attribute__((always_inline)) {
        Scores s[2][NC];
        scores(buf, s);
        float vtop[NC];  // the largest value scale of the pages that the column sees
        bool whole = t0 + 63 <= pos_lo && pos_hi - t0 < a.window;
#pragma unroll
        for (int c = 0; c < NC; ++c) vtop[c] = 0.0f;
#pragma unroll
        for (int i = 0; i < PG; ++i) {
#pragma unroll
            for (int c = 0; c < NC; ++c) vtop[c] = fmaxf(vtop[c], pages.vs[i]);
            whole = whole && pages.head[i] >= 0;
        }
        if (!whole) {
            asm("" : "+v"(s[0][0].v[0]));  // (keeps the branch: few tiles need this, and selects would cost every tile)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int first = pages.head[i * PG / 4] >= 0 ? pos[c] - t0 - 16 * i - 4 * hf : -1;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int behind = first - (8 * (e / 4) + e % 4);
                        float &x = s[i / 2][c].v[8 * (i % 2) + e];
                        x = behind >= 0 && behind < a.window ? x : kNegInf;
                    }
                }
            // (a page that a column sees nothing of has no say in its references: its scales, or those of what stands in for a
            // missing page, may be of any size, or no numbers)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                vtop[c] = 0.0f;
#pragma unroll
                for (int i = 0; i < PG; ++i) {
                    const int behind = pos[c] - (t0 + kSpan * i);
                    const bool seen = pages.head[i] >= 0 && behind >= 0 && behind - (kSpan - 1) < a.window;
                    vtop[c] = fmaxf(vtop[c], seen ? pages.vs[i] : 0.0f);
                }
            }
        }
        // scores are s * f, f one number a group and positive (0 and no numbers become next to nothing: an unseen -inf stays one)
        float f[NC][PG];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float top = kNegInf;
#pragma unroll
            for (int i = 0; i < PG; ++i) {
                f[c][i] = fmaxf(pages.ks[i] * to_score[c], 1e-37f);
                float big = kNegInf;
#pragma unroll
                for (int e = 0; e < 32 / PG; ++e) big = fmaxf(big, s[(32 / PG * i + e) / 16][c].v[(32 / PG * i + e) % 16]);
                top = fmaxf(top, big * f[c][i]);
            }
            const bool vmove = vtop[c] > vref[c] * kSlackV;
            if (__any(vmove || top > m[c] + kSlack)) {
                top = max_halves(top);
                const float m_new = top > m[c] + kSlack ? top : m[c];
                // (the first reference of a column comes from nothing: nothing is kept)
                const float fade = m_new == m[c] ? 1.0f : exp2_fast(m[c] - m_new);
                const float fade_o = vmove ? fade * (vref[c] / vtop[c]) : fade;
                m[c] = m_new;
                vref[c] = vmove ? vtop[c] : vref[c];
                per[c] = kWeight / vref[c];
                lsum[c] *= fade;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[c][t][e] *= fade_o;
            }
        }

        // 16 tokens at a time: their weights, and their share of the second product
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f16x8 wf[NC][PARTS];
            // In f16 the factor vs / r of the weights goes into the exponent (a weight of nothing still counts 2^-60 there: its
            // column's sum divides by it), in f32 an addend of both would round more than p may.
            constexpr bool kInExponent = PARTS == 1;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                // (at most that, where any of it is seen)
                const float vs_per = fminf(pages.vs[i * PG / 4] * per[c], kWeight * kSlackV);
                const float vw = kInExponent ? fmaxf(vs_per, kWeight * 0x1p-60f) : vs_per;
                const float shift = kInExponent ? __builtin_amdgcn_logf(vw) : 0.0f;
                const float back = kInExponent ? __builtin_amdgcn_rcpf(vw) : 1.0f;
                const float off = shift - (m[c] == kNegInf ? 0.0f : m[c]);
                float y[8], sum[2] = {0.0f, 0.0f};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    // (unseen: 2^-inf = 0)
                    y[e] = exp2_fast(__builtin_fmaf(s[i / 2][c].v[8 * (i % 2) + e], f[c][i * PG / 4], off));
                    sum[e % 2] += y[e];
                    if (!kInExponent) y[e] *= vw;
                }
                lsum[c] = __builtin_fmaf(sum[0] + sum[1], back, lsum[c]);
                split_f16<PARTS>(y, wf[c]);
            }
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const int d = 32 * t + n;
                const f16x8 vf = *reinterpret_cast<const f16x8 *>(&s_v[buf][d * kRowV + swz_v(2 * i + hf, d)]);
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int p = 0; p < PARTS; ++p)
                        o[c][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, wf[c][p], o[c][t], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int i = 0; i < 4 * DT - kAhead; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, NC * PARTS, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, NC * PARTS * kAhead, 0);
    };

    if (begin < end) {
        Pages now, next, after;
        fetch(begin, now);
        load(begin, now);
        fetch(begin + 64, next);
        stage_k(0);
        stage_v(0);
        load(begin + 64, next);
        fetch(begin + 128, after);
        __syncthreads();
        // (two tiles a turn: each knows its half of LDS, which saves an addition a read, 2 us of the 158)
        auto tile = [&](int t0, auto which) __attribute__((always_inline)) {
            constexpr int buf = decltype(which)::value;
            // (a tile after, or wholly before the window of, all of the wave's columns is only staged)
            if (t0 <= pos_hi && (long)t0 + 63 > (long)pos_lo - a.window) use(t0, buf, now);
            stage_k(buf ^ 1);
            stage_v(buf ^ 1);
            now = next, next = after;
            load(t0 + 128, next);
            fetch(t0 + 192, after);
            __syncthreads();
        };
        for (int t0 = begin; t0 < end; t0 += 128) {
            tile(t0, std::integral_constant<int, 0>());
            if (t0 + 64 < end) tile(t0 + 64, std::integral_constant<int, 1>());
        }
    }

#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int col = w0 + 32 * c + n;
        const float lall = sum_halves(lsum[c]);
        if (col >= cols) continue;
        const int token = rq.first + col / a.grp, head = h * a.grp + col % a.grp;
        // (one after the other: their quotient can be too small for f32 where vref is)
        const float to_out = vref[c] * (kCodeScale / kWeight), inv = lall == 0.0f ? 0.0f : 1.0f / lall;
        const size_t at = ((size_t)token * a.n_heads + head) * a.pitch + split;
        typename T::raw *out = static_cast<typename T::raw *>(a.out) + (size_t)token * a.ot + (size_t)head * a.oh;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 32 * t + 8 * e + 4 * hf;
                if (d >= a.hd) continue;
                if (sp.active > 1) {
                    *reinterpret_cast<float4 *>(a.part_o + at * a.hd + d) = make_float4(
                        o[c][t][4 * e] * to_out, o[c][t][4 * e + 1] * to_out, o[c][t][4 * e + 2] * to_out,
                        o[c][t][4 * e + 3] * to_out);
                } else {
                    typename T::raw y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = T::down(o[c][t][4 * e + i] * to_out * inv);
                    if (a.out_vec) __builtin_memcpy(__builtin_assume_aligned(out + d, 4 * sizeof(y[0])), y, sizeof y);
                    else
#pragma unroll
                        for (int i = 0; i < 4; ++i) out[d + i] = y[i];
                }
            }
        if (sp.active > 1 && hf == 0) a.part_ml[at] = make_float2(m[c], lall);
    }
}

template <typename T, int HDP, int PARTS, int PG>
static void launch_prompt(hipStream_t s, dim3 grid, const AttnDev &d) {
    if constexpr (HDP <= 128) {
        if (d.tile_cols == 256) {
            hipLaunchKernelGGL((attn_q8_prompt_kernel<T, HDP, PARTS, 1, 8, PG>), grid, dim3(512), 0, s, d);
            return;
        }
    }
    hipLaunchKernelGGL((attn_q8_prompt_kernel<T, HDP, PARTS, 1, 4, PG>), grid, dim3(256), 0, s, d);
}
template <typename T, int PARTS, int PG>
static void launch_prompt(hipStream_t s, dim3 grid, const AttnDev &d) {
    if (d.hd <= 64) launch_prompt<T, 64, PARTS, PG>(s, grid, d);
    else if (d.hd <= 128) launch_prompt<T, 128, PARTS, PG>(s, grid, d);
    else launch_prompt<T, 256, PARTS, PG>(s, grid, d);
}
template <typename T, int PARTS>
static void launch_prompt(hipStream_t s, dim3 grid, const AttnDev &d) {
    if (d.page_shift >= 6) launch_prompt<T, PARTS, 1>(s, grid, d);
    else if (d.page_shift == 5) launch_prompt<T, PARTS, 2>(s, grid, d);
    else launch_prompt<T, PARTS, 4>(s, grid, d);
}

jk_status launch_attn_prompt(hipStream_t s, int dtype, const AttnDev &d) {
    const dim3 grid((unsigned)((size_t)d.n_requests * d.n_kv * d.tiles * d.splits));
    if (dtype == JK_F32) launch_prompt<F32, 2>(s, grid, d);
    else if (dtype == JK_F16) launch_prompt<F16, 1>(s, grid, d);
    else launch_prompt<BF16, 1>(s, grid, d);
    return check_launch("attn_q8_prompt_kernel");
}

}  // namespace jk
