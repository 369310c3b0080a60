// jk_beam.hip -- one step of beam search: the best continuations of each group's hypotheses.
//
// total = score + (x - m - log(sum exp(x - m))) is monotone in the logit x within one row, so a row's candidates are its
// largest logits, and a group's best are among its rows' best. One pass over the logits: each wave takes a
// segment of a row, its maximum and sum of exponentials, and the segment's `width` largest logits as 64-bit keys (value order
// in the high word, ~token in the low one: equal logits rank by the lower token, and no two keys are equal). A second,
// small launch joins a row's segments and then a group's rows.
#include <algorithm>

#include "jk_device.hpp"

namespace jk {

typedef unsigned long long key_t64;
constexpr int kSeg = 2048;                // logits a wave takes
constexpr int kPerLane = kSeg / 64;
constexpr int kMaxSegsPerLane = 8;        // a row has at most 64 * 8 segments: vocab up to 2^20
constexpr int kMaxWidth = 32;
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float key_value(key_t64 k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ int key_token(key_t64 k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }

// Largest key of the wave (all lanes active) by lane permutations: of the high words, then of the low words beside it. (The
// shuffles of wave_max_key go through LDS: three times the latency, and a round of the joins is little else.)
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = max(v, (uint32_t)dpp_i<kDppXor1>((int)v));
    v = max(v, (uint32_t)dpp_i<kDppXor2>((int)v));
    v = max(v, (uint32_t)dpp_i<kDppHalfMirror>((int)v));
    v = max(v, (uint32_t)dpp_i<kDppMirror>((int)v));
    const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)v, 0), b = (uint32_t)__builtin_amdgcn_readlane((int)v, 16);
    const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)v, 32), e = (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
    return max(max(a, b), max(c, e));
}
__device__ __forceinline__ key_t64 max_key(key_t64 k) {
    const uint32_t hi = wave_max_u32((uint32_t)(k >> 32));
    const uint32_t lo = wave_max_u32((uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return ((key_t64)hi << 32) | lo;
}

struct BeamDev {
    const void *logits;
    const float *scores;
    const int32_t *done;
    float *scores_out;
    int32_t *parents, *tokens, *done_out;
    size_t stride;
    int groups, width, vocab, eos, segs;
    bool vec;
    key_t64 *keys;  // [rows][segs][width], largest first
    float2 *stats;  // [rows][segs]: maximum, sum of exp(x - maximum)
};

// The segment's logits of one lane, in pieces of 16 bytes: element i of the lane is token base + tok(i).
// What bounds it: the logits, read once and held in registers between the maximum, the sum and the selection. 128 rows of 128256 in
// f32: 66 MB in 17.5 us, 3.8 TB/s; 4 rows of 32000 6.3 us, one wave's latency. Segments of 2048 give 63 waves a row, so that one
// request's few rows already reach many CUs, and leave 32 logits a lane.
template <typename T>
__global__ __launch_bounds__(256) void beam_rows_kernel(BeamDev a) {
    typedef typename T::raw raw;
    constexpr int per = 16 / (int)sizeof(raw);  // elements of a piece
    const int l = threadIdx.x & 63;
    const long unit = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long row = unit / a.segs;
    const int seg = (int)(unit - row * a.segs);
    if (row >= (long)a.groups * a.width) return;
    if (a.done && a.done[row]) return;  // (goes on as itself: its logits are not looked at)
    const raw *x = static_cast<const raw *>(a.logits) + (size_t)row * a.stride;
    const int base = seg * kSeg, n = min(kSeg, a.vocab - base);
    auto tok = [&](int i) { return (i / per) * (64 * per) + l * per + i % per; };

    float v[kPerLane];
    if (a.vec && n == kSeg) {
#pragma unroll
        for (int i = 0; i < kPerLane; i += per) {
            const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(x + base + tok(i)));
            raw e[per];
            __builtin_memcpy(e, &w, 16);
#pragma unroll
            for (int j = 0; j < per; ++j) v[i + j] = T::up(e[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) v[i] = tok(i) < n ? T::up(x[base + tok(i)]) : -__builtin_inff();
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        v[i] = fmaxf(v[i], -__builtin_inff());  // (a NaN counts as -inf)
        top = fmaxf(top, v[i]);
    }
    const float m = wave_max64_dpp(top);
    float sum = 0.0f;
    if (m > -__builtin_inff()) {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) sum += __builtin_amdgcn_exp2f((v[i] - m) * kLog2e);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);

    // The width largest. At least `width` logits are no smaller than the width-th largest of the lanes' maxima, and for
    // logits that are not almost all equal hardly more: those are collected and ranked by counting, each
    // lane one of them. Where there are more than lanes, the largest are taken one a round instead.
    const size_t at = (size_t)row * a.segs + seg;
    float bar = m, rest = top;
    for (int have = 0;;) {
        have += __popcll(__ballot(rest == bar));
        if (have >= a.width || bar == -__builtin_inff()) break;
        rest = rest == bar ? -__builtin_inff() : rest;
        bar = wave_max64_dpp(rest);
    }
    __shared__ key_t64 s_keys[4][64];
    key_t64 *keys = s_keys[threadIdx.x >> 6];
    int n_keys = 0;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const bool in = v[i] >= bar && tok(i) < n;
        const unsigned long long mask = __ballot(in);
        if (mask) {
            const int to = n_keys + __popcll(mask & ((1ull << l) - 1));
            if (in && to < 64) keys[to] = argmax_key(v[i], (uint32_t)(base + tok(i)));
            n_keys += __popcll(mask);
        }
    }
    if (n_keys <= 64) {
        wave_lds_sync();
        const key_t64 mine = l < n_keys ? keys[l] : 0ull;
        int rank = 0;
        for (int i = 0; i < n_keys; ++i) rank += keys[i] > mine;
        if (l < n_keys && rank < a.width) a.keys[at * a.width + rank] = mine;
        if (l >= n_keys && l < a.width) a.keys[at * a.width + l] = 0;
    } else {
        key_t64 last = ~0ull;
        for (int b = 0; b < a.width; ++b) {
            key_t64 best = 0;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
                const key_t64 k = tok(i) < n ? argmax_key(v[i], (uint32_t)(base + tok(i))) : 0ull;
                best = k < last && k > best ? k : best;
            }
            last = max_key(best);
            if (l == 0) a.keys[at * a.width + b] = last;
        }
    }
    if (l == 0) a.stats[at] = make_float2(m, sum);
}

// One workgroup a group. A wave joins a row's segments: each lane holds the best untaken key of its segments
// (their lists are in order, so that is one position each), and the row's next best is the wave's maximum. Then the
// first wave joins the group's rows in the same way, by their totals.
// The keys are staged in LDS where a row has at most kJoinKeys of them (a vocabulary of 256k at a width of 8): a round's next key
// then comes at LDS latency.
// What bounds it: `width` rounds twice, each a maximum over the wave and the next key behind it; 16 groups of 8 rows of 63
// segments 8 us, one of 4 rows 5.
constexpr int kJoinWaves = 8, kJoinKeys = 1024;
template <int NS>  // segments a lane holds (64 * NS at most)
__global__ __launch_bounds__(64 * kJoinWaves) void beam_join_kernel(BeamDev a) {
    __shared__ float s_total[kMaxWidth][kMaxWidth];
    __shared__ int s_tok[kMaxWidth][kMaxWidth];
    __shared__ key_t64 s_keys[kJoinWaves][kJoinKeys];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6, g = blockIdx.x;
    for (int b = w; b < a.width; b += kJoinWaves) {
        const size_t row = (size_t)g * a.width + b;
        if (l < a.width) s_total[b][l] = -__builtin_inff(), s_tok[b][l] = -1;
        wave_lds_sync();
        if (a.done && a.done[row]) {
            const float t = a.scores[row];
            if (l == 0) s_total[b][0] = __builtin_isnan(t) ? -__builtin_inff() : t, s_tok[b][0] = a.eos;
            continue;
        }
        const float score = a.scores[row];
        const key_t64 *keys = a.keys + row * a.segs * a.width;
        float2 st[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i)
            st[i] = l + 64 * i < a.segs ? a.stats[row * a.segs + l + 64 * i] : make_float2(-__builtin_inff(), 0.0f);
        // (the staging's loads go out together, and before the sums are looked at)
        const int n_keys = a.segs * a.width;
        if (n_keys <= kJoinKeys) {
            key_t64 some[kJoinKeys / 64];
#pragma unroll
            for (int i = 0; i < kJoinKeys / 64; ++i)
                if (64 * i < n_keys) some[i] = keys[min(l + 64 * i, n_keys - 1)];
#pragma unroll
            for (int i = 0; i < kJoinKeys / 64; ++i)
                if (64 * i < n_keys) s_keys[w][l + 64 * i] = some[i];
            wave_lds_sync();
            keys = s_keys[w];
        }
        float m = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NS; ++i) m = fmaxf(m, st[i].x);
        m = wave_max64_dpp(m);
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (st[i].x > -__builtin_inff()) sum += st[i].y * __builtin_amdgcn_exp2f((st[i].x - m) * kLog2e);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        const float lse = logf(sum);
        key_t64 head[NS];
        int taken[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            taken[i] = 0;
            head[i] = l + 64 * i < a.segs ? keys[(size_t)(l + 64 * i) * a.width] : 0ull;
        }
        for (int r = 0; r < a.width; ++r) {
            key_t64 best = 0;
#pragma unroll
            for (int i = 0; i < NS; ++i) best = head[i] > best ? head[i] : best;
            best = max_key(best);
            if (best == 0) break;
            if (l == 0) {
                const float t = score + ((key_value(best) - m) - lse);
                s_total[b][r] = __builtin_isnan(t) ? -__builtin_inff() : t;
                s_tok[b][r] = key_token(best);
            }
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (head[i] == best) {
                    ++taken[i];
                    head[i] = taken[i] < a.width ? keys[(size_t)(l + 64 * i) * a.width + taken[i]] : 0ull;
                }
        }
    }
    __syncthreads();
    if (w) return;
    // lane b offers row b's next candidate (keys order by total, then by the lower row; no NaN among totals), and lane r keeps what
    // comes out r-th
    const size_t row0 = (size_t)g * a.width;
    const bool mine_done = l < a.width && a.done && a.done[row0 + l];
    auto offer = [&](int at) {
        const bool has = l < a.width && at < a.width && s_tok[l][at] >= 0;
        return has ? argmax_key(s_total[l][at], (uint32_t)l) : 0ull;
    };
    int next = 0, parent = 0, pos = 0;
    key_t64 key = offer(0);
    for (int r = 0; r < a.width; ++r) {
        const int b = key_token(max_key(key));  // (each row has a candidate and the first of a row comes first: there is one)
        const int at = __builtin_amdgcn_readlane(next, b);
        if (l == r) parent = b, pos = at;
        if (l == b) key = offer(++next);
    }
    const int ended = __shfl((int)mine_done, parent, 64);
    if (l < a.width) {
        const int tok = s_tok[parent][pos];
        a.scores_out[row0 + l] = s_total[parent][pos];
        a.parents[row0 + l] = parent;
        a.tokens[row0 + l] = tok;
        if (a.done_out) a.done_out[row0 + l] = ended || tok == a.eos;
    }
}

struct BeamWs {
    size_t segs, rows, keys, bytes;
};
static BeamWs beam_ws(const jk_beam_args *a) {
    BeamWs w;
    w.segs = (a->vocab + kSeg - 1) / kSeg;
    w.rows = a->groups * a->width;
    w.keys = w.rows * w.segs * a->width * sizeof(key_t64);
    w.bytes = w.keys + w.rows * w.segs * 2 * sizeof(float);
    return w;
}

static jk_status beam_check(const jk_beam_args *a) {
    if (!a) return fail(JK_TENSOR_BOUNDS, "beam_select: null arguments");
    if (!dtype_ok(a->dtype)) return fail(JK_CAPABILITY_MISMATCH, "beam_select: unknown element type %d", a->dtype);
    if (a->width == 0 || a->width > (size_t)kMaxWidth)
        return fail(JK_TENSOR_BOUNDS, "beam_select: width %zu: 1..%d", a->width, kMaxWidth);
    if (a->vocab == 0 || a->vocab > (size_t)kSeg * 64 * kMaxSegsPerLane)
        return fail(JK_CAPABILITY_MISMATCH, "beam_select: %zu logits a row: 1..%d", a->vocab,
                    kSeg * 64 * kMaxSegsPerLane);
    if (a->groups == 0 || a->groups > (size_t)1 << 16)
        return fail(JK_TENSOR_BOUNDS, "beam_select: %zu groups: 1..65536", a->groups);
    if (a->stride && a->stride < a->vocab)
        return fail(JK_TENSOR_BOUNDS, "beam_select: stride %zu < %zu logits a row", a->stride, a->vocab);
    return JK_OK;
}

}  // namespace jk

using namespace jk;

extern "C" {

size_t jk_beam_workspace_bytes(const jk_beam_args *a) { return beam_check(a) == JK_OK ? beam_ws(a).bytes : 0; }

jk_status jk_beam_select(jk_stream s, const jk_beam_args *a, void *ws, size_t ws_bytes) {
    JK_TRY(beam_check(a));
    if (!a->logits || !a->scores || !a->scores_out || !a->parents || !a->tokens)
        return fail(JK_TENSOR_BOUNDS, "beam_select: null logits, scores or output");
    if (a->done && (a->eos < 0 || (size_t)a->eos >= a->vocab))
        return fail(JK_TENSOR_BOUNDS, "beam_select: token %d does not finish hypotheses of %zu tokens", a->eos, a->vocab);
    if (a->scores_out == a->scores || (a->done_out && a->done_out == a->done))
        return fail(JK_TENSOR_BOUNDS, "beam_select: an output is the array it is computed from");
    const size_t es = dtype_bytes(a->dtype);
    if ((uintptr_t)a->logits % es) return fail(JK_TENSOR_BOUNDS, "beam_select: logits must be aligned to their elements");
    const BeamWs w = beam_ws(a);
    if (!ws || (uintptr_t)ws % 16 || ws_bytes < w.bytes)
        return fail(JK_TENSOR_BOUNDS, "beam_select: workspace of %zu bytes at %p: %zu needed, 16-byte aligned", ws_bytes,
                    ws, w.bytes);
    BeamDev d{a->logits, a->scores, a->done, a->scores_out, a->parents, a->tokens, a->done_out,
              a->stride ? a->stride : a->vocab, (int)a->groups, (int)a->width, (int)a->vocab, (int)a->eos, (int)w.segs,
              false, static_cast<key_t64 *>(ws), reinterpret_cast<float2 *>(static_cast<char *>(ws) + w.keys)};
    d.vec = (uintptr_t)a->logits % 16 == 0 && d.stride * es % 16 == 0;
    const size_t blocks = (w.rows * w.segs + 3) / 4;
    if (blocks >= (size_t)1 << 24) return fail(JK_TENSOR_BOUNDS, "beam_select: %zu rows of %zu logits are too many", w.rows, a->vocab);
    const dim3 grid((unsigned)blocks);
    if (a->dtype == JK_F32) hipLaunchKernelGGL(beam_rows_kernel<F32>, grid, dim3(256), 0, (hipStream_t)s, d);
    else if (a->dtype == JK_F16) hipLaunchKernelGGL(beam_rows_kernel<F16>, grid, dim3(256), 0, (hipStream_t)s, d);
    else hipLaunchKernelGGL(beam_rows_kernel<BF16>, grid, dim3(256), 0, (hipStream_t)s, d);
    JK_TRY(check_launch("beam_rows_kernel"));
    const dim3 joins((unsigned)a->groups);
    if (w.segs <= 64) hipLaunchKernelGGL(beam_join_kernel<1>, joins, dim3(64 * kJoinWaves), 0, (hipStream_t)s, d);
    else hipLaunchKernelGGL(beam_join_kernel<kMaxSegsPerLane>, joins, dim3(64 * kJoinWaves), 0, (hipStream_t)s, d);
    return check_launch("beam_join_kernel");
}

}  // extern "C"
