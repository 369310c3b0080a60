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
    float *stats;   // [rows][segs][2]: maximum, sum of exp(x - maximum)
};

// The segment's logits of one lane, in pieces of 16 bytes: element i of the lane is token base + tok(i).
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
        if (__builtin_isnan(v[i])) v[i] = -__builtin_inff();
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

    // the width largest, one a round: each lane offers its best remaining key below the last one taken
    const size_t at = (size_t)row * a.segs + seg;
    key_t64 last = ~0ull;
    for (int b = 0; b < a.width; ++b) {
        key_t64 best = 0;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const key_t64 k = tok(i) < n ? argmax_key(v[i], (uint32_t)(base + tok(i))) : 0ull;
            best = k < last && k > best ? k : best;
        }
        best = wave_max_key(best);
        if (l == 0) a.keys[at * a.width + b] = best;
        last = best;
        if (best == 0) {
            for (int r = b + 1 + l; r < a.width; r += 64) a.keys[at * a.width + r] = 0;
            break;
        }
    }
    if (l == 0) a.stats[2 * at] = m, a.stats[2 * at + 1] = sum;
}

// One workgroup a group. A wave joins a row's segments: each lane holds the best untaken key of its segments
// (their lists are in order, so that is one position each), and the row's next best is the wave's maximum. Then the
// first wave joins the group's rows in the same way, by their totals.
constexpr int kJoinWaves = 8;
__global__ __launch_bounds__(64 * kJoinWaves) void beam_join_kernel(BeamDev a) {
    __shared__ float s_total[kMaxWidth][kMaxWidth];
    __shared__ int s_tok[kMaxWidth][kMaxWidth];
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6, g = blockIdx.x;
    for (int b = w; b < a.width; b += kJoinWaves) {
        const size_t row = (size_t)g * a.width + b;
        if (l < a.width) s_total[b][l] = -__builtin_inff(), s_tok[b][l] = -1;
        wave_lds_sync();
        if (a.done && a.done[row]) {
            if (l == 0) s_total[b][0] = a.scores[row], s_tok[b][0] = a.eos;
            continue;
        }
        const float *st = a.stats + 2 * row * a.segs;
        float m = -__builtin_inff();
        for (int i = l; i < a.segs; i += 64) m = fmaxf(m, st[2 * i]);
        m = wave_max64_dpp(m);
        float sum = 0.0f;
        for (int i = l; i < a.segs; i += 64)
            if (st[2 * i] > -__builtin_inff()) sum += st[2 * i + 1] * __builtin_amdgcn_exp2f((st[2 * i] - m) * kLog2e);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        const float lse = logf(sum), score = a.scores[row];
        const key_t64 *keys = a.keys + row * a.segs * a.width;
        key_t64 head[kMaxSegsPerLane];
        int taken[kMaxSegsPerLane];
#pragma unroll
        for (int i = 0; i < kMaxSegsPerLane; ++i) {
            taken[i] = 0;
            head[i] = l + 64 * i < a.segs ? keys[(size_t)(l + 64 * i) * a.width] : 0ull;
        }
        for (int r = 0; r < a.width; ++r) {
            key_t64 best = 0;
#pragma unroll
            for (int i = 0; i < kMaxSegsPerLane; ++i) best = head[i] > best ? head[i] : best;
            best = wave_max_key(best);
            if (best == 0) break;
            if (l == 0) {
                const float t = score + ((key_value(best) - m) - lse);
                s_total[b][r] = __builtin_isnan(t) ? -__builtin_inff() : t;
                s_tok[b][r] = key_token(best);
            }
#pragma unroll
            for (int i = 0; i < kMaxSegsPerLane; ++i)
                if (head[i] == best) {
                    ++taken[i];
                    head[i] = taken[i] < a.width ? keys[(size_t)(l + 64 * i) * a.width + taken[i]] : 0ull;
                }
        }
    }
    __syncthreads();
    if (w) return;
    // lane b offers row b's next candidate; keys order by total, then by the lower row (no NaN among totals)
    int next = 0;
    for (int r = 0; r < a.width; ++r) {
        const bool has = l < a.width && next < a.width && s_tok[l][next] >= 0;
        const key_t64 best = wave_max_key(has ? argmax_key(s_total[l][next], (uint32_t)l) : 0ull);
        const int b = key_token(best);  // (each row has a candidate and the first of a row comes first: best != 0)
        const int pos = __shfl(next, b, 64);
        const size_t out = (size_t)g * a.width + r;
        if (l == 0) {
            const int tok = s_tok[b][pos];
            a.scores_out[out] = s_total[b][pos];
            a.parents[out] = b;
            a.tokens[out] = tok;
            if (a.done_out) a.done_out[out] = (a.done && a.done[(size_t)g * a.width + b]) || tok == a.eos;
        }
        if (l == b) ++next;
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
              false, static_cast<key_t64 *>(ws), reinterpret_cast<float *>(static_cast<char *>(ws) + w.keys)};
    d.vec = (uintptr_t)a->logits % 16 == 0 && d.stride * es % 16 == 0;
    const size_t blocks = (w.rows * w.segs + 3) / 4;
    if (blocks >= (size_t)1 << 24) return fail(JK_TENSOR_BOUNDS, "beam_select: %zu rows of %zu logits are too many", w.rows, a->vocab);
    const dim3 grid((unsigned)blocks);
    if (a->dtype == JK_F32) hipLaunchKernelGGL(beam_rows_kernel<F32>, grid, dim3(256), 0, (hipStream_t)s, d);
    else if (a->dtype == JK_F16) hipLaunchKernelGGL(beam_rows_kernel<F16>, grid, dim3(256), 0, (hipStream_t)s, d);
    else hipLaunchKernelGGL(beam_rows_kernel<BF16>, grid, dim3(256), 0, (hipStream_t)s, d);
    JK_TRY(check_launch("beam_rows_kernel"));
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)a->groups), dim3(64 * kJoinWaves), 0, (hipStream_t)s, d);
    return check_launch("beam_join_kernel");
}

}  // extern "C"
