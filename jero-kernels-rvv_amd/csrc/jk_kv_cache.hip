// jk_kv_cache.hip -- a layer's attention cache in 8 bits: new keys and values into their pages, and
// stored ones back out.
//
// A page of one head has one scale d, and a value x is the code round(x / d). d is the largest |x| of the page's
// tokens over 127, so the codes use their whole range; it is known only when the page is full, so a page that
// is still being filled keeps the scale its tokens needed so far, and when a larger value comes, its codes are
// rescaled once: round(code * d_old / d). Each rescaling adds at most half a step of its own scale to an older value's
// error; the running maximum of a page's tokens grows about ln(page) times while it fills.
#include <algorithm>

#include "jk_device.hpp"

namespace jk {

constexpr float kTiny = 0x1p-119f;  // (1 / (kTiny / 127) is finite, and so is every x / d)

struct AppendArgs {
    int8_t *codes[2];  // k, v
    float *scale[2];
    const void *x[2];
    size_t st, sh;  // strides of x in elements
    const int32_t *slots;
    int n_tokens, n_slots, n_kv, hd, page_shift;
    int chunk;  // tokens whose runs a workgroup takes, at most 64
    bool vec;
};

// |x| where it is finite, else 0: what a stored element is.
__device__ __forceinline__ float kept(float x) { return __builtin_isfinite(x) ? x : 0.0f; }

// Tokens t0, t0 + 1, .. of one page with rising rows, as far as they go: at most a page. Every wave of the
// workgroup finds the same number by itself.
__device__ __forceinline__ int run_length(const AppendArgs &a, int t0) {
    const int l = threadIdx.x & 63, page = a.slots[t0] >> a.page_shift;
    for (int base = 0;; base += 64) {
        const int t = t0 + base + l;
        bool goes_on = base + l == 0;
        if (!goes_on && t < a.n_tokens) {
            const int s = a.slots[t];
            goes_on = s >= 0 && (s >> a.page_shift) == page && s > a.slots[t - 1];
        }
        const unsigned long long stop = ~__ballot(goes_on);
        if (stop) return base + __builtin_ctzll(stop);
    }
}

// Quantizes the runs of tokens of one page that begin among tokens [chunk * x, chunk * (x + 1)) for one head
// of keys or values (blockIdx.y). One pass over the new values where the run's 8-element pieces fit kHeld a thread,
// else a second one from the caches. What bounds it: the values read and the codes written once (a page's old codes twice
// more where it is rescaled). 9360 tokens of prompts, f32, 8 heads of 128: 96 MB in 24 us, 3.9 TB/s of the 5.3 that a copy
// reaches; a step of 48 requests 4.2 us, a launch and three rounds of loads.
// A decode step has one-token runs in as many pages as requests, a prompt runs of whole pages, and the host does not know
// which a call is. Up to 1024 tokens a workgroup takes one token by 64 threads (bf16, 8 heads of 128: a step of 1024 requests 58 us,
// 132 by runs of a page; a prompt of 1024 tokens 16.7 and 17.5), beyond that a 512th of the tokens, up to a page, by 256 threads
// (a step of 2000 requests 132 us with 4 tokens, 181 with 64; 16 prompts of 2000 tokens 65 us with 64, 125 with 4).
constexpr int kHeld = 4;
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void kv_append_kernel(AppendArgs a) {
    typedef typename T::raw raw;
    __shared__ float s_max[THREADS / 64];
    const int tid = threadIdx.x, l = tid & 63, which = blockIdx.y / a.n_kv, h = blockIdx.y % a.n_kv;
    const int t_first = blockIdx.x * a.chunk;
    const raw *x = static_cast<const raw *>(a.x[which]);

    // which of the chunk's tokens begin a run
    bool begins = false;
    const int t = t_first + l;
    if (l < a.chunk && t < a.n_tokens) {
        const int s = a.slots[t], before = t ? a.slots[t - 1] : -1;
        begins = (unsigned)s < (unsigned)a.n_slots &&
                 !(before >= 0 && (before >> a.page_shift) == (s >> a.page_shift) && s > before);
    }
    unsigned long long starts = __ballot(begins);

    const int hv = a.hd / 8, page = 1 << a.page_shift;
    while (starts) {
        const int t0 = t_first + __builtin_ctzll(starts);
        starts &= starts - 1;
        const int n = run_length(a, t0), s0 = a.slots[t0], row0 = s0 & (page - 1);
        const size_t head = (size_t)(s0 >> a.page_shift) * a.n_kv + h;
        int8_t *codes = a.codes[which] + (head << a.page_shift) * a.hd;

        float held[kHeld][8], top = 0.0f;
        const int pieces = n * hv;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int v = tid + i * THREADS;
            if (v < pieces) {
                load_up<T, 8>(x + (size_t)(t0 + v / hv) * a.st + (size_t)h * a.sh + (v % hv) * 8, a.vec, held[i]);
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(kept(held[i][e])));
            }
        }
        for (int v = tid + kHeld * THREADS; v < pieces; v += THREADS) {
            float y[8];
            load_up<T, 8>(x + (size_t)(t0 + v / hv) * a.st + (size_t)h * a.sh + (v % hv) * 8, a.vec, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(kept(y[e])));
        }
        // (row 0 begins the page: whatever scale it held before is of no account)
        float old = row0 ? a.scale[which][head] : 0.0f;
        old = __builtin_isfinite(old) && old > 0.0f ? old : 0.0f;
        top = wave_max64_dpp(top);
        if constexpr (THREADS > 64) {
            __syncthreads();  // (the last run's maxima have been read)
            if (l == 0) s_max[tid >> 6] = top;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < THREADS / 64; ++i) top = fmaxf(top, s_max[i]);
        }
        const float d = fmaxf(old, top < kTiny ? 0.0f : top / 127.0f);
        const float inv = d > 0.0f ? 1.0f / d : 0.0f;

        auto store = [&](int v, const float *y) {
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float q = fminf(fmaxf(rintf(kept(y[e]) * inv), -127.0f), 127.0f);
                w[e / 4] |= (uint32_t)((int)q & 255) << (8 * (e % 4));
            }
            const int row = a.slots[t0 + v / hv] & (page - 1);
            *reinterpret_cast<uint2 *>(codes + (size_t)row * a.hd + (v % hv) * 8) = make_uint2(w[0], w[1]);
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (tid + i * THREADS < pieces) store(tid + i * THREADS, held[i]);
        for (int v = tid + kHeld * THREADS; v < pieces; v += THREADS) {
            float y[8];
            load_up<T, 8>(x + (size_t)(t0 + v / hv) * a.st + (size_t)h * a.sh + (v % hv) * 8, a.vec, y);
            store(v, y);
        }
        if (row0 && d != old) {
            const float ratio = old / d;
            for (int i = tid; i < row0 * (a.hd / 16); i += THREADS) {
                u32x4 *at = reinterpret_cast<u32x4 *>(codes) + i;
                u32x4 v = *at;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t w = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // |code| <= 128 (a code the library did not write) and ratio < 1: it stays a code
                        const float q = rintf((float)(int8_t)(v[k] >> (8 * e)) * ratio);
                        w |= (uint32_t)((int)q & 255) << (8 * e);
                    }
                    v[k] = w;
                }
                *at = v;
            }
        }
        if (tid == 0) a.scale[which][head] = d;
    }
}

// A thread turns the codes of 16 bytes of output (4 or 8) of one head and slot into values, four of them 256 apart with their
// loads in flight together; blockIdx.y: keys, values. 9360 slots, 8 heads of 128, to f32: 96 MB in 18 us, 5.3 TB/s.
constexpr int kReadPieces = 4;
struct ReadArgs {
    const int8_t *codes[2];
    const float *scale[2];
    void *out[2];
    const int32_t *slots;
    unsigned pieces;  // of 16 bytes of output
    int n_slots, n_kv, hd, page_shift;
    bool vec;
};
template <typename T>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a) {
    typedef typename T::raw raw;
    constexpr int N = 16 / (int)sizeof(raw);
    const int8_t *codes = a.codes[blockIdx.y];
    const float *scale = a.scale[blockIdx.y];
    raw *out = static_cast<raw *>(a.out[blockIdx.y]);
    if (!out) return;
    const unsigned first = blockIdx.x * (256 * kReadPieces) + threadIdx.x, per = a.hd / N;
    uint32_t w[kReadPieces][N / 4];
    float d[kReadPieces];
#pragma unroll
    for (int k = 0; k < kReadPieces; ++k) {
        const unsigned i = min(first + 256 * k, a.pieces - 1), head_of = i / per, c = (i - head_of * per) * N;
        const unsigned at = head_of / a.n_kv, h = head_of - at * a.n_kv;
        const int s = a.slots[at];
        const bool ok = (unsigned)s < (unsigned)a.n_slots;
        const size_t head = ok ? (size_t)(s >> a.page_shift) * a.n_kv + h : 0;
        const size_t place = ((head << a.page_shift) + (ok ? s & ((1 << a.page_shift) - 1) : 0)) * a.hd + c;
        __builtin_memcpy(w[k], __builtin_assume_aligned(codes + place, N), N);
        d[k] = scale[head];
        if (!ok) {  // (whatever its scale: 0 even beside an infinite one)
            d[k] = 0.0f;
#pragma unroll
            for (int e = 0; e < N / 4; ++e) w[k][e] = 0;
        }
    }
#pragma unroll
    for (int k = 0; k < kReadPieces; ++k) {
        const unsigned i = first + 256 * k;
        if (i >= a.pieces) return;
        raw y[N];
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = T::down((float)(int8_t)(w[k][e / 4] >> (8 * (e % 4))) * d[k]);
        raw *to = out + (size_t)i * N;
        if (a.vec) {
            u32x4 v;
            __builtin_memcpy(&v, y, 16);
            __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(to));  // (the caller's to read, not this launch's)
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) to[e] = y[e];
        }
    }
}

jk_status kv_check(const char *what, const jk_kv_q8 *c) {
    if (!c) return fail(JK_TENSOR_BOUNDS, "%s: null cache", what);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(JK_TENSOR_BOUNDS, "%s: null array in the cache", what);
    if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16)
        return fail(JK_TENSOR_BOUNDS, "%s: the cache's codes must be 16-byte aligned", what);
    if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1)))
        return fail(JK_TENSOR_BOUNDS, "%s: %zu tokens a page: 16, 32, 64, 128 or 256", what, c->page);
    if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16)
        return fail(JK_CAPABILITY_MISMATCH, "%s: head dimension %zu: a multiple of 16 from 16 to 256", what, c->head_dim);
    if (c->n_kv == 0 || c->n_kv > 4096) return fail(JK_TENSOR_BOUNDS, "%s: %zu kv heads: 1..4096", what, c->n_kv);
    if (c->n_pages == 0 || c->n_pages > (size_t)INT32_MAX / c->page)
        return fail(JK_TENSOR_BOUNDS, "%s: %zu pages of %zu tokens exceed the int32 range of slots", what, c->n_pages,
                    c->page);
    if (c->n_pages * c->n_kv > (size_t)INT32_MAX)
        return fail(JK_TENSOR_BOUNDS, "%s: %zu pages of %zu kv heads exceed the int32 range", what, c->n_pages, c->n_kv);
    return JK_OK;
}

template <typename T>
static void launch_append(hipStream_t s, AppendArgs a) {
    const bool step = a.n_tokens <= 1024;
    a.chunk = step ? 1 : std::min({64, 1 << a.page_shift, a.n_tokens / 512});
    const dim3 grid((unsigned)((a.n_tokens + a.chunk - 1) / a.chunk), 2 * (unsigned)a.n_kv);
    if (step) hipLaunchKernelGGL((kv_append_kernel<T, 64>), grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL((kv_append_kernel<T, 256>), grid, dim3(256), 0, s, a);
}

}  // namespace jk

using namespace jk;

extern "C" {

jk_status jk_kv_append_q8(jk_stream s, const jk_kv_q8 *c, const void *k, const void *v, int dtype, size_t n_tokens,
                          size_t stride_token, size_t stride_head, const int32_t *slots) {
    JK_TRY(kv_check("kv_append_q8", c));
    if (!dtype_ok(dtype)) return fail(JK_CAPABILITY_MISMATCH, "kv_append_q8: unknown element type %d", dtype);
    if (n_tokens == 0) return JK_OK;
    if (!k || !v || !slots) return fail(JK_TENSOR_BOUNDS, "kv_append_q8: null keys, values or slots");
    const size_t es = dtype_bytes(dtype);
    if ((uintptr_t)k % es || (uintptr_t)v % es)
        return fail(JK_TENSOR_BOUNDS, "kv_append_q8: keys and values must be aligned to their elements");
    if (n_tokens > (size_t)1 << 27)
        return fail(JK_TENSOR_BOUNDS, "kv_append_q8: %zu tokens are too many for one call", n_tokens);
    const size_t sh = stride_head ? stride_head : c->head_dim, st = stride_token ? stride_token : c->n_kv * c->head_dim;
    const bool vec = !((uintptr_t)k % 16) && !((uintptr_t)v % 16) && st * es % 16 == 0 && sh * es % 16 == 0;
    int shift = 4;
    while (((size_t)1 << shift) < c->page) ++shift;
    const AppendArgs a{{c->k, c->v}, {c->k_scale, c->v_scale}, {k, v}, st, sh, slots, (int)n_tokens,
                       (int)(c->n_pages * c->page), (int)c->n_kv, (int)c->head_dim, shift, 1, vec};
    if (dtype == JK_F32) launch_append<F32>((hipStream_t)s, a);
    else if (dtype == JK_F16) launch_append<F16>((hipStream_t)s, a);
    else launch_append<BF16>((hipStream_t)s, a);
    return check_launch("kv_append_kernel");
}

jk_status jk_kv_read_q8(jk_stream s, const jk_kv_q8 *c, const int32_t *slots, size_t n, int dtype, void *k_out,
                        void *v_out) {
    JK_TRY(kv_check("kv_read_q8", c));
    if (!dtype_ok(dtype)) return fail(JK_CAPABILITY_MISMATCH, "kv_read_q8: unknown element type %d", dtype);
    if (n == 0 || (!k_out && !v_out)) return JK_OK;
    if (!slots) return fail(JK_TENSOR_BOUNDS, "kv_read_q8: null slots");
    const size_t es = dtype_bytes(dtype);
    if ((uintptr_t)k_out % es || (uintptr_t)v_out % es)
        return fail(JK_TENSOR_BOUNDS, "kv_read_q8: outputs must be aligned to their elements");
    const size_t per = c->n_kv * c->head_dim * es / 16;
    if (n > (size_t)INT32_MAX / per) return fail(JK_TENSOR_BOUNDS, "kv_read_q8: %zu slots are too many for one call", n);
    int shift = 4;
    while (((size_t)1 << shift) < c->page) ++shift;
    const ReadArgs a{{c->k, c->v}, {c->k_scale, c->v_scale}, {k_out, v_out}, slots, (unsigned)(n * per),
                     (int)(c->n_pages * c->page), (int)c->n_kv, (int)c->head_dim, shift,
                     !((uintptr_t)k_out % 16) && !((uintptr_t)v_out % 16)};
    const dim3 grid((unsigned)((n * per + 256 * kReadPieces - 1) / (256 * kReadPieces)), 2);
    if (dtype == JK_F32) hipLaunchKernelGGL(kv_read_kernel<F32>, grid, dim3(256), 0, (hipStream_t)s, a);
    else if (dtype == JK_F16) hipLaunchKernelGGL(kv_read_kernel<F16>, grid, dim3(256), 0, (hipStream_t)s, a);
    else hipLaunchKernelGGL(kv_read_kernel<BF16>, grid, dim3(256), 0, (hipStream_t)s, a);
    return check_launch("kv_read_kernel");
}

}  // extern "C"
