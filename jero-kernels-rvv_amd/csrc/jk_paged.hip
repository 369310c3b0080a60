// jk_paged.hip -- the pages of a batch's attention cache: which page and slot each token of a step
// goes to, the free pages' stack, and the rows' reordering after a beam search step.
//
// Everything that decides (prefix sums over the requests, whether a step fits) runs in one workgroup, so
// a step's plan is one short launch with no hand-over between workgroups; only the per-token and
// per-column writing of larger steps is spread over a second launch. All indices that come from
// device memory are checked before they are used.
#include <algorithm>

#include "jk_device.hpp"

namespace jk {

constexpr int kPagedThreads = 1024;  // requests a pass of the planning workgroup takes

struct PagedDev {
    int n_requests, max_pages, n_pages, page_shift;
    int32_t *lens, *table, *owned, *free_pages, *n_free;
};

__device__ __forceinline__ int pages_of(int tokens, int shift) { return (int)(((long)tokens + (1 << shift) - 1) >> shift); }

// The page that an entry of `owned` stands for, or -1. An id is a page of the row where its place lies below the pages that the
// row's tokens reach (`used`); past them it is left of a step that was dropped, and that page is on the stack or somebody else's.
// -2 - id is a page that the row began and then went back from, to the place's first token, by a reordering: nobody reads it, and
// the row begins it again when it comes back.
__device__ __forceinline__ int owned_page(int v, bool used) { return v <= -2 ? -2 - v : used ? v : -1; }

// Exclusive prefix sum over the workgroup of one value per thread (the low and high words of v
// are summed apart: the callers' sums stay below 2^31). *total gets the sum. s: 17 words of LDS.
__device__ __forceinline__ unsigned long long wg_scan(unsigned long long v, unsigned long long *s,
                                                      unsigned long long *total) {
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    unsigned long long inc = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long t = __shfl_up(inc, o, 64);
        if (l >= o) inc += t;
    }
    __syncthreads();
    if (l == 63) s[w] = inc;
    __syncthreads();
    unsigned long long base = 0, sum = 0;
    for (int i = 0; i < (int)blockDim.x / 64; ++i) {
        if (i < w) base += s[i];
        sum += s[i];
    }
    *total = sum;
    return base + inc - v;
}

// Sums over the workgroup of N values per thread, with one pair of barriers. s: 17 * N words of LDS.
template <int N>
__device__ __forceinline__ void wg_sums(long (&v)[N], long *s) {
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v[k] += __shfl_xor(v[k], o, 64);
    __syncthreads();
    if (l == 0)
#pragma unroll
        for (int k = 0; k < N; ++k) s[w * N + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        v[k] = 0;
        for (int i = 0; i < (int)blockDim.x / 64; ++i) v[k] += s[i * N + k];
    }
}

// Largest r with start[r] <= t among start[0..n) (start[0] <= t).
template <typename P>
__device__ __forceinline__ int owner_of(const P *start, int n, int t) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int)start[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

struct StepDev {
    int max_tokens;
    int32_t *q_start, *slots, *positions, *requests, *status;
};

__device__ __forceinline__ void write_token(const StepDev &st, int t, int slot, int pos, int r) {
    st.slots[t] = slot;
    st.positions[t] = pos;
    st.requests[t] = r;
}

// The plan of a step by TH threads. FILL: this launch also numbers the tokens (few of them: one launch for a decode step).
// Its bytes are a few a request; what it takes is the latency of its rounds: the counts, their sums over the
// workgroup, a page's place found by bisection, the stack. A step of 4 requests 4.4 us, 96 prompts (49 thousand tokens, 1500
// pages) 8 us and their numbering 3.5, 128 requests of 7990 tokens (16 thousand pages, the largest share two stores a page)
// 19 and 7.5.
template <bool FILL, int TH>
__global__ __launch_bounds__(TH) void paged_extend_kernel(PagedDev p, const int32_t *__restrict__ n_new,
                                                                     StepDev st, int32_t *lens_out,
                                                                     int32_t *n_free_out) {
    __shared__ unsigned long long s_scan[17];
    __shared__ long s_sum[17 * 3];
    __shared__ int s_tok[TH + 1], s_pg[TH + 1], s_len[TH], s_kept[TH];
    const int tid = threadIdx.x, page = 1 << p.page_shift;
    const long cap = (long)p.max_pages << p.page_shift;
    const int n_free = *p.n_free;
    // the page that request r, about to begin its place j, has there already, or -1 (one array for both: there are none)
    auto kept_at = [&](int r, int j) -> int {
        const int v = p.owned == p.table ? -1 : p.owned[(size_t)r * p.max_pages + j];
        return page_ok(owned_page(v, false), p.n_pages) ? owned_page(v, false) : -1;
    };

    // does the step fit? (totals in 64 bits: counts are not trusted yet)
    long tokens = 0, pages = 0, bad = (n_free < 0 || n_free > p.n_pages), over = 0;
    for (int r = tid; r < p.n_requests; r += TH) {
        const long len = p.lens[r], n = n_new[r];
        if (len < 0 || n < 0 || len > cap) {
            bad = 1;
            continue;
        }
        if (len + n > cap) over = 1;
        tokens += n;
        const long held = (len + page - 1) >> p.page_shift, more = ((len + n + page - 1) >> p.page_shift) - held;
        pages += more;
        if (more && held < p.max_pages && kept_at(r, (int)held) >= 0) --pages;
    }
    long sums[3] = {tokens, pages, bad | (over << 32)};
    wg_sums(sums, s_sum);
    tokens = sums[0], pages = sums[1];
    const long flags = sums[2];
    const int status = (flags & 0xFFFFFFFFl) ? JK_PAGED_BAD_LENGTH
                       : (flags >> 32) || tokens > st.max_tokens ? JK_PAGED_TOO_LONG
                       : pages > n_free                          ? JK_PAGED_NO_PAGES
                                                                 : JK_PAGED_OK;
    if (tid == 0) {
        *st.status = status;
        *n_free_out = status == JK_PAGED_OK ? n_free - (int)pages : n_free;
    }
    if (status != JK_PAGED_OK) {
        for (int r = tid; r < p.n_requests; r += TH) {
            st.q_start[r] = 0;
            if (lens_out != p.lens) lens_out[r] = p.lens[r];
        }
        if (tid == 0) st.q_start[p.n_requests] = 0;
        if constexpr (FILL)
            for (int t = tid; t < st.max_tokens; t += TH) write_token(st, t, -1, -1, -1);
        return;
    }

    unsigned long long carry = 0;  // tokens (low word) and pages (high word) of the requests before this pass
    for (int r0 = 0; r0 < p.n_requests; r0 += TH) {
        const int r = r0 + tid, nr = min(TH, p.n_requests - r0);
        const int len = r < p.n_requests ? p.lens[r] : 0, n = r < p.n_requests ? n_new[r] : 0;
        int more = pages_of(len + n, p.page_shift) - pages_of(len, p.page_shift), kept = -1;
        if (more) kept = kept_at(r, pages_of(len, p.page_shift));
        if (kept >= 0) {
            --more;
            p.table[(size_t)r * p.max_pages + pages_of(len, p.page_shift)] = kept;
        }
        unsigned long long sum;
        const unsigned long long at = carry + wg_scan((unsigned long long)n | ((unsigned long long)more << 32),
                                                      s_scan, &sum);
        s_tok[tid] = (int)(uint32_t)at;
        s_pg[tid] = (int)(at >> 32);
        s_len[tid] = len;
        s_kept[tid] = kept;
        if (r < p.n_requests) st.q_start[r] = (int)(uint32_t)at;
        carry += sum;
        if (tid == 0) {
            s_tok[nr] = (int)(uint32_t)carry;
            s_pg[nr] = (int)(carry >> 32);
        }
        __syncthreads();
        if (r < p.n_requests) lens_out[r] = len + n;
        // new pages, one a thread: entry m is page m - s_pg of its request, from the top of the stack down
        for (int m = s_pg[0] + tid; m < s_pg[nr]; m += TH) {
            const int i = owner_of(s_pg, nr, m);
            const int j = pages_of(s_len[i], p.page_shift) + (s_kept[i] >= 0) + m - s_pg[i];
            const int id = p.free_pages[n_free - 1 - m];
            const size_t cell = (size_t)(r0 + i) * p.max_pages + j;
            p.table[cell] = p.owned[cell] = page_ok(id, p.n_pages) ? id : -1;
        }
        if constexpr (FILL) {
            for (int t = s_tok[0] + tid; t < s_tok[nr]; t += TH) {
                const int i = owner_of(s_tok, nr, t), held = pages_of(s_len[i], p.page_shift), kept = s_kept[i];
                const int pos = s_len[i] + t - s_tok[i], j = pos >> p.page_shift;
                const int id = j < held                ? p.table[(size_t)(r0 + i) * p.max_pages + j]
                               : kept >= 0 && j == held ? kept
                                                        : p.free_pages[n_free - 1 - (s_pg[i] + j - held - (kept >= 0))];
                write_token(st, t, page_ok(id, p.n_pages) ? (id << p.page_shift) + (pos & (page - 1)) : -1, pos,
                            r0 + i);
            }
        }
        __syncthreads();
    }
    const int total = (int)(uint32_t)carry;
    if (tid == 0) st.q_start[p.n_requests] = total;
    if constexpr (FILL)
        for (int t = total + tid; t < st.max_tokens; t += TH) write_token(st, t, -1, -1, -1);
}

// Numbers the tokens of a planned step from q_start, the new lengths and the table: a thread a token, found by bisection of
// q_start in LDS; 12 bytes written a token (1 million in 7.5 us: 1.6 TB/s).
constexpr int kFillThreads = 256;
__global__ __launch_bounds__(kFillThreads) void paged_fill_kernel(PagedDev p, StepDev st,
                                                                  const int32_t *__restrict__ lens) {
    __shared__ int s_start[kPagedThreads + 1];
    const bool staged = p.n_requests <= kPagedThreads;
    if (staged)
        for (int i = threadIdx.x; i <= p.n_requests; i += kFillThreads) s_start[i] = st.q_start[i];
    __syncthreads();
    const int t = blockIdx.x * kFillThreads + threadIdx.x;
    if (t >= st.max_tokens) return;
    if (t >= (staged ? s_start[p.n_requests] : st.q_start[p.n_requests])) return write_token(st, t, -1, -1, -1);
    const int r = staged ? owner_of(s_start, p.n_requests, t) : owner_of(st.q_start, p.n_requests, t);
    const int end = staged ? s_start[r + 1] : st.q_start[r + 1];
    const int pos = lens[r] - (end - t);
    const int id = p.table[(size_t)r * p.max_pages + (pos >> p.page_shift)];
    write_token(st, t, page_ok(id, p.n_pages) ? (id << p.page_shift) + (pos & ((1 << p.page_shift) - 1)) : -1, pos, r);
}

__global__ __launch_bounds__(256) void paged_reset_kernel(PagedDev p) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, cells = (size_t)p.n_requests * p.max_pages;
    if (i < cells) p.table[i] = p.owned[i] = -1;
    if (i < (size_t)p.n_requests) p.lens[i] = 0;
    if (i < (size_t)p.n_pages) p.free_pages[i] = p.n_pages - 1 - (int)i;
    if (i == 0) *p.n_free = p.n_pages;
}

// One workgroup. Each wave counts the owned pages of its requests, a prefix sum places them, and the wave
// writes them in order of their places. Every cell of both tables goes through the one CU, a request a wave at a time: 128
// requests with 128 columns 17 us. Requests end rarely; a launch over many CUs would need a second one for the places.
__global__ __launch_bounds__(kPagedThreads) void paged_release_kernel(PagedDev p, const int32_t *__restrict__ ended) {
    __shared__ unsigned long long s_scan[17];
    __shared__ int s_cnt[kPagedThreads], s_held[kPagedThreads];  // pages that an ended request owns; that it uses (-1: goes on)
    const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
    long height = min(max(*p.n_free, 0), p.n_pages);
    auto pages_held = [&](int r) { return min(pages_of(max(p.lens[r], 0), p.page_shift), p.max_pages); };
    // the page that request r owns at place j < max_pages, of `held` in use (one array for both: none is marked)
    auto own = [&](int r, int j, int held) {
        const int v = p.owned[(size_t)r * p.max_pages + j];
        return p.owned == p.table && v < 0 ? -1 : owned_page(v, j < held);
    };
    for (int r0 = 0; r0 < p.n_requests; r0 += kPagedThreads) {
        const int nr = min(kPagedThreads, p.n_requests - r0);
        for (int i = w; i < nr; i += kPagedThreads / 64) {
            int n = 0;
            const int held = pages_held(r0 + i);  // (its load goes out beside that of the flag)
            const bool ends = ended[r0 + i] != 0;
            if (ends)
                for (int j = l; j < p.max_pages; j += 64) n += page_ok(own(r0 + i, j, held), p.n_pages);
            n = wave_sum64_dpp(n);
            if (l == 0) s_cnt[i] = n, s_held[i] = ends ? held : -1;
        }
        __syncthreads();
        const int mine = tid < nr ? s_cnt[tid] : 0;
        unsigned long long sum;
        const int before = (int)wg_scan((unsigned long long)mine, s_scan, &sum);
        __syncthreads();
        if (tid < nr) s_cnt[tid] = before;
        __syncthreads();
        for (int i = w; i < nr; i += kPagedThreads / 64) {
            const int held = s_held[i];
            if (held < 0) continue;
            long at = height + s_cnt[i];
            for (int j0 = 0; j0 < p.max_pages; j0 += 64) {
                const int j = j0 + l;
                const size_t cell = (size_t)(r0 + i) * p.max_pages + j;
                const int id = j < p.max_pages ? own(r0 + i, j, held) : -1;
                const unsigned long long has = __ballot(page_ok(id, p.n_pages));
                const long to = at + __popcll(has & ((1ull << l) - 1));
                if (page_ok(id, p.n_pages) && to < p.n_pages) p.free_pages[to] = id;
                if (j < p.max_pages) p.owned[cell] = p.table[cell] = -1;
                at += __popcll(has);
            }
            if (l == 0) p.lens[r0 + i] = 0;
        }
        height += (long)sum;
        __syncthreads();
    }
    if (tid == 0) *p.n_free = (int)min(height, (long)p.n_pages);
}

// The row that row r of a group goes on from.
__device__ __forceinline__ int parent_row(const int32_t *parent, int row, int width) {
    const int b = row % width, q = parent[row];
    return (unsigned)q < (unsigned)width ? row - b + q : row;
}

// First half of the reordering, in one workgroup: takes a page for each row that has none to go on
// filling, and writes the new lengths. Passes hold whole groups, so that in place a group's lengths are
// all read before one of them is written.
// TABLE: it also writes the tables, of few cells (one launch instead of two).
// Latency again: parents, lengths, the page's owner, the stack, the table, each a round of loads that waits for the one before.
// Rows that take a page are counted by ballots, their sums over the waves with one barrier. One group of 4 rows 3.7 us (256
// threads; 5.9 with 1024, shuffles and a barrier a sum), 16 groups of 8 rows and 33 columns 5.8.
template <int MW>
__device__ __forceinline__ void reorder_column(const PagedDev &p, const int32_t *parent, int width, bool ok,
                                               const int32_t *lens, int32_t *table_out, int g, int j);
template <bool TABLE, int MW, int TH>
__global__ __launch_bounds__(TH) void paged_reorder_plan_kernel(PagedDev p, const int32_t *parent, int width, int32_t *status,
                                                                int32_t *lens_out, int32_t *table_out) {
    __shared__ int s_takes[2][TH / 64], s_flags[TH / 64];  // of a wave (passes in turn)
    const int tid = threadIdx.x, l = tid & 63, w = tid >> 6, mask = (1 << p.page_shift) - 1;
    const long cap = (long)p.max_pages << p.page_shift;
    const int n_free = *p.n_free, per = TH / width * width;
    // whether a row takes a page; flags get what is wrong with its parent
    enum { kBadLength = 1, kNotOwned = 2, kShorter = 4 };
    struct Row {
        int len, old, mine;  // its new length, the one that it had, and what `owned` has for it at the open page's place
    };
    auto look = [&](int row, Row *x, int *flags) -> bool {
        const int from = parent_row(parent, row, width), len = p.lens[from], old = p.lens[row];
        *x = Row{len, old, -1};
        if (len < 0 || len > cap || old < 0 || old > cap) {
            *flags |= kBadLength;
            return false;
        }
        // (a row's full pages may be read by others: it must not come back to fill one of them again)
        const int j = len >> p.page_shift;
        if (j < old >> p.page_shift) *flags |= kShorter;
        if ((len & mask) == 0) return false;
        const int own = owned_page(p.owned[(size_t)from * p.max_pages + j], true);
        if (!page_ok(own, p.n_pages) || own != p.table[(size_t)from * p.max_pages + j]) *flags |= kNotOwned;
        x->mine = p.owned[(size_t)row * p.max_pages + j];
        return !page_ok(owned_page(x->mine, j < pages_of(old, p.page_shift)), p.n_pages);
    };
    const bool one = p.n_requests <= per;  // (one pass: what it finds is kept)
    Row x{};
    int flags = 0, need = 0;
    unsigned long long takers = 0;
    for (int r0 = 0; r0 < p.n_requests; r0 += per) {
        const int row = r0 + tid;
        takers = __ballot(tid < per && row < p.n_requests && look(row, &x, &flags));
        need += __builtin_popcountll(takers);
    }
    const int met = (__ballot(flags & kBadLength) ? kBadLength : 0) | (__ballot(flags & kNotOwned) ? kNotOwned : 0) |
                    (__ballot(flags & kShorter) ? kShorter : 0);
    if (l == 0) s_takes[0][w] = need, s_flags[w] = met;
    __syncthreads();  // (every thread has read n_free and, where one pass is all, the lengths)
    // pages that the waves before this one take, and all
    auto waves = [&](int pass, int *all) {
        int before = 0;
        *all = 0;
#pragma unroll
        for (int i = 0; i < TH / 64; ++i) {
            const int n = s_takes[pass & 1][i];
            before += i < w ? n : 0;
            *all += n;
        }
        return before;
    };
    int before = waves(0, &need), wrong = 0;
#pragma unroll
    for (int i = 0; i < TH / 64; ++i) wrong |= s_flags[i];
    const int st = (wrong & kBadLength) || n_free < 0 || n_free > p.n_pages ? JK_PAGED_BAD_LENGTH
                   : (wrong & kNotOwned)                                    ? JK_PAGED_NOT_OWNED
                   : (wrong & kShorter)                                     ? JK_PAGED_SHORTER
                   : need > n_free                                          ? JK_PAGED_NO_PAGES
                                                                            : JK_PAGED_OK;
    if (tid == 0) {
        *status = st;
        if (st == JK_PAGED_OK) *p.n_free = n_free - need;
    }
    if (st != JK_PAGED_OK) {
        if (lens_out != p.lens)
            for (int row = tid; row < p.n_requests; row += TH) lens_out[row] = p.lens[row];
        if (TABLE && table_out != p.table)
            for (int i = tid; i < p.n_requests * p.max_pages; i += TH) table_out[i] = p.table[i];
        return;
    }
    int taken = 0, pass = 1;
    for (int r0 = 0; r0 < p.n_requests; r0 += per, ++pass) {
        const int row = r0 + tid;
        const bool live = tid < per && row < p.n_requests;
        int sum = 0;
        if (!one) {
            takers = __ballot(live && look(row, &x, &flags));
            if (l == 0) s_takes[pass & 1][w] = __builtin_popcountll(takers);
            __syncthreads();  // (all have read the pass's lengths, and left the counts of the pass before the last)
            before = waves(pass, &sum);
        }
        if (live) {
            const int held = pages_of(x.len, p.page_shift);
            int32_t *cells = p.owned + (size_t)row * p.max_pages;
            if (takers >> l & 1) {
                const int at = taken + before + __builtin_popcountll(takers & ((1ull << l) - 1));
                const int id = p.free_pages[n_free - 1 - at];
                cells[held - 1] = page_ok(id, p.n_pages) ? id : -1;
            } else if (x.mine <= -2) {  // come back to the page that it went back from
                cells[held - 1] = owned_page(x.mine, true);
            }
            const int had = pages_of(x.old, p.page_shift);
            if (held < had && cells[held] >= 0) cells[held] = -2 - cells[held];  // goes back from it
            // (what a dropped step left in the places that the row now reaches; steps leave it without a gap)
            for (int j = had; j < x.len >> p.page_shift && cells[j] != -1; ++j)
                if (cells[j] >= 0) cells[j] = -1;
            lens_out[row] = x.len;
        }
        taken += sum;
    }
    if constexpr (TABLE) {
        __syncthreads();
        const int groups = p.n_requests / width;
        for (int i = tid; i < groups * p.max_pages; i += TH)
            reorder_column<MW>(p, parent, width, true, lens_out, table_out, i / p.max_pages, i % p.max_pages);
    }
}

// Second half: one thread takes one column of a group's rows, reads all of them and then writes them, so the
// permutation can be in place. lens: the new lengths. (16 groups of 8 rows, 128 columns: 4.6 us)
template <int MW>
__device__ __forceinline__ void reorder_column(const PagedDev &p, const int32_t *parent, int width, bool ok,
                                               const int32_t *lens, int32_t *table_out, int g, int j) {
    const int row0 = g * width, mask = (1 << p.page_shift) - 1;
    int v[MW];
#pragma unroll
    for (int b = 0; b < MW; ++b) {
        if (b >= width) break;
        const int row = row0 + b, len = lens[row], full = len >> p.page_shift;
        if (!ok) v[b] = p.table[(size_t)row * p.max_pages + j];
        else if (j < full) v[b] = p.table[(size_t)parent_row(parent, row, width) * p.max_pages + j];
        else v[b] = j == full && (len & mask) ? p.owned[(size_t)row * p.max_pages + j] : -1;
    }
#pragma unroll
    for (int b = 0; b < MW; ++b) {
        if (b >= width) break;
        table_out[(size_t)(row0 + b) * p.max_pages + j] = v[b];
    }
}
template <int MW>
__global__ __launch_bounds__(256) void paged_reorder_table_kernel(PagedDev p, const int32_t *__restrict__ parent,
                                                                  int width, const int32_t *__restrict__ status,
                                                                  const int32_t *lens, int32_t *table_out,
                                                                  int col_blocks) {
    const int j = (blockIdx.x % col_blocks) * 256 + threadIdx.x;
    const bool ok = *status == JK_PAGED_OK;
    if (j >= p.max_pages || (!ok && table_out == p.table)) return;
    reorder_column<MW>(p, parent, width, ok, lens, table_out, blockIdx.x / col_blocks, j);
}

// Moves the pages that are being filled: one thread takes 16 bytes of one head's rows of every
// hypothesis of a group, reads all of them and then writes them (a page can be read by one row and
// overwritten by another's in the same step). Read and written once: 128 rows' begun pages, 8 heads of 64 x 128 and keys and
// values, 34 MB in 11 us (3.1 TB/s).
template <int MW>
__global__ __launch_bounds__(256) void kv_reorder_kernel(PagedDev p, jk_kv_q8 c, const int32_t *__restrict__ parent,
                                                         int width, const int32_t *__restrict__ status, int blocks) {
    if (*status != JK_PAGED_OK) return;
    const int cell = blockIdx.x / blocks, i = (blockIdx.x % blocks) * 256 + threadIdx.x;
    const int heads = (int)c.n_kv, which = cell % 2, h = cell / 2 % heads, row0 = cell / 2 / heads * width;
    int8_t *codes = which ? c.v : c.k;
    float *scales = which ? c.v_scale : c.k_scale;
    const int mask = (1 << p.page_shift) - 1, hd = (int)c.head_dim;
    const long cap = (long)p.max_pages << p.page_shift;
    u32x4 v[MW];
    float sc[MW];
    bool moves[MW];
    size_t to[MW];
#pragma unroll
    for (int b = 0; b < MW; ++b) {
        moves[b] = false;
        if (b >= width) continue;
        const int row = row0 + b, from = parent_row(parent, row, width), len = p.lens[row];
        if (from == row || len <= 0 || len > cap || (len & mask) == 0) continue;
        const int j = len >> p.page_shift;
        const int src = owned_page(p.owned[(size_t)from * p.max_pages + j], true);
        const int dst = p.owned[(size_t)row * p.max_pages + j];
        if (!page_ok(src, p.n_pages) || !page_ok(dst, p.n_pages) || i * 16 >= (len & mask) * hd) continue;
        moves[b] = true;
        const size_t from_head = (size_t)src * heads + h;
        to[b] = (size_t)dst * heads + h;
        v[b] = *reinterpret_cast<const u32x4 *>(codes + (from_head << p.page_shift) * hd + (size_t)i * 16);
        sc[b] = i == 0 ? scales[from_head] : 0.0f;  // (a head's scales are one thread's to read and write)
    }
#pragma unroll
    for (int b = 0; b < MW; ++b) {
        if (!moves[b]) continue;
        *reinterpret_cast<u32x4 *>(codes + (to[b] << p.page_shift) * hd + (size_t)i * 16) = v[b];
        if (i == 0) scales[to[b]] = sc[b];
    }
}

constexpr size_t kMaxBlocks = ((size_t)1 << 24) - 1;  // of 256 threads in one launch

static int log2_of(size_t v) {
    int s = 0;
    while (((size_t)1 << s) < v) ++s;
    return s;
}

static jk_status paged_check(const char *what, const jk_paged *p, PagedDev *out) {
    if (!p) return fail(JK_TENSOR_BOUNDS, "%s: null jk_paged", what);
    if (!p->lens || !p->table || !p->owned || !p->free_pages || !p->n_free)
        return fail(JK_TENSOR_BOUNDS, "%s: null array in jk_paged", what);
    if (p->page < 16 || p->page > 256 || (p->page & (p->page - 1)))
        return fail(JK_TENSOR_BOUNDS, "%s: %zu tokens a page: 16, 32, 64, 128 or 256", what, p->page);
    if (p->n_requests == 0 || p->max_pages == 0 || p->n_pages == 0)
        return fail(JK_TENSOR_BOUNDS, "%s: no requests, columns or pages", what);
    if (p->n_requests > (size_t)INT32_MAX / 64 || p->max_pages > (size_t)INT32_MAX / p->page ||
        p->n_pages > (size_t)INT32_MAX / p->page)
        return fail(JK_TENSOR_BOUNDS, "%s: %zu requests, %zu columns or %zu pages of %zu tokens exceed the int32 range",
                    what, p->n_requests, p->max_pages, p->n_pages, p->page);
    *out = PagedDev{(int)p->n_requests, (int)p->max_pages, (int)p->n_pages, log2_of(p->page),
                    p->lens,            p->table,          p->owned,        p->free_pages,
                    p->n_free};
    return JK_OK;
}

static jk_status width_check(const char *what, const jk_paged *p, size_t width) {
    if (width == 0 || width > 32 || p->n_requests % width)
        return fail(JK_TENSOR_BOUNDS, "%s: width %zu: 1..32, and %zu requests a multiple of it", what, width,
                    p->n_requests);
    if (p->owned == p->table)
        return fail(JK_TENSOR_BOUNDS, "%s: owned and table are the same array: rows that share pages need both", what);
    return JK_OK;
}

}  // namespace jk

using namespace jk;

extern "C" {

jk_status jk_paged_reset(jk_stream s, const jk_paged *p) {
    PagedDev d;
    JK_TRY(paged_check("paged_reset", p, &d));
    const size_t cells = std::max({p->n_requests * p->max_pages, p->n_requests, p->n_pages});
    if (cells > (size_t)INT32_MAX)
        return fail(JK_TENSOR_BOUNDS, "paged_reset: a table of %zu x %zu is too large", p->n_requests, p->max_pages);
    hipLaunchKernelGGL(paged_reset_kernel, dim3((unsigned)((cells + 255) / 256)), dim3(256), 0, (hipStream_t)s, d);
    return check_launch("paged_reset_kernel");
}

jk_status jk_paged_extend(jk_stream s, const jk_paged *p, const int32_t *n_new, const jk_paged_step *st,
                          int32_t *lens_out, int32_t *n_free_out) {
    PagedDev d;
    JK_TRY(paged_check("paged_extend", p, &d));
    if (!n_new || !st || !st->q_start || !st->status)
        return fail(JK_TENSOR_BOUNDS, "paged_extend: null counts, step, q_start or status");
    if (st->max_tokens && (!st->slots || !st->positions || !st->requests))
        return fail(JK_TENSOR_BOUNDS, "paged_extend: null slots, positions or requests");
    if (st->max_tokens > (size_t)INT32_MAX - 1024)
        return fail(JK_TENSOR_BOUNDS, "paged_extend: %zu tokens exceed the int32 range", st->max_tokens);
    const StepDev sd{(int)st->max_tokens, st->q_start, st->slots, st->positions, st->requests, st->status};
    int32_t *lo = lens_out ? lens_out : p->lens, *fo = n_free_out ? n_free_out : p->n_free;
    // One workgroup numbers up to this many tokens itself: a second launch costs more until there are some ten a thread (16
    // requests of 500 new tokens 10.8 us, 12.2 in two launches; 100 of 128 13.1 and 12.0).
    if (st->max_tokens <= 8 * kPagedThreads) {
        if (p->n_requests <= 256 && st->max_tokens <= 512)  // (few waves to a barrier: a step of 4 tokens 4.4 us on the GPU, 6.8 with 1024 threads)
            hipLaunchKernelGGL((paged_extend_kernel<true, 256>), dim3(1), dim3(256), 0, (hipStream_t)s, d, n_new, sd, lo,
                               fo);
        else
            hipLaunchKernelGGL((paged_extend_kernel<true, kPagedThreads>), dim3(1), dim3(kPagedThreads), 0,
                               (hipStream_t)s, d, n_new, sd, lo, fo);
        return check_launch("paged_extend_kernel");
    }
    hipLaunchKernelGGL((paged_extend_kernel<false, kPagedThreads>), dim3(1), dim3(kPagedThreads), 0, (hipStream_t)s, d,
                       n_new, sd, lo, fo);
    JK_TRY(check_launch("paged_extend_kernel"));
    hipLaunchKernelGGL(paged_fill_kernel, dim3((unsigned)((st->max_tokens + kFillThreads - 1) / kFillThreads)),
                       dim3(kFillThreads), 0, (hipStream_t)s, d, sd, lo);
    return check_launch("paged_fill_kernel");
}

jk_status jk_paged_release(jk_stream s, const jk_paged *p, const int32_t *ended) {
    PagedDev d;
    JK_TRY(paged_check("paged_release", p, &d));
    if (!ended) return fail(JK_TENSOR_BOUNDS, "paged_release: null flags");
    hipLaunchKernelGGL(paged_release_kernel, dim3(1), dim3(kPagedThreads), 0, (hipStream_t)s, d, ended);
    return check_launch("paged_release_kernel");
}

jk_status jk_paged_reorder(jk_stream s, const jk_paged *p, const int32_t *parent, size_t width, int32_t *status,
                           int32_t *lens_out, int32_t *table_out) {
    PagedDev d;
    JK_TRY(paged_check("paged_reorder", p, &d));
    JK_TRY(width_check("paged_reorder", p, width));
    if (!parent || !status) return fail(JK_TENSOR_BOUNDS, "paged_reorder: null parents or status");
    if (!lens_out != !table_out)
        return fail(JK_TENSOR_BOUNDS, "paged_reorder: lens_out and table_out are given both or neither");
    if (table_out == p->owned) return fail(JK_TENSOR_BOUNDS, "paged_reorder: table_out is owned");
    int32_t *lo = lens_out ? lens_out : p->lens, *to = table_out ? table_out : p->table;
    const size_t col_blocks = (p->max_pages + 255) / 256, groups = p->n_requests / width;
    if (col_blocks * groups > kMaxBlocks)
        return fail(JK_TENSOR_BOUNDS, "paged_reorder: a table of %zu x %zu is too large", p->n_requests, p->max_pages);
    const int w = (int)width;
    // (one cell a thread: 16 groups of 4 rows, 63 columns 20.6 us with the selection before it, 22.2 in two launches; of 8 rows, 126
    // columns 27.6 and 24.1)
    const size_t cells = groups * p->max_pages;
    const hipStream_t hs = (hipStream_t)s;
    if (cells <= (size_t)kPagedThreads) {
        const bool few = cells <= 256 && p->n_requests <= 256 / width * width;
        if (width <= 8 && few)
            hipLaunchKernelGGL((paged_reorder_plan_kernel<true, 8, 256>), dim3(1), dim3(256), 0, hs, d, parent, w, status, lo, to);
        else if (width <= 8)
            hipLaunchKernelGGL((paged_reorder_plan_kernel<true, 8, kPagedThreads>), dim3(1), dim3(kPagedThreads), 0, hs, d, parent,
                               w, status, lo, to);
        else
            hipLaunchKernelGGL((paged_reorder_plan_kernel<true, 32, kPagedThreads>), dim3(1), dim3(kPagedThreads), 0, hs, d,
                               parent, w, status, lo, to);
        return check_launch("paged_reorder_plan_kernel");
    }
    hipLaunchKernelGGL((paged_reorder_plan_kernel<false, 8, kPagedThreads>), dim3(1), dim3(kPagedThreads), 0, hs, d, parent, w,
                       status, lo, to);
    JK_TRY(check_launch("paged_reorder_plan_kernel"));
    const dim3 grid((unsigned)(col_blocks * groups));
    if (width <= 8)
        hipLaunchKernelGGL(paged_reorder_table_kernel<8>, grid, dim3(256), 0, (hipStream_t)s, d, parent, w, status, lo,
                           to, (int)col_blocks);
    else
        hipLaunchKernelGGL(paged_reorder_table_kernel<32>, grid, dim3(256), 0, (hipStream_t)s, d, parent, w, status, lo,
                           to, (int)col_blocks);
    return check_launch("paged_reorder_table_kernel");
}

jk_status jk_kv_reorder_q8(jk_stream s, const jk_kv_q8 *c, const jk_paged *p, const int32_t *parent, size_t width,
                           const int32_t *status) {
    PagedDev d;
    JK_TRY(kv_check("kv_reorder_q8", c));
    JK_TRY(paged_check("kv_reorder_q8", p, &d));
    JK_TRY(width_check("kv_reorder_q8", p, width));
    if (c->page != p->page || c->n_pages != p->n_pages)
        return fail(JK_TENSOR_BOUNDS, "kv_reorder_q8: a cache of %zu pages of %zu tokens for tables of %zu of %zu",
                    c->n_pages, c->page, p->n_pages, p->page);
    if (!parent || !status) return fail(JK_TENSOR_BOUNDS, "kv_reorder_q8: null parents or status");
    const size_t blocks = (c->page * c->head_dim / 16 + 255) / 256, cells = p->n_requests / width * c->n_kv * 2;
    if (cells * blocks > kMaxBlocks)
        return fail(JK_TENSOR_BOUNDS, "kv_reorder_q8: %zu requests of %zu heads are too many", p->n_requests, c->n_kv);
    const dim3 grid((unsigned)(cells * blocks));
    if (width <= 8)
        hipLaunchKernelGGL(kv_reorder_kernel<8>, grid, dim3(256), 0, (hipStream_t)s, d, *c, parent, (int)width, status,
                           (int)blocks);
    else
        hipLaunchKernelGGL(kv_reorder_kernel<32>, grid, dim3(256), 0, (hipStream_t)s, d, *c, parent, (int)width, status,
                           (int)blocks);
    return check_launch("kv_reorder_kernel");
}

}  // extern "C"
