// draft.cu — a step of drafted tokens around its attention: its plan (pages,
// slots, positions, tree masks) and the check of what was drafted.
//
// Both are integer work on a few kilobytes, bound by latency: what counts is the
// number of launches and of loads that wait for one another.
#include "attn.cuh"

namespace warp {

// The last request that starts at or before token t.
__device__ __forceinline__ int request_of(const int32_t *q_start, int batch, int t) {
    int lo = 0, hi = batch;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (q_start[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

// ------------------------------------------------------------------ plan --

struct PlanArgs {
    const int32_t *q_start, *kv_len, *parents;
    int32_t *pages, *held, *pool, *positions;
    int64_t *slots;
    uint64_t *seen;
    int64_t pages_row;
    unsigned *err;
    int batch, tokens, wide, page_shift, base, pool_n, max_q, words;
};

constexpr int kPlanThreads = 1024;

// Exclusive prefix sums over the block, two counts in one word, and their total.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t &total) {
    __shared__ uint64_t of_warp[kPlanThreads / 32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    uint64_t x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t y = __shfl_up_sync(~0u, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();                        // the last scan's words are read
    if (lane == 31) of_warp[warp] = x;
    __syncthreads();
    uint64_t w = of_warp[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t y = __shfl_up_sync(~0u, w, d);
        if (lane >= d) w += y;
    }
    total = __shfl_sync(~0u, w, 31);
    return x - v + (warp ? __shfl_sync(~0u, w, warp - 1) : 0);
}

// Pages of request b that are surplus (high word) and missing (low word).
__device__ __forceinline__ uint64_t plan_need(const PlanArgs &a, int b, int &need, int &had) {
    need = had = 0;
    if (b >= a.batch) return 0;
    const int len = a.kv_len[b], h = a.held[b];
    const int64_t n = ((int64_t)max(len, 0) + (1 << a.page_shift) - 1) >> a.page_shift;
    need = (int)min(n, (int64_t)a.wide);
    had = min(max(h, 0), a.wide);
    if (len < 0 || n > a.wide || had != h) atomicOr(a.err, kAttnBadLen);
    return (uint64_t)max(had - need, 0) << 32 | (uint32_t)max(need - had, 0);
}

// Which of the block's requests has item k of `first`'s running count.
__device__ __forceinline__ int item_of(const int *first, int k) {
    int lo = 0, hi = kPlanThreads;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (first[mid] <= k) lo = mid; else hi = mid;
    }
    return lo;
}

// The pages' part, by one block: surplus to the pool, then missing from it.  The
// pool is a stack of which pages come off from the first request's first on, so
// they are put there from the last request's last on.
__device__ __forceinline__ void plan_pages(const PlanArgs &a) {
    __shared__ int first[kPlanThreads], entry[kPlanThreads];
    const int tid = threadIdx.x;
    const bool one = a.batch <= kPlanThreads;           // all requests in one scan
    int need, had;
    uint64_t all = 0;
    if (!one) {
        uint64_t mine = 0;
        for (int b = tid; b < a.batch; b += kPlanThreads) mine += plan_need(a, b, need, had);
        block_scan(mine, all);
    }
    const int said = a.pool[0], count = min(max(said, 0), a.pool_n);
    if (said != count && tid == 0) atomicOr(a.err, kAttnBadPage);
    uint64_t before = 0, v = 0, ex = 0;
    int top = count;
    for (int b0 = 0; b0 < a.batch; b0 += kPlanThreads) {
        uint64_t total;
        v = plan_need(a, b0 + tid, need, had);
        ex = block_scan(v, total);
        if (one) all = total;
        const int64_t back = (int64_t)count + (int64_t)(all >> 32);
        top = (int)min(back, (int64_t)a.pool_n);
        if (total >> 32) {
            first[tid] = (int)(ex >> 32);
            entry[tid] = need;
            __syncthreads();
            for (int k = tid; k < (int)(total >> 32); k += kPlanThreads) {
                const int r = item_of(first, k);
                int32_t *const at = a.pages + (b0 + r) * a.pages_row + entry[r] + (k - first[r]);
                const int64_t place = back - 1 - (int64_t)(before >> 32) - k;
                const int page = *at;
                if (place < a.pool_n) a.pool[1 + place] = page;
                // a page given back twice, or one that is not of this pool
                if (place >= a.pool_n || (unsigned)page >= (unsigned)a.pool_n)
                    atomicOr(a.err, kAttnBadPage);
                *at = -1;
            }
            __syncthreads();
        }
        before += total;
    }
    __syncthreads();
    before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kPlanThreads) {
        uint64_t total = all;
        if (!one) {
            v = plan_need(a, b0 + tid, need, had);
            ex = block_scan(v, total);
        }
        const uint32_t lack = (uint32_t)total;
        if (lack) {
            first[tid] = (int)(uint32_t)ex;
            entry[tid] = had;
            __syncthreads();
            for (int k = tid; k < (int)lack; k += kPlanThreads) {
                const int64_t place = (int64_t)top - 1 - (uint32_t)before - k;
                // what was in the entry may be a page that another request has
                int32_t page = -1;
                if (place < 0) atomicOr(a.err, kAttnNoPage);
                else page = a.pool[1 + place];
                const int r = item_of(first, k);
                a.pages[(b0 + r) * a.pages_row + entry[r] + (k - first[r])] = page;
            }
        }
        if (b0 + tid < a.batch) {
            const int64_t left = (int64_t)top - (uint32_t)before - (uint32_t)ex;
            a.held[b0 + tid] = min(need, had) + (int)min((int64_t)(uint32_t)v, max(left, (int64_t)0));
        }
        before += total;
        __syncthreads();
    }
    if (tid == 0) a.pool[0] = (int)max((int64_t)top - (uint32_t)all, (int64_t)0);
}

// Node `cur` of the tokens from `first` on: its row of masks, from itself up to
// the root, and its depth.
__device__ __forceinline__ int plan_tree(const PlanArgs &a, int first, int cur, uint64_t *row) {
    int w = a.words - 1, depth = -1;
    uint64_t bits = 0;
    while (cur >= 0) {
        for (; w > cur >> 6; w--) {
            row[w] = bits;
            bits = 0;
        }
        bits |= 1ull << (cur & 63);
        depth++;
        const int up = a.parents[first + cur];
        if (up >= cur) atomicOr(a.err, kAttnBadTree);
        cur = up >= cur ? -1 : up;
    }
    for (; w >= 0; w--) {
        row[w] = bits;
        bits = 0;
    }
    return depth;
}

// What plan_tokens needs of token t before the pages are known.
struct PlanToken { int b; int64_t j; };

__device__ __forceinline__ PlanToken plan_find(const PlanArgs &a, int t) {
    const int b = request_of(a.q_start, a.batch, t);
    const int first = a.q_start[b], end = a.q_start[b + 1];
    uint64_t *const row = a.seen + (int64_t)t * a.words;
    int64_t j = -1, pos = 0;
    if (first < 0) atomicOr(a.err, kAttnBadLen);        // its parents would lie before the array
    if (first >= 0 && t >= first && t < end) {
        const int64_t base = (int64_t)a.kv_len[b] - end;
        j = base + t;
        pos = a.base + j;
        if (a.parents) {
            const int i = t - first;
            if (i < a.max_q) {
                pos = a.base + base + first + plan_tree(a, first, i, row);
            } else {
                atomicOr(a.err, kAttnBadLen);
                for (int w = 0; w < a.words; w++) row[w] = 0;
            }
        }
    } else if (a.parents) {
        for (int w = 0; w < a.words; w++) row[w] = 0;
    }
    a.positions[t] = (int32_t)pos;
    return {b, j};
}

__device__ __forceinline__ void plan_slot(const PlanArgs &a, int t, PlanToken p) {
    int64_t slot = -1;
    if (p.j >= 0) {
        if ((p.j >> a.page_shift) >= a.wide) {
            atomicOr(a.err, kAttnBadLen);
        } else {
            const int page = a.pages[p.b * a.pages_row + (p.j >> a.page_shift)];
            // a negative slot would pass for a token that is not to be stored
            if (page < 0) atomicOr(a.err, kAttnBadPage);
            else slot = ((int64_t)page << a.page_shift) + (p.j & ((1 << a.page_shift) - 1));
        }
    }
    a.slots[t] = slot;
}

// Pages, and the tokens where they are few enough for one block: what a second launch saves on
// the device (302 tokens 4.1 us a call against 4.7, 1774 tokens 4.2 against 6.1) is less than the
// 2.5 us that it costs the host as long as the one block's part is a round or less.
__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(const PlanArgs a, bool tokens) {
    pdl_trigger();
    if (a.pool) plan_pages(a);
    if (!tokens) return;
    __syncthreads();
    for (int t = threadIdx.x; t < a.tokens; t += kPlanThreads) plan_slot(a, t, plan_find(a, t));
}

__global__ void __launch_bounds__(256) plan_tokens_kernel(const PlanArgs a) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    PlanToken p = {0, -1};
    if (t < a.tokens) p = plan_find(a, t);
    pdl_wait();
    if (t < a.tokens) plan_slot(a, t, p);
}

// ---------------------------------------------------------------- accept --

constexpr int kAcceptThreads = 256;
constexpr int kAcceptNodes = 4096;          // of a request, at most
constexpr int kKeepCaches = 128;            // a launch
constexpr int kKeepDepth = 4;               // moves of a thread in flight

struct AcceptArgs {
    const int32_t *drafted, *picked, *q_start, *kv_len, *pages;
    const uint64_t *seen;
    int64_t seen_words, pages_row;
    int32_t *count, *path, *chosen, *kv_after;
    unsigned *err;
    int batch, tokens, max_q, wide;
    // the caches of a launch, none to all; the first launch writes the results
    int caches, first;
    void *k[kKeepCaches], *v[kKeepCaches];
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    int page_shift, n_pages, kv_heads, per_head;        // per_head: pieces of a head's row
};

// A node's row, up to itself.
__device__ __forceinline__ uint64_t upto(const uint64_t *row, int w, int i) {
    const uint64_t x = row[w];
    return w < i >> 6 ? x : (x & ((1ull << (i & 63)) - 1)) | 1ull << (i & 63);
}

// The accepted path, and its keys and values behind the certain ones: node path[d]
// to place d.  A block has a request and some of the caches, and finds the path itself: a
// few loads, which a kernel before this one would only put in front of them (48 trees of up
// to 61 nodes in 32 caches: 12.2 us against 13.7; one tree of 16 in two: 4.5 against 5.8).  A thread moves the same piece of
// every key, d ascending: path[d] >= d ascends, so a place is read before it is
// written.
template <typename V>
__global__ void __launch_bounds__(kAcceptThreads)
accept_kernel(const __grid_constant__ AcceptArgs a) {
    __shared__ uint32_t agrees[kAcceptNodes / 32];
    __shared__ int path[kAcceptNodes];
    __shared__ unsigned long long best;
    const int b = blockIdx.x, tid = threadIdx.x;
    const int s = a.q_start[b], e = a.q_start[b + 1], len = a.kv_len[b];
    const int t0 = min(max(s, 0), a.tokens);
    const int n = min(min(max(e - s, 0), a.max_q), a.tokens - t0);
    const bool tells = a.first && blockIdx.y == 0;
    if (tid == 0) {
        best = 0;
        if (tells && (t0 != s || n != e - s || len < n)) atomicOr(a.err, kAttnBadLen);
    }
    __syncthreads();
    const uint64_t *const rows = a.seen + t0 * a.seen_words;
    for (int i0 = 0; i0 < n; i0 += kAcceptThreads) {
        const int i = i0 + tid;
        bool ok = i == 0;
        if (i > 0 && i < n) {
            const uint64_t *const row = rows + i * a.seen_words;
            const int token = a.drafted[t0 + i];
            int parent = -1;
            for (int w = i >> 6; w >= 0 && parent < 0; w--) {
                uint64_t x = row[w];
                if (w == i >> 6) x &= (1ull << (i & 63)) - 1;
                if (x) parent = w * 64 + 63 - __clzll(x);
            }
            ok = parent >= 0 && token >= 0 && token == a.picked[t0 + parent];
        }
        const uint32_t word = __ballot_sync(~0u, ok);
        if (tid % 32 == 0) agrees[i / 32] = word;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kAcceptThreads) {
        const uint64_t *const row = rows + i * a.seen_words;
        bool whole = true;
        int bits = 0;
        for (int w = 0; w <= i >> 6 && whole; w++) {
            const uint64_t x = upto(row, w, i);
            const uint64_t ok = agrees[2 * w] | (uint64_t)agrees[2 * w + 1] << 32;
            whole = !(x & ~ok) && (w > 0 || (x & 1));
            bits += __popcll(x);
        }
        if (whole) atomicMax(&best, (unsigned long long)bits << 32 | (uint32_t)~i);
    }
    __syncthreads();
    const int count = (int)(best >> 32), last = n ? (int)~(uint32_t)best : -1;
    int32_t *const told = a.path + (int64_t)b * a.max_q, *const chosen =
                                                             a.chosen + (int64_t)b * a.max_q;
    for (int i = tid; i < a.max_q; i += kAcceptThreads) {
        if (tells && i >= count) told[i] = chosen[i] = -1;
        if (i > last) continue;
        const uint64_t *const row = rows + last * a.seen_words;
        if (!(upto(row, i >> 6, last) >> (i & 63) & 1)) continue;
        int d = 0;
        for (int w = 0; w < i >> 6; w++) d += __popcll(row[w]);
        d += __popcll(row[i >> 6] & ((1ull << (i & 63)) - 1));
        path[d] = i;
        if (tells) {
            told[d] = i;
            chosen[d] = a.picked[t0 + i];
        }
    }
    if (tells && tid == 0) {
        a.count[b] = count;
        a.kv_after[b] = max(len - n + count, 0);
    }
    if (!a.caches) return;
    __syncthreads();
    const int base = len - n;
    const int32_t *const table = a.pages + b * a.pages_row;
    const int pieces = a.kv_heads * a.per_head;
    auto place = [&](int64_t j) -> int64_t {            // page and slot of key j, or -1
        if (j < 0 || (j >> a.page_shift) >= a.wide) {
            atomicOr(a.err, kAttnBadLen);
            return -1;
        }
        const int page = table[j >> a.page_shift];
        if ((unsigned)page >= (unsigned)a.n_pages) {
            atomicOr(a.err, kAttnBadPage);
            return -1;
        }
        return (int64_t)page << a.page_shift | (j & ((1 << a.page_shift) - 1));
    };
    for (int x = tid; x < 2 * pieces; x += kAcceptThreads) {
        const bool val = x >= pieces;
        const int y = val ? x - pieces : x, head = y / a.per_head;
        const int64_t page = val ? a.v_page : a.k_page, slot = val ? a.v_slot : a.k_slot;
        const int64_t in = 2 * head * (val ? a.v_head : a.k_head) +
                           (int64_t)(y - head * a.per_head) * sizeof(V);
        auto offset = [&](int64_t p) {
            return in + 2 * ((p >> a.page_shift) * page + (p & ((1 << a.page_shift) - 1)) * slot);
        };
        for (int d0 = 0; d0 < count; d0 += kKeepDepth) {
            int64_t from[kKeepDepth], to[kKeepDepth];
#pragma unroll
            for (int i = 0; i < kKeepDepth; i++) {
                const int d = d0 + i, node = d < count ? path[d] : d;
                to[i] = -1;
                if (node == d) continue;
                const int64_t src = place((int64_t)base + node);
                const int64_t dst = src < 0 ? -1 : place((int64_t)base + d);
                if (dst < 0) continue;
                from[i] = offset(src);
                to[i] = offset(dst);
            }
            for (int c = blockIdx.y; c < a.caches; c += gridDim.y) {
                char *const at = (char *)(val ? a.v[c] : a.k[c]);
                V r[kKeepDepth];
#pragma unroll
                for (int i = 0; i < kKeepDepth; i++)
                    if (to[i] >= 0) r[i] = *(const V *)(at + from[i]);
#pragma unroll
                for (int i = 0; i < kKeepDepth; i++)
                    if (to[i] >= 0) *(V *)(at + to[i]) = r[i];
            }
        }
    }
}

// Whether an address occurs twice: a cache whose path moves twice is not in order.
static bool cache_twice(int n, void *const *k, void *const *v) {
    bool twice = false;
    for (int i = 0; i < n; i++) {
        for (int j = 0; j < i; j++) twice |= k[i] == k[j] || v[i] == v[j];
        for (int j = 0; j < n; j++) twice |= k[i] == v[j];
    }
    return twice;
}

}  // namespace warp

using namespace warp;

extern "C" int warp_step_plan(const warp_plan_desc *d, void *stream) {
    const char *who = "warp_step_plan";
    WARP_ARG(d, "%s: NULL description", who);
    WARP_ARG(d->batch >= 0 && d->tokens >= 0 && d->pages_per_row >= 0 && d->pages_row >= 0 &&
                 d->base >= 0 && d->max_q >= 0,
             "%s: negative size", who);
    WARP_ARG(d->page_size >= 16 && d->page_size <= 4096 && !(d->page_size & (d->page_size - 1)),
             "%s: page_size %d is not a power of two in 16..4096", who, d->page_size);
    // held may have no address where there is no request
    WARP_ARG(!d->held == !d->pool || d->batch == 0, "%s: held and pool go together", who);
    WARP_ARG(!d->pool || (d->pool_pages >= 0 && d->pool_pages < ((int64_t)1 << 31) - 1),
             "%s: %lld pages in the pool", who, (long long)d->pool_pages);
    WARP_ARG((int64_t)d->batch * d->pages_per_row < (int64_t)1 << 31,
             "%s: a page table of 2^31 entries and more", who);
    WARP_ARG(!d->pool || d->batch < 2 || d->pages_row >= d->pages_per_row,
             "%s: rows of the page table overlap", who);
    if (d->batch == 0 && d->tokens == 0) return WARP_OK;
    WARP_ARG(d->batch >= 1 && d->kv_len && (d->pages || !d->pages_per_row),
             "%s: NULL pointer or no request", who);
    WARP_ARG(!d->tokens || (d->q_start && d->positions && d->slots), "%s: NULL pointer", who);
    WARP_ARG(!d->parents || !d->tokens || (d->seen && ((uintptr_t)d->seen & 7) == 0),
             "%s: the masks are NULL or not 8-byte aligned", who);
    if (!d->tokens && !d->pool) return WARP_OK;
    PlanArgs a = {};
    a.q_start = d->q_start, a.kv_len = d->kv_len, a.parents = d->parents;
    a.pages = d->pages, a.held = d->held, a.pool = d->pool;
    a.positions = d->positions, a.slots = d->slots, a.seen = d->seen;
    a.pages_row = d->pages_row;
    a.batch = d->batch, a.tokens = d->tokens, a.wide = d->pages_per_row;
    a.page_shift = __builtin_ctz(d->page_size), a.base = d->base;
    a.pool_n = (int)d->pool_pages, a.max_q = d->max_q, a.words = (d->max_q + 63) / 64;
    const int rc = attn_err_word(&a.err);
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    const bool apart = d->tokens > kPlanThreads || !d->pool;
    if (d->pool) {
        plan_pages_kernel<<<1, kPlanThreads, 0, st>>>(a, !apart);
        WARP_CHECK_LAUNCH("plan_pages_kernel");
    }
    if (apart && d->tokens) {
        const cudaError_t e = attn_start(plan_tokens_kernel, dim3(cdiv(d->tokens, 256)), 256, 0, st,
                                         !d->pool, a);
        if (e != cudaSuccess) return cuda_fail(e, "plan_tokens_kernel");
        count_launch();
    }
    return WARP_OK;
}

extern "C" int warp_tree_accept(const warp_accept_desc *d, const warp_kv_pages *c, int n_caches,
                                void *const *k, void *const *v, void *stream) {
    const char *who = "warp_tree_accept";
    WARP_ARG(d, "%s: NULL description", who);
    WARP_ARG(d->batch >= 0 && d->tokens >= 0 && d->max_q >= 0 && d->pages_per_row >= 0 &&
                 d->pages_row >= 0 && n_caches >= 0,
             "%s: negative size", who);
    WARP_ARG(d->batch <= (1 << 24), "%s: %d requests", who, d->batch);
    WARP_ARG(d->seen_words >= (d->max_q + 63) / 64 && d->max_q <= kAcceptNodes,
             "%s: %lld words of 64 bits for masks of up to %d nodes (%d at most)", who,
             (long long)d->seen_words, d->max_q, kAcceptNodes);
    if (d->batch == 0) return WARP_OK;
    WARP_ARG(d->q_start && d->kv_len && d->count && d->kv_after, "%s: NULL pointer", who);
    WARP_ARG(!d->max_q || (d->path && d->chosen), "%s: NULL pointer", who);
    WARP_ARG(!d->tokens || (d->drafted && d->picked && d->seen && ((uintptr_t)d->seen & 7) == 0),
             "%s: NULL pointer, or masks that are not 8-byte aligned", who);
    WARP_ARG(d->kv_after != d->kv_len && d->count != d->kv_len,
             "%s: kv_after and count may not be kv_len", who);
    if (n_caches) {
        WARP_ARG(c && k && v && (d->pages || !d->pages_per_row), "%s: NULL pages", who);
        warp_kv_pages one = *c;
        for (int i = 0; i < n_caches; i++) {
            one.k = k[i], one.v = v[i];
            const int rc = kv_pages_check(&one, who);
            if (rc) return rc;
        }
        WARP_ARG(c->head_dim % 2 == 0, "%s: head_dim %d is odd", who, c->head_dim);
        WARP_ARG(!cache_twice(n_caches, k, v), "%s: a cache is there twice", who);
    }
    AcceptArgs a = {};
    a.drafted = d->drafted, a.picked = d->picked, a.q_start = d->q_start, a.kv_len = d->kv_len;
    a.pages = d->pages, a.seen = d->seen, a.seen_words = d->seen_words, a.pages_row = d->pages_row;
    a.count = d->count, a.path = d->path, a.chosen = d->chosen, a.kv_after = d->kv_after;
    a.batch = d->batch, a.tokens = d->tokens, a.max_q = d->max_q, a.wide = d->pages_per_row;
    const int rc = attn_err_word(&a.err);
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    bool wide = true;
    if (n_caches) {
        a.k_page = c->k_page, a.k_slot = c->k_slot, a.k_head = c->k_head;
        a.v_page = c->v_page, a.v_slot = c->v_slot, a.v_head = c->v_head;
        a.page_shift = __builtin_ctz(c->page_size), a.n_pages = (int)c->pages;
        a.kv_heads = c->kv_heads;
        wide = c->head_dim % 8 == 0;
        a.per_head = c->head_dim / (wide ? 8 : 2);
    }
    for (int c0 = 0; c0 == 0 || c0 < n_caches; c0 += kKeepCaches) {
        a.caches = n_caches - c0 < kKeepCaches ? n_caches - c0 : kKeepCaches;
        a.first = c0 == 0;
        for (int i = 0; i < a.caches; i++) a.k[i] = k[c0 + i], a.v[i] = v[c0 + i];
        // as many blocks as fit the card at once
        const int room = 8 * 148 / d->batch, most = a.caches < 1 ? 1 : a.caches;
        const dim3 grid(d->batch, room < 1 ? 1 : room < most ? room : most);
        if (wide) accept_kernel<uint4><<<grid, kAcceptThreads, 0, st>>>(a);
        else accept_kernel<uint32_t><<<grid, kAcceptThreads, 0, st>>>(a);
        WARP_CHECK_LAUNCH("accept_kernel");
    }
    return WARP_OK;
}
