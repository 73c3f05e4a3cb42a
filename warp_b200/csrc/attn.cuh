// attn.cuh — what the attention kernels share: element types, the error word
// behind warp_attn_status, and the checks of a page description.
#pragma once
#include "common.cuh"

#include <atomic>

namespace warp {

// Bits of the error word.
constexpr unsigned kAttnBadSlot = 1u;     // a slot outside the pages
constexpr unsigned kAttnBadPage = 2u;     // a page number outside the pages
constexpr unsigned kAttnBadLen = 4u;      // a length over its host bound
constexpr unsigned kAttnTimeout = 8u;     // a bounded wait gave up
constexpr unsigned kAttnNoPage = 16u;     // the pool of pages is empty
constexpr unsigned kAttnBadTree = 32u;    // a parent that does not come before its node

// Device address of the error word (one per device).
int attn_err_word(unsigned **out);

int kv_pages_check(const warp_kv_pages *c, const char *who);

template <typename T> struct AttnType;
template <> struct AttnType<float> {
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct AttnType<__half> {
    static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};
template <> struct AttnType<__nv_bfloat16> {
    static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};

// x / d for x below 2^31 by the reciprocal that the host gives with d, and a step
// of correction: a quarter of a division's time, and several stand at the start of
// a block one behind another.
struct AttnDiv { uint32_t d, mul; };
inline AttnDiv attn_div(int d) {
    const uint32_t u = d < 1 ? 1 : (uint32_t)d;
    return {u, u == 1 ? 0xffffffffu : (uint32_t)(((uint64_t)1 << 32) / u)};
}
__device__ __forceinline__ int operator/(int x, const AttnDiv &v) {
    const uint32_t q = __umulhi((uint32_t)x, v.mul);
    return (int)(q + ((uint32_t)x - q * v.d >= v.d));
}

// One attention call as its kernels see it.
struct AttnArgs {
    const void *q, *kp, *vp;
    void *out;
    int64_t q_token, q_head;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    const int32_t *q_start, *kv_len, *pages, *prefix_pages;
    int64_t pages_row;
    int pages_per_row, page_shift, n_pages;
    int batch, tokens, q_heads, kv_heads, group;
    int max_q, max_kv, causal, prefix_len;
    float scale_log2;                       // scale * log2(e)
    unsigned *err;
    // Partial results of split key ranges: o [part][token][head][D] not yet
    // divided by l, and (m, l) with m the running maximum in the log2 domain.
    // Parts 0..prefix_parts-1 are the shared prefix's where it is computed for
    // the whole batch at once (`packed`), the requests' own parts follow.
    float *part_o;
    float2 *part_ml;
    int packed, prefix_parts;
    int more;                               // another kernel of the call follows
    // Requests with more rows a kv head than rows_small go to attn_umma_kernel,
    // which counts keys in tiles of attn_wide; the others to attn_rows_kernel.
    int rows_small;
    int split_tiles;                        // key tiles of a request's part
    int prefix_split_tiles;                 // and of a part of the prefix
    int wide_each, wide_parts;              // the same for attn_umma_kernel: wide tiles
    int prefix_wide_each;                   // of a part, and parts at most
    // divisions of attn_umma_kernel: by group, by parts, by tiles of a part
    AttnDiv by_group, by_wide_parts, by_prefix_parts, by_wide_each, by_prefix_each;
    // Trees: the nodes that token t sees, bit m of seen[t * seen_words + m / 64] for node m.
    const uint64_t *seen;
    int64_t seen_words;
    int runs;                               // blocks of attn_umma_kernel, where they take runs
    struct AttnSplit *splits;               // [runs], what they leave to be joined
};

// An item that blocks c0 .. c1 had a part of each (c1 0: none).  `late`: c0's run begins
// before the item, whose part is then in its second place.
struct AttnSplit { int c0, c1, late, t0, rows, kvh; };

// What a kernel's rows and keys are: those of one request (causal or not), all the
// batch's rows and the shared prefix, or those of one request whose queries are the
// nodes of a tree; and the same with the batch's work in equal runs (AttnRuns).
enum AttnKind { kAttnOwn, kAttnPacked, kAttnTree, kAttnTreeRuns };

// Request b as the host's bounds leave it: its first token, its queries and
// its own keys.
struct AttnReq { int t0, n, len; };

__device__ __forceinline__ AttnReq attn_req(const AttnArgs &a, int b, bool report = true) {
    AttnReq r;
    const int s = a.q_start[b], e = a.q_start[b + 1], l = a.kv_len[b];
    r.t0 = min(max(s, 0), a.tokens);
    r.n = min(min(max(e - s, 0), a.max_q), a.tokens - r.t0);
    r.len = (int)min((int64_t)min(max(l, 0), a.max_kv),
                     (int64_t)a.pages_per_row << a.page_shift);
    if (report && threadIdx.x == 0 && (r.t0 != s || r.n != e - s || r.len != l))
        atomicOr(a.err, kAttnBadLen);
    return r;
}

// The page of own or prefix key j; a number outside the pages is reported and
// read as page 0.
__device__ __forceinline__ int attn_page(const AttnArgs &a, const int32_t *table, int j) {
    const int p = table[j >> a.page_shift];
    if ((unsigned)p < (unsigned)a.n_pages) return p;
    atomicOr(a.err, kAttnBadPage);
    return 0;
}

// The keys from node number `from` on that a node sees, one a bit: keys before the
// tree (negative numbers) are seen by all.  `words` is the node's row of the masks.
__device__ __forceinline__ uint64_t tree_sight(const uint64_t *words, int64_t n, int from) {
    if (from <= -64) return ~0ull;
    const int w = max(from, 0) >> 6;
    const uint64_t lo = w < n ? words[w] : 0;
    if (from < 0) return lo << -from | ((1ull << -from) - 1);
    const int s = from & 63;
    if (!s) return lo;
    return lo >> s | (w + 1 < n ? words[w + 1] << (64 - s) : 0);
}
// The first `n` bits.
__device__ __forceinline__ uint64_t low_bits(int n) {
    return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
}

// Keys come in tiles of kAttnTile; the prefix's last tile and a request's last
// one may be partly filled, and a tile never mixes the two.
constexpr int kAttnTile = 16;
// Keys a tile of attn_umma_kernel.
__host__ __device__ constexpr int attn_wide(int) { return 128; }

// The batch's work as one line of units, which the blocks take equal runs of: units are
// key tiles of an item, an item is a request's rows, one row tile at most, on one kv head,
// and items lie request by request.  An item that one block has all of is written by it; the
// parts of others go to the two places that each block has, one for what its run
// begins with and one for what it ends with, and are joined.  A request without rows or
// keys has no units.
constexpr int kAttnRunRows = 128;
struct AttnRuns {
    int all, blocks;
    __device__ __forceinline__ int begin(int block) const {
        return (int)((int64_t)all * block / blocks);
    }
    __device__ __forceinline__ int block_of(int u) const {
        return (int)((((int64_t)u + 1) * blocks - 1) / all);
    }
};
// Units of an item of n tokens and len own keys.
__device__ __forceinline__ int attn_item(int n, int len) {
    return n ? (len + attn_wide(0) - 1) / attn_wide(0) : 0;
}
// Units of request b, 0 past the batch; all are below 2^31 (the host sees to that).
__device__ __forceinline__ int attn_units_of(const AttnArgs &a, int b) {
    if (b >= a.batch) return 0;
    const AttnReq r = attn_req(a, b, false);
    return attn_item(r.n, r.len) * a.kv_heads;
}
// Units of the requests before request b, by all lanes of a warp.
__device__ __forceinline__ int attn_units_before(const AttnArgs &a, int b) {
    int sum = 0;
    for (int i = threadIdx.x % 32; i < b; i += 32) sum += attn_units_of(a, i);
    return __reduce_add_sync(~0u, sum);
}
// No more blocks than units, so that each has one.
__device__ __forceinline__ AttnRuns attn_runs(const AttnArgs &a) {
    const int all = attn_units_before(a, a.batch);
    return {all, min(all, a.runs)};
}
// The request that has unit u, and the units before it.
__device__ __forceinline__ int attn_units_at(const AttnArgs &a, int u, int &b) {
    const int lane = threadIdx.x % 32;
    int before = 0;
    for (b = 0;; b += 32) {
        const int mine = attn_units_of(a, b + lane);
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int x = __shfl_up_sync(~0u, upto, d);
            if (lane >= d) upto += x;
        }
        const unsigned has = __ballot_sync(~0u, before + upto > u);
        if (has || b + 32 >= a.batch) {
            const int k = has ? __ffs(has) - 1 : 0;
            b += k;
            return before + __shfl_sync(~0u, upto - mine, k);
        }
        before += __shfl_sync(~0u, upto, 31);
    }
}

// How many parts a range of `tiles` key tiles is split into, `each` tiles a part.
__device__ __forceinline__ int attn_parts(int tiles, int each) {
    return (tiles + each - 1) / each;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 at a time: half the instructions, though each takes the pipe as long
// as two.
__device__ __forceinline__ uint64_t pair2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 both(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// Not to be added to where its rounding counts: the compiler may fuse the two.
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *(const uint32_t *)&h;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *(const uint32_t *)&h;
}

// The softmax's weights are rounded to the pages' type for the second product, as
// the matrix instructions take both operands in one type; their sum is taken
// before.  bf16 has fp32's exponents.  fp16 rounds what is below 2^-14 ever more
// coarsely and below 2^-25 to nothing, though a long row's many small weights may
// count: so weights are measured from a maximum lowered by 2^lift, up to 2^15 of
// fp16's 2^16, and what is recorded as the maximum is the lowered one.  A weight
// is then rounded relatively down to 2^-(14 + lift) of the row's largest, and the
// error of each below is 2^-(25 + lift) at most.  `slack`: how far a row may
// outgrow its maximum (as a power of two) before that is moved.
template <typename T> __host__ __device__ constexpr float attn_lift(float) { return 0.f; }
template <> __host__ __device__ constexpr float attn_lift<__half>(float slack) {
    return 15.f - slack;
}

// The tensor-core kernel: the requests with many rows, or (kAttnPacked) the shared
// prefix for all rows of the batch.
int attn_umma(const AttnArgs &a, const warp_kv_pages *c, AttnKind kind, bool first,
              cudaStream_t st);

// The wait for the kernel before this one, by one block, the last to start: a
// grid is not complete before it, and the others leave their places at once.
__device__ __forceinline__ void attn_wait_last() {
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1)
        pdl_wait();
}

// Allows `kernel` its dynamic shared memory, once for each device; `done` is the
// kernel's own, a bit a device.
template <typename K>
inline cudaError_t attn_smem(K *kernel, int bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (e != cudaSuccess || (done.load() & bit)) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit);
    return e;
}

// Launches a call's first kernel behind everything before it on the stream, and
// each further one so that it may start early.
template <typename... KArgs, typename... Args>
inline cudaError_t attn_start(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem,
                              cudaStream_t st, bool first, const Args &...args) {
    if (!first) return launch_pdl(kernel, grid, dim3(threads), smem, st, args...);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace warp
