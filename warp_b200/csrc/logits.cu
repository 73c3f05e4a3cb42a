// logits.cu — penalties for repeated tokens, biases and masks on logits, and the
// largest of each row.
//
// One read of the logits (and, where they are kept, one write): bound by memory.
// A cluster of blocks shares the vocabulary of a few rows of one request, so that
// the blocks' choices are joined in the cluster and nothing is left to a second
// launch.  A block counts its part of the context once, in shared memory: a bit
// for each token that occurs, which a thread looks at for a whole vector of logits,
// and the numbers, which are read only where a bit is set.
#include "attn.cuh"

namespace warp {

struct PickArgs {
    const void *logits;
    void *out;
    int32_t *picked;
    const int32_t *q_start, *history, *history_len, *drafted;
    const float *repetition, *frequency, *presence, *bias;
    const uint32_t *allowed;
    const uint64_t *seen;
    int64_t row, out_row, history_row, bias_row, allowed_row, seen_words;
    unsigned *err;
    int tokens, batch, vocab, history_wide;
    int max_q, rows, groups;                // rows a cluster, clusters a request
    int part;                               // tokens of the vocabulary a block and pass
    int passes;
};

constexpr int kPickThreads = 256;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kPickRows = 16;               // rows a cluster, at most
constexpr int kPickPart = 32768;            // tokens a block and pass, at most

// A choice as one number that the larger of two is the better of: larger logit,
// then lower token.  0 is no choice.
__device__ __forceinline__ unsigned long long pick_key(float x, int v) {
    const uint32_t u = __float_as_uint(x + 0.f);        // -0 is 0
    const uint32_t up = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (unsigned long long)up << 32 | (uint32_t)~v;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// A word of block `rank`'s shared memory, at the address that it has in this one's.
__device__ __forceinline__ unsigned long long cluster_ld64(uint32_t addr, uint32_t rank) {
    unsigned long long v;
    asm volatile(
        "{\n\t.reg .u32 a;\n\t"
        "mapa.shared::cluster.u32 a, %1, %2;\n\t"
        "ld.shared::cluster.u64 %0, [a];\n\t}\n" : "=l"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// 16 bytes of a row's values.
template <typename T> struct alignas(16) PickVec {
    static constexpr int n = 16 / sizeof(T);
    T x[n];
};

// The context's part of the penalties of one request.
struct PickLess { float repetition, frequency, presence; };

__device__ __forceinline__ float pick_less(float x, int count, const PickLess &p) {
    x = x > 0.f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
    x = __fsub_rn(x, __fmul_rn(p.frequency, (float)count));
    return __fsub_rn(x, p.presence);
}

// Shared memory: counts [part], bits [part / 32], bits of each row's own nodes
// [rows][part / 32].
template <typename T>
__global__ void __launch_bounds__(kPickThreads) pick_kernel(const __grid_constant__ PickArgs a) {
    extern __shared__ __align__(16) uint32_t smem[];
    __shared__ unsigned long long best[kPickRows][kPickWarps];
    constexpr int N = PickVec<T>::n;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int rank = (int)cluster_rank(), size = (int)cluster_size();
    const int cluster = blockIdx.x / size;
    const int b = cluster / a.groups, group = cluster - b * a.groups;
    int t0 = b, n = 1;
    if (a.q_start) {
        const int s = a.q_start[b], e = a.q_start[b + 1];
        t0 = min(max(s, 0), a.tokens);
        n = min(min(max(e - s, 0), a.max_q), a.tokens - t0);
        if (tid == 0 && (t0 != s || n != e - s)) atomicOr(a.err, kAttnBadLen);
    }
    const int r0 = group * a.rows, rows = min(a.rows, n - r0);
    if (rows <= 0) return;                  // all blocks of the cluster
    const int words = a.part / 32;
    int *const counts = (int *)smem;
    uint32_t *const occurs = smem + a.part, *const own = occurs + words;
    const bool context = a.history || a.seen;
    PickLess less = {1.f, 0.f, 0.f};
    if (a.repetition) less.repetition = a.repetition[b];
    if (a.frequency) less.frequency = a.frequency[b];
    if (a.presence) less.presence = a.presence[b];
    for (int x = tid; x < kPickRows * kPickWarps; x += kPickThreads) (&best[0][0])[x] = 0;

    for (int pass = 0; pass < a.passes; pass++) {
        const int64_t from = ((int64_t)pass * size + rank) * a.part;
        const int v0 = (int)min(from, (int64_t)a.vocab);
        const int v1 = (int)min(from + a.part, (int64_t)a.vocab);
        __syncthreads();
        if (context) {
            for (int x = tid; x < a.part + words + rows * words; x += kPickThreads) smem[x] = 0;
            __syncthreads();
            if (a.history) {
                const int said = a.history_len[b], len = min(max(said, 0), a.history_wide);
                if (tid == 0 && said != len) atomicOr(a.err, kAttnBadLen);
                const int32_t *const past = a.history + b * a.history_row;
                for (int i = tid; i < len; i += kPickThreads) {
                    const int v = past[i];
                    if (v < v0 || v >= v1) continue;
                    atomicAdd(counts + (v - v0), 1);
                    atomicOr(occurs + (v - v0) / 32, 1u << (v - v0) % 32);
                }
            }
            if (a.seen)
                for (int x = tid; x < rows * n; x += kPickThreads) {
                    const int r = x / n, m = x - r * n;
                    const int v = a.drafted[t0 + m];
                    if (v < v0 || v >= v1 || m >= a.seen_words * 64) continue;
                    const uint64_t *const row = a.seen + (t0 + r0 + r) * a.seen_words;
                    if (row[m >> 6] >> (m & 63) & 1)
                        atomicOr(own + r * words + (v - v0) / 32, 1u << (v - v0) % 32);
                }
            __syncthreads();
        }
        for (int r = 0; r < rows; r++) {
            const int t = t0 + r0 + r;
            const T *const x = (const T *)a.logits + t * a.row;
            T *const y = a.out ? (T *)a.out + t * a.out_row : nullptr;
            const float *const bias = a.bias ? a.bias + b * a.bias_row : nullptr;
            const uint32_t *const allowed = a.allowed ? a.allowed + t * a.allowed_row : nullptr;
            float top = -INFINITY;
            int at = -1;
            auto adjust = [&](float f, int v) {
                if (context) {
                    const int w = (v - v0) / 32, bit = (v - v0) % 32;
                    const bool mine = own[r * words + w] >> bit & 1;
                    if (mine || (occurs[w] >> bit & 1)) {
                        int count = counts[v - v0];
                        if (mine) {
                            const uint64_t *const row = a.seen + t * a.seen_words;
                            for (int m = 0; m < n && m < a.seen_words * 64; m++)
                                if (row[m >> 6] >> (m & 63) & 1) count += a.drafted[t0 + m] == v;
                        }
                        f = pick_less(f, count, less);
                    }
                }
                if (bias) f = __fadd_rn(f, bias[v]);
                if (allowed && !(allowed[v >> 5] >> (v & 31) & 1)) f = -INFINITY;
                if (f > top) {
                    top = f;
                    at = v;
                }
                return f;
            };
            for (int v = v0 + tid; v < v1; v += kPickThreads) {
                const float f = adjust(AttnType<T>::up(x[v]), v);
                if (y) y[v] = AttnType<T>::down(f);
            }
            unsigned long long key = at < 0 ? 0 : pick_key(top, at);
#pragma unroll
            for (int d = 16; d; d >>= 1) key = max(key, __shfl_xor_sync(~0u, key, d));
            if (lane == 0) best[r][warp] = max(best[r][warp], key);
        }
    }
    cluster_sync();
    for (int r = rank * kPickWarps + warp; r < rows; r += size * kPickWarps) {
        unsigned long long key = 0;
        for (int x = lane; x < size * kPickWarps; x += 32)
            key = max(key, cluster_ld64(smem_u32(&best[r][x % kPickWarps]), x / kPickWarps));
#pragma unroll
        for (int d = 16; d; d >>= 1) key = max(key, __shfl_xor_sync(~0u, key, d));
        if (lane == 0) a.picked[t0 + r0 + r] = key ? (int)~(uint32_t)key : -1;
    }
    cluster_sync();                         // no block leaves while its words are read
}

template <typename T>
static int pick_launch(const PickArgs &a, int size, cudaStream_t st) {
    static std::atomic<uint64_t> done;
    const int words = a.part / 32;
    constexpr int most = (kPickPart + kPickPart / 32 * (1 + kPickRows)) * 4;
    static_assert(most + kPickRows * kPickWarps * 8 <= 227 * 1024, "shared memory of a block");
    cudaError_t e = attn_smem(pick_kernel<T>, most, done);
    if (e != cudaSuccess) return cuda_fail(e, "pick smem attribute");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.batch * a.groups * size));
    cfg.blockDim = dim3(kPickThreads);
    cfg.dynamicSmemBytes = a.history || a.seen ? (a.part + words * (1 + a.rows)) * 4 : 0;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = size;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, pick_kernel<T>, a);
    if (e != cudaSuccess) return cuda_fail(e, "pick_kernel");
    count_launch();
    return WARP_OK;
}

}  // namespace warp

using namespace warp;

extern "C" int warp_pick_tokens(const warp_pick_desc *d, void *stream) {
    const char *who = "warp_pick_tokens";
    WARP_ARG(d, "%s: NULL description", who);
    WARP_ARG(d->tokens >= 0 && d->batch >= 0 && d->max_q >= 0 && d->history_wide >= 0,
             "%s: negative size", who);
    WARP_ARG(d->vocab >= 1 && d->vocab < (1 << 30), "%s: a vocabulary of %d", who, d->vocab);
    WARP_ARG(d->type == WARP_T_F32 || d->type == WARP_T_F16 || d->type == WARP_T_BF16,
             "%s: type %d", who, d->type);
    WARP_ARG(d->row >= 0 && d->out_row >= 0 && d->history_row >= 0 && d->bias_row >= 0 &&
                 d->allowed_row >= 0 && d->seen_words >= 0,
             "%s: negative stride", who);
    WARP_ARG(d->q_start || d->tokens == d->batch, "%s: %d rows of %d requests", who, d->tokens,
             d->batch);
    if (d->tokens == 0 || d->batch == 0 || (d->q_start && d->max_q == 0)) return WARP_OK;
    WARP_ARG(d->logits && d->picked, "%s: NULL pointer", who);
    WARP_ARG(!d->history == !d->history_len, "%s: history and history_len go together", who);
    WARP_ARG(!d->drafted == !d->seen && (!d->seen || d->q_start),
             "%s: drafted, seen and q_start go together", who);
    WARP_ARG(((uintptr_t)d->seen & 7) == 0, "%s: the masks are not 8-byte aligned", who);
    const int size_of = d->type == WARP_T_F32 ? 4 : 2;
    WARP_ARG((((uintptr_t)d->logits | (uintptr_t)d->out) & (size_of - 1)) == 0,
             "%s: logits are not aligned to their type", who);
    WARP_ARG(d->out != d->logits || d->out_row == d->row || d->tokens == 1,
             "%s: results in the logits' place have their layout", who);
    PickArgs a = {};
    a.logits = d->logits, a.out = d->out, a.picked = d->picked, a.q_start = d->q_start;
    a.history = d->history, a.history_len = d->history_len, a.drafted = d->drafted;
    a.repetition = d->repetition, a.frequency = d->frequency, a.presence = d->presence;
    a.bias = d->bias, a.allowed = d->allowed, a.seen = d->seen;
    a.row = d->row, a.out_row = d->out_row, a.history_row = d->history_row;
    a.bias_row = d->bias_row, a.allowed_row = d->allowed_row, a.seen_words = d->seen_words;
    a.tokens = d->tokens, a.batch = d->batch, a.vocab = d->vocab;
    a.history_wide = d->history_wide;
    a.max_q = d->q_start ? (d->max_q < d->tokens ? d->max_q : d->tokens) : 1;
    const int rc = attn_err_word(&a.err);
    if (rc) return rc;
    const int size = 8;
    a.part = (int)((cdiv(d->vocab, size) + 31) / 32 * 32);
    if (a.part > kPickPart) a.part = kPickPart;
    a.passes = (int)cdiv(d->vocab, (size_t)a.part * size);
    a.rows = a.max_q < 4 ? a.max_q : 4;
    a.groups = (int)cdiv(a.max_q, a.rows);
    WARP_ARG((int64_t)a.batch * a.groups * size < (int64_t)1 << 31, "%s: %d requests of %d rows",
             who, a.batch, a.max_q);
    cudaStream_t st = (cudaStream_t)stream;
    return d->type == WARP_T_F32   ? pick_launch<float>(a, size, st)
           : d->type == WARP_T_F16 ? pick_launch<__half>(a, size, st)
                                   : pick_launch<__nv_bfloat16>(a, size, st);
}
