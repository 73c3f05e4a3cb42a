// logits.cu — penalties for repeated tokens, biases and masks on logits, and the
// largest of each row.
//
// The logits are read once (and, where they are kept, written once).  Two kernels: the
// first counts each request's history, a block to a slice of the vocabulary, and leaves
// a bit for each token that occurs, and the numbers where there are such bits.  The second streams over the rows, in equal runs, and joins
// a row's parts by an atomic maximum of (logit, token) in one number, which any order
// leaves the same.  A few rows are one kernel's, a cluster of blocks to a row.
//
// Measured: 160 rows of 131072 fp32 22.5 us, 3.7 TB/s; about as many (64 streams of 1 to 5) with
// biases of each stream 37, and with histories of up to 30000 tokens 66; 138 rows of 100003 bf16
// with histories of 8000 and masks, kept, 39.  What bounds it is the arithmetic of each value
// (issue slots are used to 69 and 65 % in the last two) more than the stream, and the
// counting (15 and 7 us) that comes before it.  Tried and slower than two kernels for many
// rows: a cluster that counts for itself (64 streams: 83 to 97), counts in the shared memory of
// others (200), tokens sorted into buckets first (89), penalties spread out densely (86).
//
// Division: x / r for a row's many x and one r is by the reciprocal, kept in two words
// y + z (z what y, rounded, is off by): q = x y + x z is one place off at most, and q + y (x - q r)
// is the quotient rounded to nearest (Markstein, "Computation of elementary functions on
// the IBM RISC System/6000 processor", 1990; the two words are those of Brisebarre, Muller and
// Raina, "Accelerating correctly rounded floating-point division when the divisor is known
// in advance", 2004).  The remainder is exact as long as no number here leaves the normal
// ones; where one could, it divides.
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
    int tokens, batch, vocab, history_wide, max_q;
    // the first kernel's results: [batch][words], and [batch][32 * words]
    uint32_t *bits;
    void *counts;
    int words;                              // of 32 tokens in the vocabulary
    int slice, slices;                      // words a block of the first, blocks a request
    unsigned long long *best;               // [tokens]; and how many pieces are done
    unsigned *done;
    int pieces;                             // of a row, for the second
    int part;                               // tokens a block, where a cluster has a row
};

// ------------------------------------------------------------- the history --

// A block reads all of the history and counts the tokens of its slice.  Slices are as
// large as lets the blocks fill the card once, or as an SM's shared memory allows: with
// smaller ones the histories' reads from the L2 are what takes the time (64 of up to 30000
// tokens, 131072 in the vocabulary: 14 us for the reads alone with slices of an eighth), with
// larger ones SMs have nothing to do (8 requests: 45 us for the call with 16 blocks, 42 with 144).
constexpr int kPickCounters = 1024;         // threads
constexpr int kPickSlice = 2048;            // words of 16-bit counts a block, at most

template <typename C>
__global__ void __launch_bounds__(kPickCounters)
pick_history_kernel(const __grid_constant__ PickArgs a) {
    extern __shared__ __align__(16) uint32_t counts[];  // [slice * 32] of C
    constexpr int PER = 4 / sizeof(C), U = 4;
    pdl_trigger();
    const int tid = threadIdx.x;
    // (2^21 requests and more have blocks whose product is past 31 bits)
    for (int64_t t = (int64_t)blockIdx.x * kPickCounters + tid; t < a.tokens;
         t += (int64_t)gridDim.x * kPickCounters) {
        a.best[t] = 0;
        a.done[t] = 0;
    }
    if (!a.history) return;
    const int b = blockIdx.x / a.slices, w0 = (blockIdx.x - b * a.slices) * a.slice;
    const int n = min(a.slice, a.words - w0), v0 = w0 * 32;
    const int end = min(n * 32, a.vocab - v0);          // tokens of the slice
    const int said = a.history_len[b], len = min(max(said, 0), a.history_wide);
    if (tid == 0 && said != len) atomicOr(a.err, kAttnBadLen);
    const int32_t *const past = a.history + b * a.history_row;
    const int lead = min((int)(-((uintptr_t)past / 4) % 4), len), fours = (len - lead) / 4;
    int4 v[U];
    auto read = [&](int i) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            v[u] = make_int4(-1, -1, -1, -1);
            if (i + u * kPickCounters < fours)
                v[u] = __ldg((const int4 *)(past + lead) + i + u * kPickCounters);
        }
    };
    read(tid);
    for (int x = 4 * tid; x < n * (32 / PER); x += 4 * kPickCounters)
        *(uint4 *)(counts + x) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    auto add = [&](int token) {
        const int at = token - v0;
        if (token >= v0 && at < end)
            atomicAdd(counts + at / PER, 1u << at % PER * (8 * (int)sizeof(C)));
    };
    if (tid < lead) add(past[tid]);
    if (tid < len - lead - 4 * fours) add(past[lead + 4 * fours + tid]);
    for (int i = tid; i < fours; i += U * kPickCounters) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            add(v[u].x);
            add(v[u].y);
            add(v[u].z);
            add(v[u].w);
        }
        read(i + U * kPickCounters);
    }
    __syncthreads();
    // a word of bits from 32 counts, which are written where there is one
    for (int w = tid; w < n; w += kPickCounters) {
        uint32_t bits = 0;
        uint4 z[8 / PER];
#pragma unroll
        for (int q = 0; q < 8 / PER; q++) {
            z[q] = *(const uint4 *)(counts + w * (32 / PER) + 4 * q);
            const uint32_t y[4] = {z[q].x, z[q].y, z[q].z, z[q].w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int at = (4 * q + k) * PER;
                if (PER == 1) {
                    bits |= (uint32_t)(y[k] != 0) << at;
                } else {
                    bits |= (uint32_t)((y[k] & 0xffffu) != 0) << at;
                    bits |= (uint32_t)(y[k] >> 16 != 0) << (at + 1);
                }
            }
        }
        const int64_t word = b * (int64_t)a.words + w0 + w;
        a.bits[word] = bits;
        uint4 *const to = (uint4 *)((C *)a.counts + word * 32);
        if (bits)
#pragma unroll
            for (int q = 0; q < 8 / PER; q++) to[q] = z[q];
    }
}

// ---------------------------------------------------------------- the rows --

// A choice as one number that the larger of two is the better of: larger logit,
// then lower token.  0 is no choice.
__device__ __forceinline__ unsigned long long pick_key(float x, int v) {
    const uint32_t u = __float_as_uint(x + 0.f);        // -0 is 0
    const uint32_t up = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (unsigned long long)up << 32 | (uint32_t)~v;
}

// The warp's largest value.
__device__ __forceinline__ float warp_max(float x) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
    return m;
}

// 16 bytes of a row's values.
template <typename T> struct alignas(16) PickVec {
    static constexpr int n = 16 / sizeof(T);
    T x[n];
};

// The penalties of one request.
struct PickLess {
    float repetition, frequency, presence;
    float inverse, low;                     // of the first, in two words; 0 where it is divided by
};

__device__ __forceinline__ float pick_less(float x, float count, const PickLess &p) {
    x = x > 0.f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
    x = __fsub_rn(x, __fmul_rn(p.frequency, count));
    return __fsub_rn(x, p.presence);
}
// The same of two tame values, by the reciprocal.
__device__ __forceinline__ float2 pick_less2(float x0, float x1, float count0, float count1,
                                             const PickLess &p) {
    const uint64_t x = pair2(x0, x1), inverse = pair2(p.inverse, p.inverse);
    const uint64_t by = pair2(-p.repetition, -p.repetition);
    uint64_t q = fma2(x, inverse, mul2(x, pair2(p.low, p.low)));
    q = fma2(fma2(q, by, x), inverse, q);
    const float2 over = both(q), times = both(mul2(x, by));
    const uint64_t w = pair2(x0 > 0.f ? over.x : -times.x, x1 > 0.f ? over.y : -times.y);
    // one by one: a product of two that is added to would not be rounded by itself
    const uint64_t less = pair2(__fmul_rn(-p.frequency, count0), __fmul_rn(-p.frequency, count1));
    return both(add2(add2(w, less), pair2(-p.presence, -p.presence)));
}
// Whether all x are so far from the normal numbers' ends that the products above are
// exact where they have to be.  A NaN is one with either.
template <int N> __device__ __forceinline__ bool pick_tame(const float (&x)[N]) {
    float lo = fabsf(x[0]), hi = lo;
#pragma unroll
    for (int q = 1; q < N; q++) {
        lo = fminf(lo, fabsf(x[q]));
        hi = fmaxf(hi, fabsf(x[q]));
    }
    return lo >= 0x1p-80f && hi <= 0x1p80f;
}
// A count as a number: 16 bits below the last place of 2^23, and 2^23 taken off.
__device__ __forceinline__ float pick_float(uint16_t c) {
    return __fsub_rn(__uint_as_float(0x4b000000u | c), 8388608.f);
}
__device__ __forceinline__ float pick_float(uint32_t c) { return (float)c; }

// Row t's request b (the last one that starts at or before it), whose node i of n the
// row is.  A row of none is kPickNone and stays as it is; one past the bound is
// kPickPast, which is reported and has no choice.
enum { kPickTaken, kPickNone, kPickPast };
__device__ __forceinline__ int pick_request(const PickArgs &a, int t, int &b, int &i, int &n,
                                            bool report) {
    b = t, i = 0, n = 1;
    if (!a.q_start) return kPickTaken;
    const int lane = threadIdx.x % 32;
    b = -1;
    for (int i0 = 0; i0 < a.batch; i0 += 32) {
        const unsigned hit = __ballot_sync(~0u, i0 + lane < a.batch && a.q_start[i0 + lane] <= t);
        if (hit) b = i0 + 31 - __clz(hit);
        if (hit != ~0u) break;
    }
    if (b < 0) return kPickNone;
    const int s = a.q_start[b], e = a.q_start[b + 1];
    if (t >= e) return kPickNone;
    i = t - s;
    n = min(e - s, a.max_q);
    if (report && threadIdx.x == 0 && (s < 0 || e > a.tokens || i >= n)) atomicOr(a.err, kAttnBadLen);
    if (s < 0 || i >= n) return kPickPast;
    n = min(n, a.tokens - s);
    return kPickTaken;
}

// What a kernel does besides the penalties: asked for each value, this would cost
// more than the rest of the stream.
constexpr int kPickBias = 1, kPickAllowed = 2, kPickKeep = 4;
constexpr int kPickThreads = 256;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kPickOwn = 256;               // nodes' tokens that a block keeps
constexpr int kPickPart = 49152;            // tokens of a row at once, where nodes' are marked
constexpr int kPickPiece = 2048;            // tokens of a row that one block takes, at least
// What a block's start on a row takes, in pieces: who has two rows gets fewer of them (160 rows
// of 131072 22.5 us with 5 and 26 with 0, 8 trees of 26 39 and 42; with 9 and many penalties it is
// slower again).
constexpr int kPickLead = 5;

template <int BYTES>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES)
                 : "memory");
}

// A thread's place in the ring, for each vector under way: the values, the biases of a
// kernel that adds some, and the counts, of which there are twice as many where
// vectors are not aligned to their words.
template <typename T, typename C, int OPT> struct PickSlot {
    static constexpr int n = PickVec<T>::n;
    static constexpr int bias = 16;
    static constexpr int window = n * sizeof(C);        // bytes of a vector's counts
    static constexpr int counts = bias + (OPT & kPickBias ? n * 4 : 0);
    static constexpr int bytes = counts + 2 * window;
    // vectors under way: what lets four blocks fit an SM, with biases and counts three.  The
    // stream is as much arithmetic as memory, so more warps are worth more than deeper rings: 8
    // masked trees of 26 in bf16 take 45 us so and 49 us with eight vectors and two blocks.
    static constexpr int ahead = 192 / bytes > 3 ? 192 / bytes : 3;
    static constexpr int round = bytes * kPickThreads, ring = ahead * round;
    static_assert(n * ahead <= 32, "what is hit in them, a bit each, is one word");
};

// The rows lie one behind another in pieces of kPickPiece tokens, and the blocks take
// equal runs of them; a row's part in a run is gone through at once.
//
// A thread's vectors of 16 bytes come through a ring of its own in shared memory: the
// loads that are under way take no registers, and no thread waits for another.  With a
// vector come its biases and, if one of its tokens occurs, its counts.  That is
// known ahead: a warp's bits of G vectors are one register a lane (N words a vector, and one
// more where they are not aligned), asked for G vectors before they are needed.
template <typename T, typename C, int OPT>
__global__ void __launch_bounds__(kPickThreads, 4)
pick_rows_kernel(const __grid_constant__ PickArgs a) {
    using Slot = PickSlot<T, C, OPT>;
    constexpr int N = Slot::n, STEP = kPickThreads * N, R = Slot::ahead;
    constexpr int G = 32 / (N + 1);
    constexpr bool BIAS = OPT & kPickBias, ALLOWED = OPT & kPickAllowed, KEEP = OPT & kPickKeep;
    __shared__ uint32_t drafts[kPickPart / 32 + 1];     // the row's nodes' tokens, a bit each
    __shared__ int own[kPickOwn];                       // and themselves
    __shared__ int n_own;
    __shared__ unsigned long long best[kPickWarps];
    extern __shared__ __align__(16) uint8_t ring[];     // [vector][part of a slot][thread]
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    // this block's pieces
    const int64_t span = a.pieces + kPickLead, all = a.tokens * span, blocks = gridDim.x;
    auto piece_of = [&](int64_t u) {
        const int64_t t = u / span;
        return t * a.pieces + max((int)(u - t * span) - kPickLead, 0);
    };
    const int64_t last = piece_of((blockIdx.x + 1) * all / blocks);
    bool waited = false;
    for (int64_t piece = piece_of(blockIdx.x * all / blocks), next; piece < last; piece = next) {
        const int t = (int)(piece / a.pieces), first = (int)(piece - (int64_t)t * a.pieces);
        next = min(last, piece - first + a.pieces);
        if (a.seen) next = min(next, piece + kPickPart / kPickPiece);
        const int v0 = first * kPickPiece;
        const int v1 = (int)min((int64_t)a.vocab, v0 + (next - piece) * kPickPiece);
        const T *const x = (const T *)a.logits + t * a.row;
        T *const y = KEEP ? (T *)a.out + t * a.out_row : nullptr;
        // Vectors are aligned in memory, from value a0 on; what is left over at the
        // part's ends goes one by one.
        const int a0 = min(v1, v0 + (int)(-((uintptr_t)(x + v0) / sizeof(T)) % N));
        const int vectors = (v1 - a0) / N, end = a0 + vectors * N;
        const int rounds = (vectors + kPickThreads - 1) / kPickThreads;
        const int v_tid = a0 + tid * N, skew = a0 % N;
        // The first vectors are asked for before it is known whose row this is.
        const uint32_t ring0 = smem_u32(ring);
        auto part_of = [&](uint32_t at, int part, int bytes) {
            return at + part * kPickThreads + tid * bytes;
        };
        auto ask_row = [&](uint32_t at, int v) {
            if (v < end) cp_async16(part_of(at, 0, 16), x + v);
        };
#pragma unroll 1
        for (int k = 0; k < R - 1; k++) ask_row(ring0 + k * Slot::round, v_tid + k * STEP);
        int b, i, n;
        if (const int not_taken = pick_request(a, t, b, i, n, true)) {
            if (not_taken == kPickPast && tid == 0) a.picked[t] = -1;
            cp_async_commit();
            cp_async_wait<0>();
            continue;
        }
        const int t0 = t - i;
        const uint64_t *const sees = a.seen ? a.seen + t * a.seen_words : nullptr;
        const float *const bias = BIAS ? a.bias + b * a.bias_row : nullptr;
        const uint32_t *const allowed = ALLOWED ? a.allowed + t * a.allowed_row : nullptr;
        const uint32_t *const occurs = a.history ? a.bits + b * (int64_t)a.words : nullptr;
        const C *const counts = (const C *)a.counts + b * (int64_t)a.words * 32;
        const bool y_vec = ((uintptr_t)(y + a0) & 15) == 0;
        const bool bias_vec = ((uintptr_t)(bias + a0) & 15) == 0;
        PickLess less = {1.f, 0.f, 0.f, 0.f, 0.f};
        if (a.repetition) less.repetition = a.repetition[b];
        if (a.frequency) less.frequency = a.frequency[b];
        if (a.presence) less.presence = a.presence[b];
        if (less.repetition >= 0x1p-20f && less.repetition <= 0x1p20f) {
            less.inverse = __frcp_rn(less.repetition);
            less.low = __fmul_rn(__fmaf_rn(-less.inverse, less.repetition, 1.f), less.inverse);
        }
        if (sees) {
            __syncthreads();                // the last part's are read
            for (int w = tid; w < (v1 - v0 + 31) / 32 + 1; w += kPickThreads) drafts[w] = 0;
            if (tid == 0) n_own = 0;
            __syncthreads();
            for (int m = tid; m < n && m < a.seen_words * 64; m += kPickThreads) {
                const int v = a.drafted[t0 + m];
                if (!(sees[m >> 6] >> (m & 63) & 1) || v < v0 || v >= v1) continue;
                const int k = atomicAdd(&n_own, 1);
                if (k < kPickOwn) own[k] = v;
                atomicOr(drafts + (v - v0) / 32, 1u << (v - v0) % 32);
            }
            __syncthreads();
        }
        float top = -INFINITY;
        int at = -1;

        // how many of the nodes that the row sees have token v
        auto nodes_with = [&](int v) {
            int count = 0;
            if (n_own <= kPickOwn)
                for (int k = 0; k < n_own; k++) count += own[k] == v;
            else
                for (int m = 0; m < n && m < a.seen_words * 64; m++)
                    if (sees[m >> 6] >> (m & 63) & 1) count += a.drafted[t0 + m] == v;
            return count;
        };
        // the value of token v less what its context takes off, the long way
        auto adjusted = [&](float f, int v) {
            uint32_t count = 0;
            if (occurs && (occurs[v >> 5] >> (v & 31) & 1)) count = (uint32_t)counts[v];
            if (sees && (drafts[(v - v0) >> 5] >> (v & 31) & 1)) count += nodes_with(v);
            return count ? pick_less(f, (float)count, less) : f;
        };
        auto single = [&](int v) {
            float f = adjusted(AttnType<T>::up(x[v]), v);
            if (BIAS) f = __fadd_rn(f, __ldg(bias + v));
            if (ALLOWED && !(__ldg(allowed + (v >> 5)) >> (v & 31) & 1)) f = -INFINITY;
            if (f > top || (f == top && v < at)) {
                top = f;
                at = v;
            }
            if (KEEP) y[v] = AttnType<T>::down(f);
        };
        const int lane_g = lane / (N + 1), lane_w = lane % (N + 1);
        const int word0 = ((a0 + lane_g * STEP + warp * 32 * N) >> 5) + lane_w;
        // a lane's word of the bits of G vectors from round k on
        auto hits_of = [&](int k) {
            const int w = word0 + k * (STEP / 32);
            if (lane_g >= G || w >= a.words || k >= rounds) return 0u;
            uint32_t bits = occurs ? occurs[w] : 0;
            if (sees && w <= (v1 - v0 + 31) / 32 + (v0 >> 5)) bits |= drafts[w - (v0 >> 5)];
            return bits;
        };
        auto may_of = [&](int k) {
            const int w = word0 + k * (STEP / 32);
            return ALLOWED && lane_g < G && w < a.words && k < rounds ? __ldg(allowed + w) : 0u;
        };
        const int shift = (a0 + lane * N) & 31, in_vector = ((a0 & 31) + lane * N) >> 5;
        auto bits_of = [&](uint32_t word, int g) {
            const uint32_t lo = __shfl_sync(~0u, word, g * (N + 1) + in_vector);
            const uint32_t hi = __shfl_sync(~0u, word, g * (N + 1) + min(in_vector + 1, N));
            return __funnelshift_r(lo, hi, shift) & ((1u << N) - 1);
        };
        if (!waited) pdl_wait();
        waited = true;
        const bool context = occurs || sees;
        // Vectors asked for so far: round `ask`, number `ask_g` of the group whose bits are
        // in `ask_hits`, with the next group's behind them.  What is hit in the vectors
        // under way queues in `queue`, N bits each.
        int ask = 0, ask_g = 0;
        uint32_t ask_hits = context ? hits_of(0) : 0, next_hits = context ? hits_of(G) : 0;
        uint32_t queue = 0;
        // places in the ring of what is asked for next, and of what is next in turn
        uint32_t ask_at = ring0, turn_at = ring0;
        auto behind = [&](uint32_t at) {
            return at + Slot::round == ring0 + Slot::ring ? ring0 : at + Slot::round;
        };
        auto fetch = [&](bool row) {
            const int v = v_tid + ask * STEP;
            uint32_t hit = 0;
            if (context) {
                hit = bits_of(ask_hits, ask_g);
                if (++ask_g == G) {
                    ask_g = 0;
                    ask_hits = next_hits;
                    next_hits = hits_of(ask + 1 + G);
                }
                if (v >= end) hit = 0;
                queue = queue >> N | hit << N * (R - 1);
            }
            if (row) ask_row(ask_at, v);
            if (BIAS && v < end && bias_vec) {
#pragma unroll
                for (int k = 0; k < N; k += 4)
                    cp_async16(part_of(ask_at, Slot::bias, 4 * N) + 4 * k, bias + v + k);
            }
            if (hit && occurs) {
                const C *const z = counts + (v - skew);
                const uint32_t to = part_of(ask_at, Slot::counts, 2 * Slot::window);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    if (k && !skew) break;
#pragma unroll
                    for (int q = 0; q < Slot::window; q += 8)
                        cp_async_small<8>(to + k * Slot::window + q, (const char *)(z + k * N) + q);
                }
            }
            cp_async_commit();
            ask++;
            ask_at = behind(ask_at);
        };
#pragma unroll 1
        for (int k = 0; k < R - 1; k++) fetch(false);
        uint32_t may = may_of(0), next_may = may_of(G);
        int g = 0;
        float bound = -INFINITY;            // what the warp has seen is at least this
#pragma unroll 1
        for (int k = 0; k < rounds; k++) {
            fetch(true);
            const uint32_t hit = queue & ((1u << N) - 1);
            const uint32_t allow = ALLOWED ? bits_of(may, g) : 0;
            cp_async_wait<R - 1>();
            const int v = v_tid + k * STEP;
            float f[N], most = -INFINITY;
            if (v < end) {
                PickVec<T> raw;
                *(uint4 *)&raw = lds_u4(part_of(turn_at, 0, 16));
#pragma unroll
                for (int q = 0; q < N; q++) f[q] = AttnType<T>::up(raw.x[q]);
                if (hit) {
                    const int d = (v - v0) >> 5;
                    const uint32_t mine =
                        sees ? __funnelshift_r(drafts[d], drafts[d + 1], v & 31) & hit : 0;
                    if (__builtin_expect(less.inverse != 0.f && !mine && pick_tame(f), 1)) {
                        const C *const z = (const C *)(
                            ring + (part_of(turn_at, Slot::counts, 2 * Slot::window) - ring0));
                        alignas(16) C c[N];
                        if (!skew) {
#pragma unroll
                            for (int q = 0; q < Slot::window; q += 8)
                                *(uint2 *)((char *)c + q) = *(const uint2 *)((const char *)z + q);
                        } else {
#pragma unroll
                            for (int q = 0; q < N; q++) c[q] = z[q + skew];
                        }
#pragma unroll
                        for (int q = 0; q < N; q += 2) {
                            const float2 w = pick_less2(f[q], f[q + 1], pick_float(c[q]),
                                                        pick_float(c[q + 1]), less);
                            f[q] = hit >> q & 1 ? w.x : f[q];
                            f[q + 1] = hit >> q & 2 ? w.y : f[q + 1];
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < N; q++)
                            if (hit >> q & 1) f[q] = adjusted(f[q], v + q);
                    }
                }
                if (BIAS) {
                    alignas(16) float w[N];
                    if (bias_vec) {
#pragma unroll
                        for (int q = 0; q < N; q += 4)
                            *(uint4 *)(w + q) = lds_u4(part_of(turn_at, Slot::bias, 4 * N) + 4 * q);
                    } else {
#pragma unroll
                        for (int q = 0; q < N; q++) w[q] = __ldg(bias + v + q);
                    }
#pragma unroll
                    for (int q = 0; q < N; q += 2) {
                        const float2 y = both(add2(pair2(f[q], f[q + 1]), pair2(w[q], w[q + 1])));
                        f[q] = y.x, f[q + 1] = y.y;
                    }
                }
#pragma unroll
                for (int q = 0; q < N; q++) {
                    if (ALLOWED && !(allow >> q & 1)) f[q] = -INFINITY;
                    most = fmaxf(most, f[q]);
                }
                if (KEEP) {
                    PickVec<T> z;
#pragma unroll
                    for (int q = 0; q < N; q++) z.x[q] = AttnType<T>::down(f[q]);
                    if (y_vec) {
                        *(uint4 *)(y + v) = *(const uint4 *)&z;
                    } else {
#pragma unroll
                        for (int q = 0; q < N; q++) y[v + q] = z.x[q];
                    }
                }
            }
            if (__any_sync(~0u, most > bound)) {
                if (most > top) {
                    top = most;
#pragma unroll
                    for (int q = N - 1; q >= 0; q--)
                        if (f[q] == most) at = v + q;
                }
                bound = warp_max(top);
            }
            if (ALLOWED && ++g == G) {
                g = 0;
                may = next_may;
                next_may = may_of(k + 1 + G);
            }
            turn_at = behind(turn_at);
        }
        cp_async_wait<0>();
        if (tid < a0 - v0) single(v0 + tid);
        if (tid < v1 - end) single(end + tid);

        unsigned long long key = at < 0 ? 0 : pick_key(top, at);
#pragma unroll
        for (int d = 16; d; d >>= 1) key = max(key, __shfl_xor_sync(~0u, key, d));
        __syncthreads();                    // the last part's are read
        if (lane == 0) best[warp] = key;
        __syncthreads();
        if (tid) continue;
#pragma unroll
        for (int k = 1; k < kPickWarps; k++) key = max(key, best[k]);
        if (v1 - v0 < a.vocab) {
            // the last of the row's parts, whoever has it, says what is picked
            const unsigned mine = (unsigned)(next - piece);
            atomicMax(a.best + t, key);
            __threadfence();
            if (atomicAdd(a.done + t, mine) + mine < (unsigned)a.pieces) continue;
            __threadfence();
            key = atomicMax(a.best + t, 0ull);
        }
        a.picked[t] = key ? (int)~(uint32_t)key : -1;
    }
    if (!waited) pdl_wait();                // a grid is not complete before the one before it
}

// ---------------------------------------------------------------- few rows --

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// A word of block `rank`'s shared memory, at the address that it has in this one's.
__device__ __forceinline__ unsigned long long cluster_u64(const void *p, uint32_t rank) {
    unsigned long long v;
    asm volatile(
        "{\n\t.reg .u32 a;\n\t"
        "mapa.shared::cluster.u32 a, %1, %2;\n\t"
        "ld.shared::cluster.u64 %0, [a];\n\t}\n"
        : "=l"(v) : "r"(smem_u32(p)), "r"(rank) : "memory");
    return v;
}

constexpr int kPickCluster = 8;
constexpr int kPickFewPart = 16384;         // tokens a block, at most
constexpr int kPickFewValues = 6 << 20;     // and logits of a call
constexpr int kPickFewHistory = 16384;      // and places of a history, which each block reads

// A cluster has a row, each block a part of the vocabulary, whose tokens it counts for
// itself: one launch and no scratch, and better as long as rows are few (on the device,
// against the two kernels: a row of 32000 behind 700 tokens 5.3 us and 8.2, 32 of 131072
// with biases behind 8000 tokens each 18.6 and 21.7, 100 of 60000 behind 700 21.7 and 22.3; 80 of
// 75000 with biases behind 8000 34.0 and 30.4, as each row counts its history anew).
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) pick_few_kernel(const __grid_constant__ PickArgs a) {
    extern __shared__ __align__(16) uint32_t counts[];  // [part]
    constexpr int U = 8, WARPS = THREADS / 32;
    __shared__ unsigned long long best[WARPS];
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int rank = (int)cluster_rank(), t = blockIdx.x / kPickCluster;
    const int v0 = min(rank * a.part, a.vocab), v1 = min(v0 + a.part, a.vocab);
    int b = t, i = 0, n = 1;
    if (const int not_taken = pick_request(a, t, b, i, n, rank == 0)) {     // in all of the cluster
        if (not_taken == kPickPast && rank == 0 && tid == 0) a.picked[t] = -1;
        return;
    }
    const int t0 = t - i;
    const bool context = a.history || a.seen;
    PickLess less = {1.f, 0.f, 0.f, 0.f, 0.f};
    if (a.repetition) less.repetition = a.repetition[b];
    if (a.frequency) less.frequency = a.frequency[b];
    if (a.presence) less.presence = a.presence[b];
    if (context) {
        for (int x = 4 * tid; x < a.part; x += 4 * THREADS)
            *(uint4 *)(counts + x) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        auto add = [&](int v) {
            if (v >= v0 && v < v1) atomicAdd(counts + (v - v0), 1u);
        };
        if (a.history) {
            const int said = a.history_len[b], len = min(max(said, 0), a.history_wide);
            if (tid == 0 && said != len) atomicOr(a.err, kAttnBadLen);
            const int32_t *const past = a.history + b * a.history_row;
            for (int x = tid; x < len; x += U * THREADS) {
                int v[U];
#pragma unroll
                for (int u = 0; u < U; u++)
                    v[u] = x + u * THREADS < len ? __ldg(past + x + u * THREADS) : -1;
#pragma unroll
                for (int u = 0; u < U; u++) add(v[u]);
            }
        }
        if (a.seen) {
            const uint64_t *const sees = a.seen + t * a.seen_words;
            for (int m = tid; m < n && m < a.seen_words * 64; m += THREADS)
                if (sees[m >> 6] >> (m & 63) & 1) add(a.drafted[t0 + m]);
        }
        __syncthreads();
    }
    const T *const x = (const T *)a.logits + t * a.row;
    T *const y = a.out ? (T *)a.out + t * a.out_row : nullptr;
    const float *const bias = a.bias ? a.bias + b * a.bias_row : nullptr;
    const uint32_t *const allowed = a.allowed ? a.allowed + t * a.allowed_row : nullptr;
    float top = -INFINITY;
    int at = -1;
    for (int base = v0 + tid; base < v1; base += U * THREADS) {
        float f[U], w[U];
        uint32_t may[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = base + u * THREADS;
            f[u] = v < v1 ? AttnType<T>::up(x[v]) : -INFINITY;
            w[u] = bias && v < v1 ? __ldg(bias + v) : 0.f;
            may[u] = allowed && v < v1 ? __ldg(allowed + (v >> 5)) : ~0u;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = base + u * THREADS;
            if (v >= v1) break;
            const uint32_t count = context ? counts[v - v0] : 0;
            if (count) f[u] = pick_less(f[u], (float)count, less);
            if (bias) f[u] = __fadd_rn(f[u], w[u]);
            if (!(may[u] >> (v & 31) & 1)) f[u] = -INFINITY;
            if (f[u] > top) {
                top = f[u];
                at = v;
            }
            if (y) y[v] = AttnType<T>::down(f[u]);
        }
    }
    unsigned long long key = at < 0 ? 0 : pick_key(top, at);
#pragma unroll
    for (int d = 16; d; d >>= 1) key = max(key, __shfl_xor_sync(~0u, key, d));
    if (lane == 0) best[warp] = key;
    cluster_sync();
    if (rank == 0 && warp == 0) {
        key = 0;
        for (int k = lane; k < kPickCluster * WARPS; k += 32)
            key = max(key, cluster_u64(best + k % WARPS, k / WARPS));
#pragma unroll
        for (int d = 16; d; d >>= 1) key = max(key, __shfl_xor_sync(~0u, key, d));
        if (lane == 0) a.picked[t] = key ? (int)~(uint32_t)key : -1;
    }
    cluster_sync();                         // no block leaves while its words are read
}

// ------------------------------------------------------------ host side --

// Scratch: the choices and how many pieces are done, the history's bits and counts.
struct PickPlan {
    int words, slice, slices, pieces;
    bool wide;                              // counts of 32 bits
    int part;                               // of pick_few_kernel; 0: not its
    int64_t done_at, bits_at, counts_at, bytes;
};

static int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

static PickPlan pick_plan(const warp_pick_desc *d) {
    PickPlan p = {};
    const bool past = d->history || d->history_len;
    p.words = (d->vocab + 31) / 32;
    p.part = (p.words + kPickCluster - 1) / kPickCluster * 32;
    if ((int64_t)d->tokens * d->vocab <= kPickFewValues && p.part <= kPickFewPart &&
        (!past || d->history_wide <= kPickFewHistory))
        return p;
    p.part = 0;
    // 16 bits where no history is long enough to outgrow them
    p.wide = d->history_wide >= 65536;
    const int most = p.wide ? kPickSlice / 2 : kPickSlice;
    const int least = (p.words + most - 1) / most, room = 148 / (d->batch ? d->batch : 1);
    p.slices = room > least ? room : least;
    p.slice = (p.words + p.slices - 1) / p.slices;
    p.slices = (p.words + p.slice - 1) / p.slice;
    p.pieces = (d->vocab + kPickPiece - 1) / kPickPiece;
    int64_t at = align256((int64_t)d->tokens * 8);
    p.done_at = at;
    at += align256((int64_t)d->tokens * 4);
    p.bits_at = at;
    if (past) {
        at += align256((int64_t)d->batch * p.words * 4);
        p.counts_at = at;
        // a vector's window may reach past the last word's
        at += align256(((int64_t)d->batch * p.words + 1) * 32 * (p.wide ? 4 : 2));
    } else if (p.pieces == 1) {
        at = 0;
    }
    p.bytes = at;
    return p;
}

template <typename C>
static int pick_history(const PickArgs &a, cudaStream_t st) {
    static std::atomic<uint64_t> done;
    constexpr int most = kPickSlice * 32 * 2;
    cudaError_t e = attn_smem(pick_history_kernel<C>, most, done);
    if (e != cudaSuccess) return cuda_fail(e, "pick smem attribute");
    e = attn_start(pick_history_kernel<C>,
                   dim3(a.history ? (unsigned)a.batch * a.slices : cdiv(a.tokens, kPickCounters)),
                   kPickCounters, a.history ? (size_t)a.slice * 32 * sizeof(C) : 0, st, true, a);
    if (e != cudaSuccess) return cuda_fail(e, "pick_history_kernel");
    count_launch();
    return WARP_OK;
}

template <typename T, typename C, int OPT>
static int pick_rows(const PickArgs &a, bool first, cudaStream_t st) {
    static std::atomic<uint64_t> done;
    constexpr int ring = PickSlot<T, C, OPT>::ring, fixed = kPickPart / 8 + 4 * kPickOwn + 256;
    static_assert(ring + fixed <= 227 * 1024, "shared memory of a block");
    cudaError_t e = attn_smem(pick_rows_kernel<T, C, OPT>, ring, done);
    if (e != cudaSuccess) return cuda_fail(e, "pick smem attribute");
    // as many blocks as fit, by their shared memory
    constexpr int fit = 228 * 1024 / (ring + fixed + 1024);
    const int64_t all = (int64_t)a.tokens * a.pieces, room = (fit < 4 ? fit : 4) * 148;
    e = attn_start(pick_rows_kernel<T, C, OPT>, dim3((unsigned)(all < room ? all : room)),
                   kPickThreads, ring, st, first, a);
    if (e != cudaSuccess) return cuda_fail(e, "pick_rows_kernel");
    count_launch();
    return WARP_OK;
}

template <typename T, int THREADS> static int pick_few(const PickArgs &a, cudaStream_t st) {
    static std::atomic<uint64_t> done;
    cudaError_t e = attn_smem(pick_few_kernel<T, THREADS>, kPickFewPart * 4, done);
    if (e != cudaSuccess) return cuda_fail(e, "pick smem attribute");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.tokens * kPickCluster);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = a.history || a.seen ? a.part * 4 : 0;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = kPickCluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, pick_few_kernel<T, THREADS>, a);
    if (e != cudaSuccess) return cuda_fail(e, "pick_few_kernel");
    count_launch();
    return WARP_OK;
}

template <typename T, typename C>
static int pick_run(const PickArgs &a, cudaStream_t st) {
    // more threads a block as long as the card holds all of them, two blocks an SM (16 rows of
    // 131072 9.0 us and 10.3 with 256 threads, 100 of 60000 20.1 and 13.8)
    if (a.part && a.tokens * kPickCluster <= 2 * 148) return pick_few<T, 512>(a, st);
    if (a.part) return pick_few<T, 256>(a, st);
    const bool alone = !a.history && a.pieces == 1;
    if (!alone) {
        const int rc = pick_history<C>(a, st);
        if (rc) return rc;
    }
    switch ((a.bias ? kPickBias : 0) | (a.allowed ? kPickAllowed : 0) | (a.out ? kPickKeep : 0)) {
    case 0: return pick_rows<T, C, 0>(a, alone, st);
    case 1: return pick_rows<T, C, 1>(a, alone, st);
    case 2: return pick_rows<T, C, 2>(a, alone, st);
    case 3: return pick_rows<T, C, 3>(a, alone, st);
    case 4: return pick_rows<T, C, 4>(a, alone, st);
    case 5: return pick_rows<T, C, 5>(a, alone, st);
    case 6: return pick_rows<T, C, 6>(a, alone, st);
    default: return pick_rows<T, C, 7>(a, alone, st);
    }
}

static int pick_check(const warp_pick_desc *d) {
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
    WARP_ARG(d->batch <= (1 << 27), "%s: %d requests", who, d->batch);
    return WARP_OK;
}

}  // namespace warp

using namespace warp;

extern "C" int64_t warp_pick_scratch(const warp_pick_desc *d) {
    const int rc = pick_check(d);
    return rc ? rc : pick_plan(d).bytes;
}

extern "C" int warp_pick_tokens(const warp_pick_desc *d, void *scratch, void *stream) {
    const char *who = "warp_pick_tokens";
    int rc = pick_check(d);
    if (rc) return rc;
    if (d->tokens == 0 || d->batch == 0 || (d->q_start && d->max_q == 0)) return WARP_OK;
    WARP_ARG(d->logits && d->picked, "%s: NULL pointer", who);
    // no address is needed for a history without places
    WARP_ARG(!d->history == !d->history_len || (d->history_len && d->history_wide == 0),
             "%s: history and history_len go together", who);
    WARP_ARG(!d->drafted == !d->seen && (!d->seen || d->q_start),
             "%s: drafted, seen and q_start go together", who);
    WARP_ARG(((uintptr_t)d->seen & 7) == 0, "%s: the masks are not 8-byte aligned", who);
    const int size_of = d->type == WARP_T_F32 ? 4 : 2;
    WARP_ARG((((uintptr_t)d->logits | (uintptr_t)d->out) & (size_of - 1)) == 0,
             "%s: logits are not aligned to their type", who);
    WARP_ARG(d->out != d->logits || d->out_row == d->row || d->tokens == 1,
             "%s: results in the logits' place have their layout", who);
    const PickPlan p = pick_plan(d);
    WARP_ARG(p.bytes == 0 || (scratch && ((uintptr_t)scratch & 255) == 0),
             "%s: scratch must be 256-byte aligned", who);
    WARP_ARG((int64_t)d->batch * p.slices < (int64_t)1 << 31, "%s: %d requests", who, d->batch);
    PickArgs a = {};
    a.logits = d->logits, a.out = d->out, a.picked = d->picked, a.q_start = d->q_start;
    // without places the lengths alone are looked at, and any address says that there are some
    a.history = d->history ? d->history : d->history_len;
    a.history_len = d->history_len, a.drafted = d->drafted;
    a.repetition = d->repetition, a.frequency = d->frequency, a.presence = d->presence;
    a.bias = d->bias, a.allowed = d->allowed, a.seen = d->seen;
    a.row = d->row, a.out_row = d->out_row, a.history_row = d->history_row;
    a.bias_row = d->bias_row, a.allowed_row = d->allowed_row, a.seen_words = d->seen_words;
    a.tokens = d->tokens, a.batch = d->batch, a.vocab = d->vocab;
    a.history_wide = d->history_wide, a.max_q = d->max_q;
    char *const s = (char *)scratch;
    a.best = (unsigned long long *)s, a.done = (unsigned *)(s + p.done_at);
    a.bits = (uint32_t *)(s + p.bits_at), a.counts = s + p.counts_at;
    a.words = p.words, a.slice = p.slice, a.slices = p.slices, a.pieces = p.pieces;
    a.part = p.part;
    rc = attn_err_word(&a.err);
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (d->type == WARP_T_F32)
        return p.wide ? pick_run<float, uint32_t>(a, st) : pick_run<float, uint16_t>(a, st);
    if (d->type == WARP_T_F16)
        return p.wide ? pick_run<__half, uint32_t>(a, st) : pick_run<__half, uint16_t>(a, st);
    return p.wide ? pick_run<__nv_bfloat16, uint32_t>(a, st)
                  : pick_run<__nv_bfloat16, uint16_t>(a, st);
}
