// attn_umma.cuh — attention over paged keys and values for many query rows a
// key head: prompts, chunks and the rows of a batch behind a shared prefix.
//
// A CTA holds 256 rows (token, head of the group) of one kv head as two tiles
// of 128 and walks the keys a tile of 128 a step. Per step and row tile, on the
// tensor cores with the accumulators in tensor memory:
//     S = Q K^T      (both from shared memory, 128B-swizzled, K-major)
//     O += P V       (P from tensor memory, V as it lies: N-major)
// and between them, two threads a row: the running maximum m, p = 2^(c s - c m)
// and the sum l. P takes the place of S, half of each thread's share at a time,
// so that O += P V starts on the first while the second is computed. While one
// row tile's exponentials are computed the other's products run.
//
// The maximum that p is measured from moves only when a row outgrows it by
// 2^8 (fp16: 2^4), so the accumulated O is rescaled rarely; p then stays below 2^8
// (fp16, whose weights attn_lift raises: 2^15), which the type holds, and the result
// is the same as O and l carry the same factor.
//
// What bounds it: per pair of 128 x 128 tiles the products take
// 2 * 2 * 128 * 128 * D / 4096 FMA a clock = 2048 cycles at D = 128 (half at
// 64), and so do 2 * 128 * 128 exponentials at 16 a clock; a row tile's step is
// its softmax and then its products, and two row tiles in turn do not quite hide
// the one behind the other. Measured with 256 rows on each of 148 SMs and 4096
// keys: 59.6 us, 1333 TFLOP/s at D = 128; 774 to 797 TFLOP/s at 64, 49.8 us at
// best; whatever the page size. Tried and slower: two places of S for 64 keys
// each (966), P apart from S with 80 keys a step (904 to 1031), one warp a 32
// rows (843), one loading warp for both (1207 with pages of 16, whose boxes it
// issues one after another).
//
// Warps: 0-7 rows of tile 0, 8-15 rows of tile 1, two warps a 32 rows, each with
// half the keys of a step (with one, a scheduler has two warps, which do not hide
// each other's latency); 16 issues the products, 17 loads keys and 18 values by TMA,
// a box a page (its issue takes some 70 cycles), into a ring of tiles.
//
// Nodes of trees see the keys before their tree and the bits of their row of masks
// (kAttnTree): only the last steps look at them, others cost what they cost without.
// With few rows a request and lengths that differ, a block takes a run of the batch's
// key tiles instead (kAttnTreeRuns; AttnRuns), which is bound by the keys' stream: the
// two row tiles take the run's tasks in turn, one's rows are written while the other's keys
// come, and the keys' ring goes on from task to task.  32 trees of up to 16 nodes, 56 heads
// of 128 over 8, behind up to 8192 keys: 141 us, 4.7 TB/s.  Two places of scores in turn, the
// next ones there before a step's weights, took 138 and were wrong: the barrier at a task's end
// could be one use behind, so that results were read before the last products, and a wait put
// before it was one use ahead and gave up.
#pragma once
#include "attn.cuh"
#include "umma.cuh"

#include <cuda.h>

namespace warp {
namespace {

constexpr int kRows = 128;                  // rows a tile
// With runs the rows' warps need more registers than an even share, which four other
// warps give up: 512 * 104 + 128 * 64 is what 640 threads start with, 96 each.
constexpr int kRowRegs = 104, kOtherRegs = 64;
__host__ __device__ constexpr int threads_of(AttnKind kind) {
    return (kind == kAttnTreeRuns ? 20 : 19) * 32;
}
static_assert(512 * kRowRegs + 128 * kOtherRegs <= 640 * 96, "no warp waits for registers");

template <int D> struct Lay {
    static constexpr int keys = attn_wide(D);           // keys a tile
    static constexpr int q_tile = kRows * D * 2;
    static constexpr int q_half = kRows * 128;          // 64 columns of a tile
    static constexpr int kv_tile = keys * D * 2;
    static constexpr int kv_half = keys * 128;
    static constexpr int stages = D == 128 ? 5 : 8;
    static constexpr int ring = 2 * q_tile;
    static constexpr int swap = ring + stages * kv_tile;  // [tile][half][row] fp32
    static constexpr int bars = swap + 4 * kRows * 4;
    static constexpr int cols = keys / 2;               // keys of a row and thread
    // offsets in the barrier section
    static constexpr int kv_full = 0, kv_empty = kv_full + stages * 8,
                         q_full = kv_empty + stages * 8, s_full = q_full + 16,
                         p_full = s_full + 16, o_end = p_full + 32, drain = o_end + 16,
                         tmem = drain + 8, fail = tmem + 4, dirty = fail + 4;
    // a word for each of four tasks, as the row tiles' may be up to three apart; a row
    // tile's notes
    static constexpr int note = dirty + 16;
    static constexpr int notes = 20;
    static constexpr int bytes = bars + note + 2 * notes * 4;
    static_assert(bytes <= 227 * 1024, "shared memory of a block");
    static_assert(cols % 32 == 0 && keys == 128, "whole boxes, swizzle atoms of 8 rows");
    // tensor memory columns
    static constexpr int o(int t) { return t * D; }
    static constexpr int s(int t) { return 2 * D + t * keys; }
    static_assert(2 * D + 2 * keys <= 512, "tensor memory");
};

// Shared-memory matrix descriptor, 128-byte swizzle (layout type 2).
__device__ __forceinline__ uint64_t desc128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return umma::desc(saddr, lbo, sbo) | ((uint64_t)2 << 61);
}

template <typename T> constexpr uint32_t fmt16();
template <> constexpr uint32_t fmt16<__half>() { return 0; }
template <> constexpr uint32_t fmt16<__nv_bfloat16>() { return 1; }

// kind::f16 with fp32 D of 128 x N; b_mn: B is N-major.
template <typename T> __host__ __device__ constexpr uint32_t idesc(int N, bool b_mn) {
    return (1u << 4) | (fmt16<T>() << 7) | (fmt16<T>() << 10) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}

// The products and commits are issued by one lane, by predicate rather than by
// branch: in uniform control flow the descriptors stay in uniform registers,
// where the instruction wants them.
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b,
                                       uint32_t id, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"((uint32_t)accumulate), "r"(leader)
        : "memory");
}
// A from tensor memory.
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b,
                                       uint32_t id, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
        ::"r"(d), "r"(a), "l"(b), "r"(id), "r"((uint32_t)accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t leader, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n"
        ::"r"(bar), "r"(leader) : "memory");
}
__device__ __forceinline__ uint32_t elect() {
    uint32_t e;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(e));
    return e;
}

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap *map, int x, int slot,
                                        int head, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                 ::"r"(bar), "r"(bytes) : "memory");
}

// Largest of three; a NaN wins.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 2^x on the FMA pipe: x = n + f with n the nearest integer (by adding and
// taking off 1.5 * 2^23, whose low bits then hold n) and 2^f on [-1/2, 1/2] by
// the cubic of least relative error, 2^-13.7: an eighth of the last place of
// fp16, which the result is rounded to at the least.  Below -125 it stays at
// 2^-125, so it is not for steps with masked scores, which have to give 0.
__device__ __forceinline__ float2 ex2_poly(uint64_t x2) {
    float2 x = both(x2);
    x.x = fmaxf(x.x, -125.f);
    x.y = fmaxf(x.y, -125.f);
    x2 = pair2(x.x, x.y);
    const uint64_t big = pair2(12582912.f, 12582912.f), less = pair2(-12582912.f, -12582912.f);
    const uint64_t r = add2(x2, big);
    const uint64_t f = fma2(add2(r, less), pair2(-1.f, -1.f), x2);
    uint64_t p = fma2(pair2(0.055171669f, 0.055171669f), f, pair2(0.24261113f, 0.24261113f));
    p = fma2(p, f, pair2(0.69326097f, 0.69326097f));
    p = fma2(p, f, pair2(0.99992806f, 0.99992806f));
    const float2 n = both(r), v = both(p);
    return make_float2(
        __uint_as_float(__float_as_uint(v.x) + (__float_as_uint(n.x) << 23)),
        __uint_as_float(__float_as_uint(v.y) + (__float_as_uint(n.y) << 23)));
}

// x / g for x below 2^20: the quotient of x + 1/2 stays 1/(2g) away from the
// integers, further than its rounding.
__device__ __forceinline__ int small_div(int x, float inv_g) {
    return (int)(((float)x + 0.5f) * inv_g);
}

// Barriers of the two warps that share 32 rows, and of a tile's eight warps.
__device__ __forceinline__ void pair_sync(int t, int quad) {
    asm volatile("bar.sync %0, 64;" ::"r"(1 + t * 4 + quad) : "memory");
}
// The same barrier of the two warps, and whether any of their threads says so.
__device__ __forceinline__ bool pair_any(int t, int quad, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %2, 0;\n\t"
        "bar.red.or.pred q, %1, 64, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}\n"
        : "=r"(r) : "r"(1 + t * 4 + quad), "r"((uint32_t)x) : "memory");
    return r;
}
__device__ __forceinline__ void tile_sync(int t) {
    asm volatile("bar.sync %0, 256;" ::"r"(9 + t) : "memory");
}

// Polls before a wait gives up (each may itself wait a while in hardware):
// seconds, far longer than any tile takes.
constexpr uint32_t kPolls = 1u << 19;

// A bounded wait, in as few instructions as a wait that is over already can do
// with: it has no result, and every role goes on step by step either way. One
// that gives up sets `fail` (a word of shared memory), which ends all others at
// once; results are then unusable, and the launch says so.
__device__ __forceinline__ void wait(uint32_t bar, uint32_t parity, uint32_t fail) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .u32 n, f;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1;\n\t"
        "@p bra DONE;\n\t"
        "mov.u32 n, 0;\n\t"
        "POLL:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1;\n\t"
        "@p bra DONE;\n\t"
        "ld.volatile.shared.u32 f, [%2];\n\t"
        "setp.ne.u32 p, f, 0;\n\t"
        "@p bra DONE;\n\t"
        "add.u32 n, n, 1;\n\t"
        "setp.lt.u32 p, n, %3;\n\t"
        "@p bra POLL;\n\t"
        "st.volatile.shared.u32 [%2], 1;\n\t"
        "DONE:\n\t}\n"
        ::"r"(bar), "r"(parity), "r"(fail), "n"(kPolls) : "memory");
    __syncwarp();
}
// The same that ends with `fail` set or not, for copies and products in flight.
__device__ __forceinline__ void wait_over(uint32_t bar, uint32_t parity) {
    umma::mbar_wait(bar, parity, kPolls);
}

__device__ __forceinline__ void tmem_ld_wait() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float *v) {
    uint32_t *r = (uint32_t *)v;
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
          "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
          "r"(r[14]), "r"(r[15])
        : "memory");
}

// Of every 4 pairs of exponentials, those computed by ex2_poly: at D = 64, where
// the products are half as long, one (4096 keys: 742 TFLOP/s against 667 for
// none, at the time); at 128 none (1247 against 1172 for one).
constexpr int poly_pairs(int D) { return D == 64 ? 1 : 0; }

// How far a row outgrows its maximum before that is moved, see attn_lift.  fp16 with
// 4 and a lift of 11 in place of 8 and 7 rounds weights 16 times finer; 4096 causal
// tokens, 32 heads of 64 over 8: 119 us either way with scores of deviation 1, 143
// against 133 with scores of deviation 4, which move it more often.
template <typename T> __device__ constexpr float slack() { return 8.f; }
template <> __device__ constexpr float slack<__half>() { return 4.f; }

// A warp's weights, in tensor memory by now, to the issuing warp.
__device__ __forceinline__ void hand_over(uint32_t ready) {
    umma::fence_before();
    __syncwarp();
    if (threadIdx.x % 32 == 0) arrive(ready);
}

// p = 2^(c s - c m) of a thread's scores of one step into their place,
// handed over by halves, and their sum.
template <typename T, int POLY, int N>
__device__ __forceinline__ void weights(const float (&s)[N], uint64_t c2, uint64_t mc2,
                                        uint64_t &sum, uint32_t st, uint32_t ready) {
#pragma unroll
    for (int x = 0; x < N; x += 32) {
        uint32_t p[16];
#pragma unroll
        for (int y = 0; y < 16; y++) {
            const uint64_t v = fma2(pair2(s[x + 2 * y], s[x + 2 * y + 1]), c2, mc2);
            float2 e;
            if (y % 4 < POLY) {
                e = ex2_poly(v);
            } else {
                e = both(v);
                e.x = ex2(e.x);
                e.y = ex2(e.y);
            }
            sum = add2(sum, pair2(e.x, e.y));
            p[y] = pack2<T>(e.x, e.y);
        }
        tmem_st16(st + x / 2, p);
        tmem_st_wait();
        hand_over(ready + (x ? 8 : 0));
    }
}

}  // namespace

// What a block does at a time: rows row0 .. row0 + 255 of one kv head of one request (or,
// packed, of the batch) against `cnt` key tiles from `first` on.
struct WideTask {
    AttnReq rq;
    int b, kvh, row0, rows, part, parts;
    int first, cnt, cnt0;                   // cnt0: of the first row tile
    int own_seen;                           // own keys in sight of the last row
    int steps;                              // before this one, of all of the block's
    // Which row tile has rows row0 .. row0 + 127.  In runs the two take tasks, of one row
    // tile each, in turn, so that one writes its results while the other is at work.
    int tile;

    __device__ __forceinline__ bool has(int t) const { return t == tile || rows - row0 > kRows; }
    __device__ __forceinline__ int row_of(int t) const { return row0 + (t == tile ? 0 : kRows); }
    __device__ __forceinline__ int cnt_of(int t) const { return !has(t) ? 0 : t == tile ? cnt0 : cnt; }
};

template <typename T, int D, AttnKind KIND> struct WideTasks {
    static constexpr bool PACKED = KIND == kAttnPacked, RUNS = KIND == kAttnTreeRuns;
    static constexpr int KEYS = attn_wide(D);
    const AttnArgs &a;
    int u, hi;                              // RUNS: the run's next unit and its end
    int total;                              // key tiles of all tasks

    __device__ __forceinline__ int pre_tiles() const {
        return ((PACKED || !a.packed ? a.prefix_len : 0) + KEYS - 1) / KEYS;
    }
    // own keys that row r of a request sees
    __device__ __forceinline__ int sees(const AttnReq &rq, int r) const {
        return KIND == kAttnOwn && a.causal
                   ? max(0, min(rq.len, rq.len - rq.n + r / a.by_group + 1))
                   : rq.len;
    }
    __device__ __forceinline__ bool begin(WideTask &k) {
        k.steps = 0;
        k.tile = 0;
        if (RUNS) {
            const AttnRuns runs = attn_runs(a);
            if ((int)blockIdx.x >= runs.blocks) {
                if (threadIdx.x == 0) a.splits[blockIdx.x] = {};
                return false;
            }
            u = runs.begin(blockIdx.x);
            hi = runs.begin(blockIdx.x + 1);
            total = hi - u;
            k.cnt = 0;
            k.tile = 1;
            if (!next(k, true)) return false;
            // The block that is the first to go on with an item tells the join of it.
            if (threadIdx.x == 0) {
                AttnSplit x = {};
                const int from = u - k.cnt - k.first, c0 = k.first ? runs.block_of(from) : 0;
                if (k.first && c0 == (int)blockIdx.x - 1)
                    x = {c0, runs.block_of(from + attn_item(k.rq.n, k.rq.len) - 1),
                         runs.begin(c0) < from, k.rq.t0, k.rows, k.kvh};
                a.splits[blockIdx.x] = x;
            }
            return true;
        }
        k.b = blockIdx.z;
        k.kvh = blockIdx.y;
        k.rq = PACKED ? AttnReq{0, a.tokens, 0} : attn_req(a, blockIdx.z);
        k.rows = k.rq.n * a.group;
        if (!PACKED && k.rows <= a.rows_small) return false;
        const int bx = (int)blockIdx.x / (PACKED ? a.by_prefix_parts : a.by_wide_parts);
        k.part = (int)blockIdx.x - bx * (PACKED ? a.prefix_parts : a.wide_parts);
        const int pairs = (k.rows + 2 * kRows - 1) / (2 * kRows);
        // the rows that see the most keys first
        const int pair = pairs - 1 - bx;
        if (pair < 0) return false;
        k.row0 = pair * 2 * kRows;
        const int all_tiles = pre_tiles() + (PACKED ? 0 : (k.rq.len + KEYS - 1) / KEYS);
        const int each = PACKED ? a.prefix_wide_each : a.wide_each;
        k.parts = max(1, (all_tiles + each - 1) / (PACKED ? a.by_prefix_each : a.by_wide_each));
        if (k.part >= k.parts) return false;
        k.own_seen = PACKED ? 0 : sees(k.rq, min(k.rows, k.row0 + 2 * kRows) - 1);
        const int seen_t0 = PACKED ? 0 : sees(k.rq, min(k.rows, k.row0 + kRows) - 1);
        k.first = k.part * each;
        auto count_of = [&](int seen) {
            return max(0, min(k.first + each, pre_tiles() + (seen + KEYS - 1) / KEYS) - k.first);
        };
        k.cnt0 = count_of(seen_t0), k.cnt = count_of(k.own_seen);
        total = k.cnt;
        return true;
    }
    // The next task of a run.
    __device__ __forceinline__ bool next(WideTask &k, bool first = false) {
        if (!RUNS || u >= hi) return false;
        k.steps += k.cnt;
        const int in = u - attn_units_at(a, u, k.b);
        k.rq = attn_req(a, k.b);
        k.rows = k.rq.n * a.group;
        const int tiles = attn_item(k.rq.n, k.rq.len);
        k.kvh = in / tiles;
        k.first = in - k.kvh * tiles;
        k.row0 = 0;
        k.cnt = k.cnt0 = min(tiles - k.first, hi - u);
        k.parts = k.cnt == tiles ? 1 : 2;    // one: all of the item
        k.part = first ? 0 : 1;
        k.own_seen = k.rq.len;
        k.tile ^= 1;
        u += k.cnt;
        return true;
    }
};

// kAttnPacked: rows are those of all the batch's tokens, keys the shared prefix.
template <typename T, int D, AttnKind KIND>
__device__ __forceinline__ void attn_wide_rows(const AttnArgs &a, const CUtensorMap &kmap,
                                               const CUtensorMap &vmap, uint8_t *basep) {
    using L = Lay<D>;
    constexpr bool PACKED = KIND == kAttnPacked, RUNS = KIND == kAttnTreeRuns;
    constexpr bool TREE = KIND == kAttnTree || RUNS;
    constexpr int NS = L::stages, KEYS = L::keys, THREADS = threads_of(KIND);
    WideTasks<T, D, KIND> tasks{a};
    WideTask task;
    if (!tasks.begin(task)) return;
    const int n_pre = !RUNS && (PACKED || !a.packed) ? a.prefix_len : 0;
    const int pre_tiles = (n_pre + KEYS - 1) / KEYS;

    const uint32_t base = smem_u32(basep);
    const uint32_t bars = base + L::bars;
    const uint32_t kv_full = bars + L::kv_full, kv_empty = bars + L::kv_empty,
                   q_full = bars + L::q_full, s_full = bars + L::s_full,
                   p_full = bars + L::p_full, o_end = bars + L::o_end, drain = bars + L::drain,
                   tmem_slot = bars + L::tmem;
    const uint32_t fail = bars + L::fail;
    volatile int *const failed = (volatile int *)(basep + L::bars + L::fail);
    volatile int *const dirty = (volatile int *)(basep + L::bars + L::dirty);
    // the warp's number from one lane, so that it counts as uniform
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;

    // The rows' warps: row tile, half of the keys, quarter of the rows, row.
    const int t = warp / 8, h = warp / 4 % 2, quad = warp % 4, r = threadIdx.x % kRows;
    const int tid = threadIdx.x % (2 * kRows);          // in the tile
    const float inv_group = 1.f / (float)a.group;
    // Q is asked for first of all, a row by D / 8 neighbouring threads.
    constexpr int CH = D / 8, RP = 2 * kRows / CH, N = kRows / RP;
    uint4 qv[N];
    auto ask_q = [&](const WideTask &k) {
        if (!k.has(t)) return;
        // row0 + x is token tok0 + (rem0 + x) / group
        const int row0 = k.row_of(t), tok0 = row0 / a.by_group, rem0 = row0 - tok0 * a.group;
        const T *q = (const T *)a.q + (int64_t)(k.rq.t0 + tok0) * a.q_token +
                     (int64_t)k.kvh * a.group * a.q_head + (tid % CH) * 8;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int x = i * RP + tid / CH;
            const int y = rem0 + x, tok = small_div(y, inv_group);
            qv[i] = make_uint4(0, 0, 0, 0);
            if (row0 + x < k.rows)
                qv[i] = *(const uint4 *)(q + tok * a.q_token + (y - tok * a.group) * a.q_head);
        }
    };
    if (!RUNS) ask_q(task);

    // The loading warp makes the barriers and goes on at once; the others meet
    // behind it.
    if (warp == 17) {
        if (lane == 0) {
            for (int i = 0; i < NS; i++) {
                umma::mbar_init(kv_full + 8 * i, 1);
                umma::mbar_init(kv_empty + 8 * i, 1);
            }
            for (int x = 0; x < 2; x++) {
                umma::mbar_init(q_full + 8 * x, 2 * kRows);
                umma::mbar_init(s_full + 8 * x, 1);
                umma::mbar_init(p_full + 16 * x, 8);
                umma::mbar_init(p_full + 16 * x + 8, 8);
                umma::mbar_init(o_end + 8 * x, 1);
            }
            umma::mbar_init(drain, 1);
            *failed = 0;
            for (int i = 0; i < 4; i++) dirty[i] = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        asm volatile("bar.arrive 11, %0;" ::"n"(THREADS) : "memory");
    } else {
        if (warp == 16) umma::tmem_alloc(tmem_slot, 512);
        umma::fence_before();
        asm volatile("bar.sync 11, %0;" ::"n"(THREADS) : "memory");
        umma::fence_after();
    }
    const uint32_t tmem = warp >= 17 ? 0 : *(volatile uint32_t *)(basep + L::bars + L::tmem);

    if (RUNS) {
        if (warp >= 16)
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        else
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegs));
    }
    if (warp == 19) {
        // one more only because registers change hands by four warps
    } else if (warp >= 17) {
        // ---- keys (warp 17) and values (18): K of tile j in ring tile 2j, V in 2j + 1 --
        const int w = warp - 17;
        const CUtensorMap *const map = w ? &vmap : &kmap;
        // a box is a page, or a tile's part of one
        const int box_shift = min(7, a.page_shift), box = 1 << box_shift;
        const int bi = lane & ((KEYS >> box_shift) - 1);        // this lane's box
        const int bh = lane >> (7 - box_shift);                 // and column half
        int issued = 0;
        do {
            const int32_t *own_pages = PACKED ? nullptr : a.pages + (int64_t)task.b * a.pages_row;
            auto page_of = [&](int j, int &key, bool &want) {
                const bool pre = task.first + j < pre_tiles;
                key = (task.first + j - (pre ? 0 : pre_tiles)) * KEYS + (bi << box_shift);
                want = j < task.cnt && bh < D / 64 && key < (pre ? n_pre : task.own_seen);
                return want ? attn_page(a, pre ? a.prefix_pages : own_pages, key) : 0;
            };
            int key, next_key;
            bool want, next_want;
            int page = page_of(0, key, want);
            // A further task's queries, which its rows' warps will ask for when they are
            // done with the last one's results, are on their way into L2 by then.
            if (RUNS && task.steps)
                for (int x = lane; x < task.rows; x += 32) {
                    const int tok = x / a.by_group;
                    prefetch_l2_bulk((const T *)a.q + (int64_t)(task.rq.t0 + tok) * a.q_token +
                                         ((int64_t)task.kvh * a.group + x - tok * a.group) * a.q_head,
                                     D * 2);
                }
            for (int j = 0; j < task.cnt; j++) {
                if (__any_sync(~0u, *failed)) break;
                const int next_page = page_of(j + 1, next_key, next_want);
                const uint32_t bytes = __popc(__ballot_sync(~0u, want)) * box * 128;
                const int i = 2 * issued + w, st = i % NS;
                if (i >= NS) wait(kv_empty + 8 * st, (i / NS - 1) & 1, fail);
                if (__any_sync(~0u, *failed)) break;
                if (lane == 0) arrive_tx(kv_full + 8 * st, bytes);
                __syncwarp();
                if (want)
                    tma_box(base + L::ring + st * L::kv_tile + bh * L::kv_half + bi * box * 128, map,
                            bh * 64, key & ((1 << a.page_shift) - 1), task.kvh, page,
                            kv_full + 8 * st);
                issued++;
                page = next_page;
                key = next_key;
                want = next_want;
            }
        } while (RUNS && !*failed && tasks.next(task));
        if (*failed)                        // let the copies in flight land
            for (int j = max(0, issued - NS); j < issued; j++)
                wait_over(kv_full + 8 * ((2 * j + w) % NS), ((2 * j + w) / NS) & 1);
    } else if (warp == 16) {
        // ---- the products ------------------------------------------------------------
        if (tasks.total > 0) {
            const uint32_t leader = elect();
            // descriptors of tile 0 and ring tile 0; the address field counts 16 bytes
            const uint64_t q_desc = desc128(base, 16, 1024),
                           k_desc = desc128(base + L::ring, 16, 1024),
                           v_desc = desc128(base + L::ring, L::kv_half, 1024);
            auto qk = [&](int t, int st) {
                const uint64_t q = q_desc + t * (L::q_tile >> 4),
                               k = k_desc + st * (L::kv_tile >> 4);
#pragma unroll
                for (int x = 0; x < D / 16; x++)
                    mma_ss(leader, tmem + L::s(t), q + (((x / 4) * L::q_half + (x % 4) * 32) >> 4),
                           k + (((x / 4) * L::kv_half + (x % 4) * 32) >> 4), idesc<T>(KEYS, false),
                           x > 0);
                commit(leader, s_full + 8 * t);
            };
            // The weights of each half of the keys lie where its scores did, and come
            // in two parts: part w is keys w * cols/2 on of both halves.
            auto pv = [&](int t, int st, int w, bool acc) {
                const uint64_t v = v_desc + st * (L::kv_tile >> 4);
                constexpr int H = L::cols / 16, Q = H / 2;
#pragma unroll
                for (int i = 0; i < H; i++) {
                    const int x = i / Q * H + w * Q + i % Q;
                    mma_ts(leader, tmem + L::o(t), tmem + L::s(t) + x / H * L::cols + x % H * 8,
                           v + x * (2048 >> 4), idesc<T>(D, true), acc || i > 0);
                }
            };
            int used[2] = {0, 0};           // tasks of each row tile so far, and their steps
            int past[2] = {0, 0};
            do {
                const int cnt = task.cnt, cnt0 = task.cnt_of(0), cnt1 = task.cnt_of(1);
                const int n0 = 2 * task.steps, all = 2 * tasks.total;  // ring tiles before, in all
                if (task.has(0)) wait(q_full, used[0]++ & 1, fail);
                if (task.has(1)) wait(q_full + 8, used[1]++ & 1, fail);
                const int s0 = n0 % NS;
                wait(kv_full + 8 * s0, (n0 / NS) & 1, fail);
                umma::fence_after();
                if (cnt0 > 0) qk(0, s0);
                if (cnt1 > 0) qk(1, s0);
                if (n0 + NS < all) commit(leader, kv_empty + 8 * s0);
                // ring tiles of V j and K j + 1, their parities
                int sv = (n0 + 1) % NS, sk = (n0 + 2) % NS;
                int fv = (n0 + 1) / NS & 1, fk = (n0 + 2) / NS & 1;
                for (int j = 0; j < cnt; j++) {
                    if (__any_sync(~0u, *failed)) break;
                    wait(kv_full + 8 * sv, fv, fail);
                    if (j + 1 < cnt) wait(kv_full + 8 * sk, fk, fail);
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const int mine = t == 0 ? cnt0 : cnt1;
                        if (j >= mine) continue;
                        const int turn = (past[t] + j) & 1;
                        wait(p_full + 16 * t, turn, fail);
                        umma::fence_after();
                        pv(t, sv, 0, j > 0);
                        wait(p_full + 16 * t + 8, turn, fail);
                        umma::fence_after();
                        pv(t, sv, 1, true);
                        // in order behind it: the next scores take the weights' place
                        if (j + 1 < mine) qk(t, sk);
                        else commit(leader, o_end + 8 * t);
                    }
                    // only what the loader will wait for
                    if (n0 + 2 * j + 1 + NS < all) commit(leader, kv_empty + 8 * sv);
                    if (j + 1 < cnt && n0 + 2 * j + 2 + NS < all) commit(leader, kv_empty + 8 * sk);
                    sv += 2, sk += 2;
                    if (sv >= NS) sv -= NS, fv ^= 1;
                    if (sk >= NS) sk -= NS, fk ^= 1;
                }
                past[0] += cnt0;
                past[1] += cnt1;
            } while (RUNS && !__any_sync(~0u, *failed) && tasks.next(task));
            if (*failed) {                  // let the products in flight end
                commit(leader, drain);
                wait_over(drain, 0);
            }
        }
    } else {
        // ---- the rows ----------------------------------------------------------------
        int turn = 0;                       // parities: 1 of this row tile's steps, 2 of its tasks
        // What a task has to say after its steps is kept in shared memory in between, where the
        // registers are needed.
        volatile int *const note = (volatile int *)(basep + L::bars + L::note) + t * L::notes;
        enum { kT0, kN, kLen, kB, kHead, kRow0, kRowsOf, kPart, kParts, kFirst, kCnt, kSteps, kU, kHi,
               kDone, kTile, kMask, kNotes };
        static_assert(kNotes <= L::notes, "place for the notes");
        auto kept = [&](int i, int v) { return RUNS ? note[i] : v; };
        int done = 0;
        while (true) {
            if (RUNS && tid == 0) {
                note[kT0] = task.rq.t0, note[kN] = task.rq.n, note[kLen] = task.rq.len;
                note[kB] = task.b, note[kHead] = task.kvh, note[kRow0] = task.row_of(t);
                note[kRowsOf] = task.rows, note[kPart] = task.part, note[kParts] = task.parts;
                note[kFirst] = task.first, note[kCnt] = task.cnt, note[kSteps] = task.steps;
                note[kU] = tasks.u, note[kHi] = tasks.hi, note[kDone] = done;
                note[kTile] = task.tile;
                note[kMask] = max(task.rq.len - task.rq.n, 0) / KEYS - task.first;
            }
            if (RUNS) tile_sync(t);
            const bool live = task.has(t);
            const int mine = task.cnt_of(t);
            if (RUNS) ask_q(task);
            if (live) {
                // into its swizzled place
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int qr = i * RP + tid / CH, c = tid % CH;
                    *(uint4 *)(basep + t * L::q_tile + (c / 8) * L::q_half + qr * 128 +
                               (((c % 8) ^ (qr & 7)) << 4)) = qv[i];
                }
                umma::fence_smem_async();
                arrive(q_full + 8 * t);
            }
            const uint32_t lanes = (uint32_t)quad * 32 << 16;
            // this thread's half of the scores and of the weights
            const uint32_t ot = tmem + L::o(t) + lanes, st = tmem + L::s(t) + h * L::cols + lanes;
            float *const swap = (float *)(basep + L::swap) + t * 2 * kRows;
            const bool warp_live = task.row_of(t) + quad * 32 < task.rows;
            const float c = a.scale_log2;
            // what p is measured from, in the log2 domain
            auto lowered = [&](float m) { return __fmaf_rn(m, c, -attn_lift<T>(slack<T>())); };
            float m = -INFINITY;
            float2 l = make_float2(0.f, 0.f);    // two halves of the sum
            // Steps that are not full, and those with keys that only some rows see: what
            // lies behind the keys may be anything, and a weight of zero does not hide a
            // NaN.  They are the last ones, and the prefix's last.
            const bool some = TREE || (KIND == kAttnOwn && a.causal);
            int masked_from = 0, masked_pre = n_pre % KEYS ? pre_tiles - 1 - task.first : -1;
            int see = 0, see_first = 0;     // own keys in sight of this row, and of the first
            if (!RUNS) {
                const AttnReq &rq = task.rq;
                const int row = task.row_of(t) + r;
                if (!PACKED) see = row < task.rows ? tasks.sees(rq, row) : 0;
                see_first = TREE ? rq.len - rq.n
                            : some ? rq.len - rq.n + task.row0 / a.by_group + 1 : rq.len;
                const int whole = min(some ? max(see_first, 0) : task.own_seen, task.own_seen) / KEYS;
                masked_from = pre_tiles + whole - task.first;
            }
            // the nodes that this row's sees, where it is one of a tree's
            auto sight_of = [&] {
                const int row = kept(kRow0, task.row_of(t)) + r;
                return a.seen + (int64_t)(kept(kT0, task.rq.t0) +
                                          min(row, kept(kRowsOf, task.rows) - 1) / a.by_group) *
                                    a.seen_words;
            };
            for (int j = 0; j < mine; j++) {
                const bool masked =
                    RUNS ? j >= note[kMask] : j >= masked_from || j == masked_pre;
                int lim = 0;                    // keys of the step that this row sees
                uint64_t bits = 0;              // and of this thread's half, one a bit
                if (__builtin_expect(masked, 0)) {
                    const int first = kept(kFirst, task.first);
                    const int own_seen = RUNS ? note[kLen] : task.own_seen;
                    if (RUNS) see_first = note[kLen] - note[kN];
                    const bool pre = first + j < pre_tiles;
                    const int k0 = (first + j - (pre ? 0 : pre_tiles)) * KEYS;
                    const int held = (pre ? n_pre : own_seen) - k0;
                    lim = pre ? held : min(held, see - k0);
                    if (TREE) {
                        bits = low_bits(held - h * L::cols);
                        if (!pre)
                            bits &= tree_sight(sight_of(), a.seen_words,
                                               k0 + h * L::cols - see_first);
                    }
                    // A task's warps may be here long before its turn in the ring, whose
                    // barriers say nothing of uses that far ahead: its scores do.
                    if (RUNS) wait(s_full + 8 * t, (turn + j) & 1, fail);
                    const int n = 2 * (kept(kSteps, task.steps) + j) + 1;   // the n-th tile in the ring
                    wait(kv_full + 8 * (n % NS), (n / NS) & 1, fail);
                    // two threads a key
                    const int key = r, x0 = r < KEYS ? h * D : 0, x1 = r < KEYS ? x0 + D : 0;
                    uint8_t *v = basep + L::ring + (n % NS) * L::kv_tile + key * 128;
                    auto at = [&](int x) { return v + (x / 128) * L::kv_half + x % 128; };
                    if (key >= held) {
                        for (int x = x0; x < x1; x += 16) *(uint4 *)at(x) = make_uint4(0, 0, 0, 0);
                    } else if (some && !pre && k0 + key >= see_first) {
                        constexpr uint32_t E = fmt16<T>() ? 0x7f80u : 0x7c00u;
                        bool bad = false;
                        for (int x = x0; x < x1; x += 16) {
                            const uint4 q = *(const uint4 *)at(x);
                            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                            for (int y = 0; y < 4; y++)
                                bad |= (w[y] & E) == E || (w[y] >> 16 & E) == E;
                        }
                        if (bad) {
                            const int d = kept(kDone, 0);
                            dirty[d & 3] = d + 1;
                            __threadfence_block();
                            for (int x = x0; x < x1; x += 4) {
                                uint32_t *q = (uint32_t *)at(x), w = *q;
                                if ((w & E) == E) w &= 0xffff0000u;
                                if ((w >> 16 & E) == E) w &= 0xffffu;
                                *q = w;
                            }
                        }
                    }
                    umma::fence_smem_async();
                }
                wait(s_full + 8 * t, (turn + j) & 1, fail);
                umma::fence_after();
                if (warp_live) {
                    float s[L::cols];
#pragma unroll
                    for (int x = 0; x < L::cols; x += 32) tmem_ld32(st + x, s + x);
                    tmem_ld_wait();
                    if (__builtin_expect(masked, 0)) {
                        lim -= h * L::cols;
#pragma unroll
                        for (int x = 0; x < L::cols; x++)
                            s[x] = (TREE ? (bool)(bits >> x & 1) : x < lim) ? s[x] : -INFINITY;
                    }
                    float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int x = 4; x + 8 <= L::cols; x += 8)
#pragma unroll
                        for (int y = 0; y < 4; y++) mx[y] = max3(mx[y], s[x + y], s[x + y + 4]);
                    mx[0] = max3(mx[0], s[L::cols - 4], s[L::cols - 3]);
                    mx[1] = max3(mx[1], s[L::cols - 2], s[L::cols - 1]);
                    float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
                    // the halves' maxima are exchanged only if one outgrows the old one
                    if (__builtin_expect(pair_any(t, quad, !((top - m) * c <= slack<T>())), 0)) {
                        swap[h * kRows + r] = top;
                        pair_sync(t, quad);
                        top = max3(top, swap[(h ^ 1) * kRows + r], top);
                        const bool grow = !((top - m) * c <= slack<T>());
                        const float to = grow ? top : m;
                        const float w = !grow || to == -INFINITY ? 1.f : ex2(m * c - to * c);
                        if (j > 0) {
#pragma unroll 1
                            for (int x = h * (D / 2); x < (h + 1) * (D / 2); x += 16) {
                                float o[16];
                                umma::tmem_ld16(ot + x, o);
                                uint32_t u[16];
#pragma unroll
                                for (int y = 0; y < 16; y++) u[y] = __float_as_uint(o[y] * w);
                                tmem_st16(ot + x, u);
                            }
                        }
                        l.x *= w;
                        l.y *= w;
                        m = to;
                    }
                    // a row with an infinite or NaN score is NaN altogether
                    const float mc = m == -INFINITY ? 0.f : m < INFINITY ? lowered(m) : NAN;
                    const uint64_t c2 = pair2(c, c), mc2 = pair2(-mc, -mc);
                    uint64_t l2 = pair2(l.x, l.y);
                    if (__builtin_expect(masked, 0)) weights<T, 0>(s, c2, mc2, l2, st, p_full + 16 * t);
                    else weights<T, poly_pairs(D)>(s, c2, mc2, l2, st, p_full + 16 * t);
                    l = both(l2);
                } else {
                    hand_over(p_full + 16 * t);
                    hand_over(p_full + 16 * t + 8);
                }
            }
            if (mine > 0) wait(o_end + 8 * t, turn >> 1, fail);
            if (RUNS && mine > 0) turn ^= 2 | (mine & 1);
            umma::fence_after();
            if (live) {
                const int t0 = kept(kT0, task.rq.t0), row0 = kept(kRow0, task.row_of(t)),
                          rows = kept(kRowsOf, task.rows), kvh = kept(kHead, task.kvh),
                          part = kept(kPart, task.part), first = kept(kFirst, task.first);
                const int row = row0 + r;
                const int tok0 = row0 / a.by_group, rem0 = row0 - tok0 * a.group;
                if (RUNS) {
                    done = note[kDone];
                    see = note[kLen];
                    see_first = see - note[kN];
                }
                // The results go through the tile's place of Q, which is done with, so
                // that rows are written by neighbouring threads.
                const bool direct = !PACKED && !a.packed && kept(kParts, task.parts) == 1;
                const int y = rem0 + r, tok = small_div(y, inv_group);
                const int64_t part_row =
                    RUNS ? ((int64_t)blockIdx.x * 2 + part) * kAttnRunRows
                         : (int64_t)(PACKED ? part : a.prefix_parts + part) * a.tokens * a.q_heads;
                const int64_t out_row = (int64_t)(t0 + tok0) * a.q_heads + kvh * a.group;
                __threadfence_block();
                const bool mend = dirty[done & 3] == done + 1 && some;
                uint8_t *const stage = basep + t * L::q_tile;
                tile_sync(t);                   // the last maxima are read
                swap[h * kRows + r] = l.x + l.y;
                tile_sync(t);
                // (a row without a finite score has what ex2_poly makes of -inf: nothing)
                const float sum = m == -INFINITY ? 0.f : swap[r] + swap[kRows + r];
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                // columns at a time, half of them by each of a row's threads: all of 16
                // bits, or half of 32
                const int wide = direct ? D : D / 2;
                for (int x0 = 0; x0 < D; x0 += wide) {
#pragma unroll 1
                    for (int x = x0 + h * (wide / 2); x < x0 + (h + 1) * (wide / 2); x += 16) {
                        __syncwarp();
                        float o[16];
                        if (mine > 0 && warp_live) {
                            umma::tmem_ld16(ot + x, o);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] = 0.f;
                        }
                        if (mend && row < rows) {
                            // what was wiped and is in sight of this row
                            const int end = min(see, max(0, first + kept(kCnt, task.cnt) - pre_tiles) * KEYS);
                            for (int k = max(max(see_first, 0), (first - pre_tiles) * KEYS); k < end;
                                 k++) {
                                if (TREE &&
                                        !(tree_sight(sight_of(), a.seen_words, k - see_first) & 1))
                                        continue;
                                const int page =
                                    attn_page(a, a.pages + (int64_t)kept(kB, task.b) * a.pages_row, k);
                                const T *v = (const T *)a.vp + (int64_t)page * a.v_page +
                                             (int64_t)(k & ((1 << a.page_shift) - 1)) * a.v_slot +
                                             (int64_t)kvh * a.v_head + x;
#pragma unroll
                                for (int i = 0; i < 16; i++) {
                                    const float f = AttnType<T>::up(v[i]);
                                    if (!isfinite(f)) o[i] += f;
                                }
                            }
                        }
                        // 16-byte pieces, their places in the row turned by the row
                        uint8_t *const at = stage + r * (D * 2);
                        constexpr int turn = D / 8 - 1;
                        if (direct) {
#pragma unroll
                            for (int i = 0; i < 16; i += 8)
                                *(uint4 *)(at + ((((x + i) / 8) ^ (r & turn)) << 4)) =
                                    make_uint4(pack2<T>(o[i] * inv, o[i + 1] * inv),
                                               pack2<T>(o[i + 2] * inv, o[i + 3] * inv),
                                               pack2<T>(o[i + 4] * inv, o[i + 5] * inv),
                                               pack2<T>(o[i + 6] * inv, o[i + 7] * inv));
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; i += 4)
                                *(float4 *)(at + ((((x - x0 + i) / 4) ^ (r & turn)) << 4)) =
                                    make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        }
                    }
                    tile_sync(t);
                    // CH pieces a row, either way
#pragma unroll 4
                    for (int i = 0; i < CH / 2; i++) {
                        const int or_ = i * (2 * kRows / CH) + tid / CH, c = tid % CH,
                                  yy = rem0 + or_;
                        if (row0 + or_ >= rows) break;
                        const int tk = small_div(yy, inv_group);
                        const int64_t o_row = out_row + (int64_t)tk * a.q_heads + (yy - tk * a.group);
                        const uint4 v =
                            *(const uint4 *)(stage + or_ * (D * 2) + ((c ^ (or_ & (CH - 1))) << 4));
                        if (direct) *(uint4 *)((T *)a.out + o_row * D + c * 8) = v;
                        else *(uint4 *)(a.part_o + (part_row + (RUNS ? or_ : o_row)) * D + x0 + c * 4) = v;
                    }
                    tile_sync(t);
                }
                if (!direct && h == 0 && row < rows)
                    a.part_ml[part_row +
                              (RUNS ? r : out_row + (int64_t)tok * a.q_heads + (y - tok * a.group))] =
                        make_float2(lowered(m), sum);
            }
            if (!RUNS) break;
            tasks.u = note[kU], tasks.hi = note[kHi];
            task.steps = note[kSteps], task.cnt = note[kCnt], task.tile = note[kTile];
            done = note[kDone] + 1;
            tile_sync(t);                   // the notes are read
            if (!tasks.next(task)) break;
        }
    }
    umma::fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *failed) atomicOr(a.err, kAttnTimeout);
    if (warp == 16) {
        umma::fence_after();
        umma::tmem_free(tmem, 512);
    }
}

// See attn_rows_kernel.
template <typename T, int D, AttnKind KIND>
__global__ void __launch_bounds__(threads_of(KIND), 1)
attn_umma_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap) {
    extern __shared__ __align__(1024) uint8_t shared[];
    if (a.more) pdl_trigger();
    attn_wide_rows<T, D, KIND>(a, kmap, vmap, shared);
    attn_wait_last();
}

// How a kernel of one kind is started, whatever its type and head_dim.
struct WideLaunch {
    const AttnArgs &a;
    const CUtensorMap &km, &vm;
    dim3 grid;
    bool first;
    cudaStream_t st;

    template <typename T, int D, AttnKind KIND> int go() const {
        static std::atomic<uint64_t> done;
        cudaError_t e = cudaSuccess;
        if (KIND == kAttnTreeRuns && !done.load()) {
            // fewer registers at the start than change hands, and a warp would wait for good
            cudaFuncAttributes at;
            e = cudaFuncGetAttributes(&at, attn_umma_kernel<T, D, KIND>);
            if (e != cudaSuccess) return cuda_fail(e, "attention kernel attributes");
            if (at.numRegs * threads_of(KIND) < 512 * kRowRegs + 128 * kOtherRegs) {
                set_error("attn_umma_kernel: built with %d registers", at.numRegs);
                return WARP_E_CUDA;
            }
        }
        e = attn_smem(attn_umma_kernel<T, D, KIND>, Lay<D>::bytes, done);
        if (e != cudaSuccess) return cuda_fail(e, "attention smem attribute");
        e = attn_start(attn_umma_kernel<T, D, KIND>, grid, threads_of(KIND), Lay<D>::bytes, st, first,
                       a, km, vm);
        if (e != cudaSuccess) return cuda_fail(e, "attn_umma_kernel");
        count_launch();
        return WARP_OK;
    }
    template <AttnKind KIND> int typed(const warp_kv_pages *c) const {
        const bool d64 = c->head_dim == 64;
        if (c->type == WARP_T_F16)
            return d64 ? go<__half, 64, KIND>() : go<__half, 128, KIND>();
        return d64 ? go<__nv_bfloat16, 64, KIND>() : go<__nv_bfloat16, 128, KIND>();
    }
};

// The kinds of trees, which are compiled apart (attn_umma_tree.cu).
int attn_umma_tree(const WideLaunch &l, const warp_kv_pages *c, AttnKind kind);

}  // namespace warp
