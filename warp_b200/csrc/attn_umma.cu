// attn_umma.cu — attention over paged keys and values for many query rows a
// key head: prompts, chunks and the rows of a batch behind a shared prefix.
//
// A CTA holds 256 rows (token, head of the group) of one kv head as two tiles
// of 128 and walks the keys in tiles of 128. Per tile, on the tensor cores
// with the accumulators in tensor memory:
//     S = Q K^T      (both from shared memory, 128B-swizzled, K-major)
//     O += P V       (P from tensor memory, V as it lies: N-major)
// and between them, one thread a row: the running maximum m, p = 2^(c s - c m)
// and the sum l. P takes the place of S. While one tile's exponentials are
// computed the other's products run, so neither pipe waits for the other.
//
// The maximum that p is measured from moves only when a row outgrows it by
// 2^8, so the accumulated O is rescaled rarely; p then stays below 2^8, which
// both 16-bit types hold, and the result is the same as O and l carry the same
// factor.
//
// What bounds it: per pair of 128 x 128 tiles the products take
// 2 * 2 * 128 * 128 * D / 8192 FMA a clock = 1024 cycles at D = 128, and
// 2 * 128 * 128 exponentials at 16 a clock 2048. So a share of them is
// computed on the FMA pipe instead (ex2_poly).
//
// Warps: 0-3 rows of tile 0, 4-7 rows of tile 1, 8 issues the products, 9
// loads keys and values by TMA, a box a page, into a ring of tiles.
#include "attn.cuh"
#include "umma.cuh"

#include <cuda.h>

namespace warp {
namespace {

constexpr int kRows = 128;                  // rows a tile
constexpr int kKeys = kAttnWide;            // keys a tile
constexpr int kThreads = 320;

template <int D> struct Lay {
    static constexpr int q_tile = kRows * D * 2;
    static constexpr int kv_tile = kKeys * D * 2;
    static constexpr int half = kKeys * 128;            // 64 columns of a tile
    static constexpr int stages = D == 128 ? 5 : 8;
    static constexpr int ring = 2 * q_tile;
    static constexpr int bars = ring + stages * kv_tile;
    static constexpr int bytes = bars + 256 + 1024;     // 1024: alignment of the base
    // tensor memory columns
    static constexpr int s(int t) { return t * 128; }
    static constexpr int o(int t) { return 256 + t * D; }
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

// A from tensor memory.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id,
                                       bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
        ::"r"(d), "r"(a), "l"(b), "r"(id), "r"((uint32_t)accumulate)
        : "memory");
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

// A bounded wait.  Once one has given up, `fail` ends all others at once.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int *fail) {
    for (int i = 0; i < 1 << 10; i++) {
        if (umma::mbar_wait(bar, parity, umma::kWaitLimit >> 10)) return true;
        if (*fail) return false;
    }
    *fail = 1;
    return false;
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
__device__ __forceinline__ void tmem_ld_wait() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
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

}  // namespace

// PACKED: rows are those of all the batch's tokens, keys the shared prefix.
template <typename T, int D, bool PACKED>
__global__ void __launch_bounds__(kThreads, 1)
attn_umma_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap) {
    using L = Lay<D>;
    constexpr int NS = L::stages;
    extern __shared__ uint8_t smem_raw[];
    const int kvh = blockIdx.y;
    const AttnReq rq = PACKED ? AttnReq{0, a.tokens, 0} : attn_req(a, blockIdx.z);
    const int rows = rq.n * a.group;
    if (!PACKED && rows <= a.rows_small) return;
    const int parts_max = PACKED ? a.prefix_parts : a.wide_parts;
    const int part = blockIdx.x % parts_max;
    const int pairs = (rows + 2 * kRows - 1) / (2 * kRows);
    // the rows that see the most keys first
    const int pair = pairs - 1 - (int)(blockIdx.x / parts_max);
    if (pair < 0) return;
    const int row0 = pair * 2 * kRows;

    const int n_pre = PACKED || !a.packed ? a.prefix_len : 0;
    const int pre_tiles = (n_pre + kKeys - 1) / kKeys;
    const int all_tiles = pre_tiles + (PACKED ? 0 : (rq.len + kKeys - 1) / kKeys);
    const int each = PACKED ? a.prefix_wide_each : a.wide_each;
    const int parts = max(1, attn_parts(all_tiles, each));
    if (part >= parts) return;
    // own keys that row r sees
    const bool causal = !PACKED && a.causal;
    auto sees = [&](int r) {
        return causal ? max(0, min(rq.len, rq.len - rq.n + r / a.group + 1)) : rq.len;
    };
    const int tiles_rows = rows - row0 > kRows ? 2 : 1;
    // keys in sight of each tile's last row, and the key tiles that hold them
    const int own_seen = PACKED ? 0 : sees(min(rows, row0 + 2 * kRows) - 1);
    const int seen_t0 = PACKED ? 0 : sees(min(rows, row0 + kRows) - 1);
    const int first = part * each;
    auto count_of = [&](int seen) {
        return max(0, min(first + each, pre_tiles + (seen + kKeys - 1) / kKeys) - first);
    };
    const int cnt0 = count_of(seen_t0), cnt = count_of(own_seen);
    const int see_first = PACKED ? 0 : causal ? rq.len - rq.n + row0 / a.group + 1 : rq.len;

    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *const basep = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + L::bars;
    const uint32_t kv_full = bars, kv_empty = bars + NS * 8, q_full = kv_empty + NS * 8,
                   s_full = q_full + 16, p_full = s_full + 16, o_done = p_full + 16,
                   drain = o_done + 16, tmem_slot = drain + 8;
    volatile int *const fail = (volatile int *)(basep + L::bars + (tmem_slot - bars) + 4);
    volatile int *const dirty = fail + 1;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; i++) {
            umma::mbar_init(kv_full + 8 * i, 1);
            umma::mbar_init(kv_empty + 8 * i, 1);
        }
        for (int t = 0; t < 2; t++) {
            umma::mbar_init(q_full + 8 * t, kRows);
            umma::mbar_init(s_full + 8 * t, 1);
            umma::mbar_init(p_full + 8 * t, kRows);
            umma::mbar_init(o_done + 8 * t, 1);
        }
        umma::mbar_init(drain, 1);
        *fail = 0;
        *dirty = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) umma::tmem_alloc(tmem_slot, 512);
    umma::fence_before();
    __syncthreads();
    umma::fence_after();
    const uint32_t tmem = *(volatile uint32_t *)(basep + (tmem_slot - base));

    if (warp == 9) {
        // ---- keys and values: K of tile j in ring tile 2j, V in 2j + 1 --------------
        const int32_t *own_pages = PACKED ? nullptr : a.pages + (int64_t)blockIdx.z * a.pages_row;
        const int box = min(kKeys, 1 << a.page_shift);  // keys a box
        const int boxes = kKeys / box;
        const int bi = lane % boxes, bh = lane / boxes;  // this lane's box and column half
        auto page_of = [&](int j, int &key, bool &want) {
            const bool pre = first + j < pre_tiles;
            key = (first + j - (pre ? 0 : pre_tiles)) * kKeys + bi * box;
            want = j < cnt && bh < D / 64 && key < (pre ? n_pre : own_seen);
            return want ? attn_page(a, pre ? a.prefix_pages : own_pages, key) : 0;
        };
        int key, next_key;
        bool want, next_want;
        int page = page_of(0, key, want), issued = 0;
        bool ok = true;
        for (int j = 0; j < cnt && ok; j++) {
            const int next_page = page_of(j + 1, next_key, next_want);
            const uint32_t bytes = __popc(__ballot_sync(~0u, want)) * box * 128;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const int i = 2 * j + w, st = i % NS;
                if (i >= NS && !wait(kv_empty + 8 * st, (i / NS - 1) & 1, fail)) ok = false;
                ok = __all_sync(~0u, ok);
                if (!ok) break;
                if (lane == 0) arrive_tx(kv_full + 8 * st, bytes);
                __syncwarp();
                if (want)
                    tma_box(base + L::ring + st * L::kv_tile + bh * L::half + bi * box * 128,
                            w ? &vmap : &kmap, bh * 64, key & ((1 << a.page_shift) - 1), kvh, page,
                            kv_full + 8 * st);
                issued++;
            }
            page = next_page;
            key = next_key;
            want = next_want;
        }
        if (!ok)                            // let the copies in flight land
            for (int i = max(0, issued - NS); i < issued; i++)
                umma::mbar_wait(kv_full + 8 * (i % NS), (i / NS) & 1, umma::kWaitLimit);
    } else if (warp == 8) {
        // ---- the products, issued by one thread ------------------------------------
        if (lane == 0 && cnt > 0) {
            auto qk = [&](int t, int st) {
                const uint32_t q = base + t * L::q_tile, k = base + L::ring + st * L::kv_tile;
#pragma unroll
                for (int x = 0; x < D / 16; x++) {
                    const uint32_t off = (x / 4) * L::half + (x % 4) * 32;
                    umma::mma_f16(tmem + L::s(t), desc128(q + off, 16, 1024),
                                  desc128(k + off, 16, 1024), idesc<T>(kKeys, false), x > 0);
                }
                umma::commit(s_full + 8 * t);
            };
            auto pv = [&](int t, int st, bool acc) {
                const uint32_t v = base + L::ring + st * L::kv_tile;
#pragma unroll
                for (int x = 0; x < kKeys / 16; x++)
                    mma_ts(tmem + L::o(t), tmem + L::s(t) + x * 8,
                           desc128(v + x * 2048, L::half, 1024), idesc<T>(D, true), acc || x > 0);
                umma::commit(o_done + 8 * t);
            };
            bool ok = wait(q_full, 0, fail);
            if (ok && tiles_rows == 2) ok = wait(q_full + 8, 0, fail);
            if (ok) ok = wait(kv_full, 0, fail);
            umma::fence_after();
            if (ok) {
                if (cnt0 > 0) qk(0, 0);
                if (tiles_rows == 2) qk(1, 0);
                if (NS < 2 * cnt) umma::commit(kv_empty);
            }
            for (int j = 0; j < cnt && ok; j++) {
                const int iv = 2 * j + 1, ik = 2 * j + 2, sv = iv % NS, sk = ik % NS;
                ok = wait(kv_full + 8 * sv, (iv / NS) & 1, fail);
                bool k_here = false;
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const int mine = t == 0 ? cnt0 : tiles_rows == 2 ? cnt : 0;
                    if (ok && j < mine) {
                        ok = wait(p_full + 8 * t, j & 1, fail);
                        umma::fence_after();
                        if (ok) pv(t, sv, j > 0);
                    }
                    if (ok && j + 1 < mine) {
                        if (!k_here) ok = wait(kv_full + 8 * sk, (ik / NS) & 1, fail);
                        k_here = true;
                        if (ok) qk(t, sk);
                    }
                }
                if (!ok) break;
                // only what the loader will wait for
                if (iv + NS < 2 * cnt) umma::commit(kv_empty + 8 * sv);
                if (ik + NS < 2 * cnt) umma::commit(kv_empty + 8 * sk);
            }
            if (!ok) {                      // let the products in flight end
                umma::commit(drain);
                umma::mbar_wait(drain, 0, umma::kWaitLimit);
            }
        }
        __syncwarp();
    } else {
        // ---- the rows ----------------------------------------------------------------
        const int t = warp / 4, r = threadIdx.x % kRows;
        const int row = row0 + t * kRows + r;
        const int mine = t == 0 ? cnt0 : tiles_rows == 2 ? cnt : 0;
        if (t < tiles_rows) {
            // Q into its swizzled place, a row by D / 8 neighbouring threads
            constexpr int CH = D / 8;
            for (int i = r; i < kRows * CH; i += kRows) {
                const int qr = i / CH, c = i % CH, x = row0 + t * kRows + qr;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (x < rows)
                    v = *(const uint4 *)((const T *)a.q + (int64_t)(rq.t0 + x / a.group) * a.q_token +
                                         (int64_t)(kvh * a.group + x % a.group) * a.q_head + c * 8);
                *(uint4 *)(basep + t * L::q_tile + (c / 8) * L::half + qr * 128 +
                           (((c % 8) ^ (qr & 7)) << 4)) = v;
            }
            umma::fence_smem_async();
            arrive(q_full + 8 * t);
        }
        const uint32_t lanes = (uint32_t)(warp % 4) * 32 << 16;
        const uint32_t st = tmem + L::s(t) + lanes, ot = tmem + L::o(t) + lanes;
        const bool warp_live = row0 + t * kRows + (warp % 4) * 32 < rows;
        const int see = PACKED ? 0 : row < rows ? sees(row) : 0;
        const float c = a.scale_log2;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < mine; j++) {
            const bool pre = first + j < pre_tiles;
            const int k0 = (first + j - (pre ? 0 : pre_tiles)) * kKeys;
            const int held = (pre ? n_pre : own_seen) - k0;     // keys in the tile
            // A tile that is not full: what lies behind its keys may be anything,
            // and a weight of zero does not hide a NaN.  The same for keys that
            // only some rows see, unless they are finite.
            const bool cut = causal && !pre && min(own_seen, k0 + kKeys) > see_first;
            if (held < kKeys || cut) {
                const int i = 2 * j + 1;
                ok = ok && wait(kv_full + 8 * (i % NS), (i / NS) & 1, fail);
                uint8_t *v = basep + L::ring + (i % NS) * L::kv_tile + r * 128;
                bool wipe = r >= held;
                if (cut && !wipe && k0 + r >= see_first) {
                    constexpr uint32_t E = fmt16<T>() ? 0x7f80u : 0x7c00u;
                    bool bad = false;
                    for (int x = 0; x < D / 8; x++) {
                        const uint4 q = *(const uint4 *)(v + (x / 8) * L::half + (x % 8) * 16);
                        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                        for (int y = 0; y < 4; y++)
                            bad |= (w[y] & E) == E || (w[y] >> 16 & E) == E;
                    }
                    if (bad) {
                        *dirty = 1;
                        __threadfence_block();
                        for (int x = 0; x < D / 2; x++) {
                            uint32_t *q = (uint32_t *)(v + (x / 32) * L::half + (x % 32) * 4);
                            uint32_t w = *q;
                            if ((w & E) == E) w &= 0xffff0000u;
                            if ((w >> 16 & E) == E) w &= 0xffffu;
                            *q = w;
                        }
                    }
                }
                if (wipe)
                    for (int x = 0; x < D / 8; x++)
                        *(uint4 *)(v + (x / 8) * L::half + (x % 8) * 16) = make_uint4(0, 0, 0, 0);
                umma::fence_smem_async();
            }
            ok = ok && wait(s_full + 8 * t, j & 1, fail);
            if (!__all_sync(~0u, ok)) break;
            umma::fence_after();
            if (warp_live) {
                float s[kKeys];
#pragma unroll
                for (int x = 0; x < kKeys; x += 32) tmem_ld32(st + x, s + x);
                tmem_ld_wait();
                const int lim = pre ? held : min(held, see - k0);
                if (held < kKeys || cut) {
#pragma unroll
                    for (int x = 0; x < kKeys; x++) s[x] = x < lim ? s[x] : -INFINITY;
                }
                float mx0 = s[0], mx1 = s[1], mx2 = s[2], mx3 = s[3];
#pragma unroll
                for (int x = 4; x < kKeys; x += 4) {
                    mx0 = fmaxf(mx0, s[x]);
                    mx1 = fmaxf(mx1, s[x + 1]);
                    mx2 = fmaxf(mx2, s[x + 2]);
                    mx3 = fmaxf(mx3, s[x + 3]);
                }
                const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));
                const bool grow = (mx - m) * c > 8.f;
                if (__any_sync(~0u, grow)) {
                    const float to = grow ? mx : m;
                    const float w = grow ? ex2(m * c - to * c) : 1.f;
                    if (j > 0) {
                        ok = wait(o_done + 8 * t, (j - 1) & 1, fail);
                        if (!__all_sync(~0u, ok)) break;
                        umma::fence_after();
#pragma unroll
                        for (int x = 0; x < D; x += 16) {
                            float o[16];
                            umma::tmem_ld16(ot + x, o);
                            uint32_t u[16];
#pragma unroll
                            for (int y = 0; y < 16; y++) u[y] = __float_as_uint(o[y] * w);
                            tmem_st16(ot + x, u);
                        }
                    }
                    l *= w;
                    m = to;
                }
                const float mc = m == -INFINITY ? 0.f : m * c;
                float l0 = 0.f, l1 = 0.f;
#pragma unroll
                for (int x = 0; x < kKeys; x += 32) {
                    uint32_t p[16];
#pragma unroll
                    for (int y = 0; y < 16; y++) {
                        const float p0 = ex2(fmaf(s[x + 2 * y], c, -mc));
                        const float p1 = ex2(fmaf(s[x + 2 * y + 1], c, -mc));
                        l0 += p0;
                        l1 += p1;
                        p[y] = pack2<T>(p0, p1);
                    }
                    tmem_st16(st + x / 2, p);
                }
                l += l0 + l1;
                tmem_st_wait();
            }
            umma::fence_before();
            arrive(p_full + 8 * t);
        }
        if (mine > 0 && ok) ok = wait(o_done + 8 * t, (mine - 1) & 1, fail);
        umma::fence_after();
        ok = __all_sync(~0u, ok);
        if (t < tiles_rows && warp_live && ok) {
            const bool direct = !PACKED && !a.packed && parts == 1;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int64_t orow = (int64_t)(rq.t0 + row / a.group) * a.q_heads + kvh * a.group +
                                 row % a.group;
            const int64_t slot = (int64_t)(PACKED ? part : a.prefix_parts + part) * a.tokens *
                                     a.q_heads + orow;
            __threadfence_block();
            const bool mend = *dirty && causal;
#pragma unroll 1
            for (int x = 0; x < D; x += 32) {
                __syncwarp();
                float o[32];
                if (mine > 0) {
                    tmem_ld32(ot + x, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int y = 0; y < 32; y++) o[y] = 0.f;
                }
                if (row >= rows) continue;
                if (mend) {
                    // what was wiped and is in sight of this row
                    const int end = min(see, max(0, first + each - pre_tiles) * kKeys);
                    for (int k = max(max(see_first, 0), (first - pre_tiles) * kKeys); k < end; k++) {
                        const int page = attn_page(a, a.pages + (int64_t)blockIdx.z * a.pages_row, k);
                        const T *v = (const T *)a.vp + (int64_t)page * a.v_page +
                                     (int64_t)(k & ((1 << a.page_shift) - 1)) * a.v_slot +
                                     (int64_t)kvh * a.v_head + x;
#pragma unroll
                        for (int y = 0; y < 32; y++) {
                            const float f = AttnType<T>::up(v[y]);
                            if (!isfinite(f)) o[y] += f;
                        }
                    }
                }
                if (direct) {
#pragma unroll
                    for (int y = 0; y < 32; y += 8) {
                        uint4 w;
                        w.x = pack2<T>(o[y] * inv, o[y + 1] * inv);
                        w.y = pack2<T>(o[y + 2] * inv, o[y + 3] * inv);
                        w.z = pack2<T>(o[y + 4] * inv, o[y + 5] * inv);
                        w.w = pack2<T>(o[y + 6] * inv, o[y + 7] * inv);
                        *(uint4 *)((T *)a.out + orow * D + x + y) = w;
                    }
                } else {
#pragma unroll
                    for (int y = 0; y < 32; y += 4)
                        *(float4 *)(a.part_o + slot * D + x + y) =
                            make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]);
                }
            }
            if (!direct && row < rows) a.part_ml[slot] = make_float2(m * c, l);
        }
    }
    umma::fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *fail) atomicOr(a.err, kAttnTimeout);
    if (warp == 8) {
        umma::fence_after();
        umma::tmem_free(tmem, 512);
    }
}

// ------------------------------------------------------------ host side --

static CUresult (*encode_fn())(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                               const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                               const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
    static const auto fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                             &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return (decltype(encode_fn()))p;
    }();
    return fn;
}

// The pages as a tensor (dim, slot, head, page), boxes of 64 columns by the
// keys of a page (128 at most).
static int page_map(CUtensorMap *m, const warp_kv_pages *c, void *ptr, int64_t page, int64_t slot,
                    int64_t head) {
    const auto fn = encode_fn();
    if (!fn) {
        set_error("warp_paged_attention: the driver has no cuTensorMapEncodeTiled");
        return WARP_E_CUDA;
    }
    const cuuint64_t row = (cuuint64_t)c->head_dim * 2;
    const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->page_size,
                                (cuuint64_t)c->kv_heads, (cuuint64_t)c->pages};
    // the stride of an axis of one entry may be given as 0
    const cuuint64_t strides[3] = {slot ? (cuuint64_t)slot * 2 : row,
                                   head ? (cuuint64_t)head * 2 : row,
                                   page ? (cuuint64_t)page * 2 : row};
    const cuuint32_t box[4] = {64, (cuuint32_t)(c->page_size < kKeys ? c->page_size : kKeys), 1, 1};
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    const CUresult r = fn(m, c->type == WARP_T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                   : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          4, ptr, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("warp_paged_attention: the pages' layout does not make a tensor map (%d)", (int)r);
        return WARP_E_ARG;
    }
    return WARP_OK;
}

template <typename T, int D, bool PACKED>
static int umma_launch(const AttnArgs &a, const CUtensorMap &km, const CUtensorMap &vm, int pairs,
                       int parts, cudaStream_t st) {
    static bool attr_done = false;                      // per instantiation, per process
    if (!attr_done) {
        const cudaError_t e =
            cudaFuncSetAttribute(attn_umma_kernel<T, D, PACKED>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<D>::bytes);
        if (e != cudaSuccess) return cuda_fail(e, "attention smem attribute");
        attr_done = true;
    }
    attn_umma_kernel<T, D, PACKED>
        <<<dim3((unsigned)pairs * parts, a.kv_heads, PACKED ? 1 : a.batch), kThreads,
           Lay<D>::bytes, st>>>(a, km, vm);
    WARP_CHECK_LAUNCH("attn_umma_kernel");
    return WARP_OK;
}

int attn_umma(const AttnArgs &a, const warp_kv_pages *c, bool packed, cudaStream_t st) {
    CUtensorMap km, vm;
    int rc = page_map(&km, c, c->k, c->k_page, c->k_slot, c->k_head);
    if (!rc) rc = page_map(&vm, c, c->v, c->v_page, c->v_slot, c->v_head);
    if (rc) return rc;
    const int64_t rows = (int64_t)(packed ? a.tokens : a.max_q) * a.group;
    const int pairs = (int)((rows + 2 * kRows - 1) / (2 * kRows));
    const int parts = packed ? a.prefix_parts : a.wide_parts;
    const bool h = c->type == WARP_T_F16, d64 = c->head_dim == 64;
    if (packed)
        return h ? d64 ? umma_launch<__half, 64, true>(a, km, vm, pairs, parts, st)
                       : umma_launch<__half, 128, true>(a, km, vm, pairs, parts, st)
                 : d64 ? umma_launch<__nv_bfloat16, 64, true>(a, km, vm, pairs, parts, st)
                       : umma_launch<__nv_bfloat16, 128, true>(a, km, vm, pairs, parts, st);
    return h ? d64 ? umma_launch<__half, 64, false>(a, km, vm, pairs, parts, st)
                   : umma_launch<__half, 128, false>(a, km, vm, pairs, parts, st)
             : d64 ? umma_launch<__nv_bfloat16, 64, false>(a, km, vm, pairs, parts, st)
                   : umma_launch<__nv_bfloat16, 128, false>(a, km, vm, pairs, parts, st);
}

}  // namespace warp
