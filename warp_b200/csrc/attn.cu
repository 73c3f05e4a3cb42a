// attn.cu — attention over paged keys and values for few query rows a key
// head: single-token decoding and short chunks.
//
// The rows of one CTA are 16 (token, head) pairs that read the same kv head,
// so each key and value is read once for the heads that share it.  With few
// rows a key the work is a stream of K and V at a handful of operations a
// byte: bound by memory.  The running maximum m and sum l make one pass of it:
//     m' = max(m, max_j x_j),  p_j = 2^(x_j - m'),
//     l' = l 2^(m - m') + sum p_j,  o' = o 2^(m - m') + sum p_j v_j
// with x = scale * log2(e) * q.k.  Key ranges are independent until they are
// joined the same way, which is done for the warps of a CTA in shared memory
// and for the parts of a long range by attn_join_kernel.
//
// Each warp streams its own tiles of 16 keys (every fourth of the CTA's range)
// through a private ring of shared memory filled by cp.async, so the loop has
// no barrier between warps.  Both products are mma.sync m16n8k16: S = Q K^T
// with Q held in registers, then O += P V with the accumulators of S repacked
// as P.  The tensor cores' rate does not matter here: 16 rows are far too few
// to fill a tcgen05 tile.  Measured: 32 streams of 8192 keys, 56 heads over 8 of
// 128, 168 us, 6.4 TB/s; one stream of 777 keys, 18 heads over 2, 8.3 us with
// the join.
#include "attn.cuh"

#include <math.h>

namespace warp {

constexpr int kADWarps = 4;
constexpr int kADStages = 3;
constexpr int kADRows = 16;

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4],
                                                 uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                        uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// 16 bytes, or zeros where `live` is false (the source is then not read).
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                 ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

template <typename T> struct F16Bits;
template <> struct F16Bits<__half> { static constexpr uint32_t exp = 0x7c00u, one = 0x3c00u; };
template <> struct F16Bits<__nv_bfloat16> { static constexpr uint32_t exp = 0x7f80u, one = 0x3f80u; };

// A weight of zero does not hide a value that is not finite (0 * inf is NaN),
// so where a tile holds keys that only some of its rows see, such values are
// taken out of the B operand (b0, b1) and counted for each row by products of
// the rows' visibility with indicators instead: what sees a NaN or both
// infinities becomes NaN, what sees one infinity becomes it.
template <typename T>
__device__ __forceinline__ void mend_values(uint32_t &b0, uint32_t &b1, const uint32_t (&seen)[4],
                                            float (&o)[4]) {
    constexpr uint32_t E = F16Bits<T>::exp, one = F16Bits<T>::one;
    const auto odd = [](uint32_t x) { return (x & E) == E || (x >> 16 & E) == E; };
    if (!__any_sync(~0u, odd(b0) || odd(b1))) return;
    float n_nan[4] = {}, n_pos[4] = {}, n_neg[4] = {};
    uint32_t is[3][2] = {};
    auto part = [&](uint32_t &b, int w) {
#pragma unroll
        for (int h = 0; h < 32; h += 16) {
            const uint32_t x = b >> h & 0xffffu;
            if ((x & E) != E) continue;
            b &= ~(0xffffu << h);
            is[(x & 0x7fffu) != E ? 0 : x >> 15 ? 2 : 1][w] |= one << h;
        }
    };
    part(b0, 0);
    part(b1, 1);
    mma16816<T>(n_nan, seen, is[0][0], is[0][1]);
    mma16816<T>(n_pos, seen, is[1][0], is[1][1]);
    mma16816<T>(n_neg, seen, is[2][0], is[2][1]);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (n_pos[e] > 0.f) o[e] += INFINITY;
        if (n_neg[e] > 0.f) o[e] -= INFINITY;
        if (n_nan[e] > 0.f) o[e] = NAN;
    }
}

template <int D> struct ADLay {
    static constexpr int row_bytes = D * 2;
    static constexpr int tile_bytes = kAttnTile * row_bytes;
    static constexpr int stage_bytes = 2 * tile_bytes;          // K, then V
    static constexpr int warp_bytes = kADStages * stage_bytes;
    static constexpr int ring = kADWarps * warp_bytes;
    // the warps' results when the ring is done with: o [warp][16][D + 4], m and l
    static constexpr int o_pitch = D + 4;
    static constexpr int join = kADWarps * kADRows * (o_pitch + 2) * 4;
    static constexpr int bytes = ring > join ? ring : join;
};

// PACKED: rows are those of all the batch's tokens, keys the shared prefix
// (one "request" for the batch).  Otherwise rows and keys of one request, with
// the prefix's keys in front where there is one that is not computed apart.
template <typename T, int D, bool PACKED>
__device__ __forceinline__ void attn_rows(const AttnArgs &a, uint8_t *smem) {
    using Lay = ADLay<D>;
    const int kvh = blockIdx.y;
    AttnReq rq;
    int part, row0, pre_tiles, own_tiles;
    if (PACKED) {
        rq = {0, a.tokens, 0};
        part = blockIdx.x % a.prefix_parts;
        row0 = (blockIdx.x / a.prefix_parts) * kADRows;
    } else {
        rq = attn_req(a, blockIdx.z);
        const int tiles_max = (a.packed ? 0 : (a.prefix_len + kAttnTile - 1) / kAttnTile) +
                              (a.max_kv + kAttnTile - 1) / kAttnTile;
        const int parts_max = max(1, attn_parts(tiles_max, a.split_tiles));
        part = blockIdx.x % parts_max;
        row0 = (blockIdx.x / parts_max) * kADRows;
    }
    const int rows = rq.n * a.group;
    if (row0 >= rows || (!PACKED && rows > a.rows_small)) return;
    const int n_pre = PACKED || !a.packed ? a.prefix_len : 0;
    pre_tiles = (n_pre + kAttnTile - 1) / kAttnTile;
    // own keys that the tile's last row sees
    const int last_row = min(rows, row0 + kADRows) - 1;
    int own_seen = rq.len;
    if (!PACKED && a.causal)
        own_seen = max(0, min(rq.len, rq.len - rq.n + last_row / a.group + 1));
    own_tiles = PACKED ? 0 : (own_seen + kAttnTile - 1) / kAttnTile;
    // parts are counted by the request's keys, whatever a tile's rows see, so
    // that the join knows their number
    const int all_tiles = pre_tiles + (PACKED ? 0 : (rq.len + kAttnTile - 1) / kAttnTile);
    const int each = PACKED ? a.prefix_split_tiles : a.split_tiles;
    const int parts = max(1, attn_parts(all_tiles, each));
    if (part >= parts) return;
    const int tile0 = part * each;
    const int tile1 = min(tile0 + each, pre_tiles + own_tiles);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int32_t *own_pages = PACKED ? nullptr : a.pages + (int64_t)blockIdx.z * a.pages_row;
    const T *kp = (const T *)a.kp + (int64_t)kvh * a.k_head;
    const T *vp = (const T *)a.vp + (int64_t)kvh * a.v_head;
    const uint32_t ring = smem_u32(smem) + warp * Lay::warp_bytes;

    // Page numbers of the warp's next 32 tiles, one a lane.
    int page_of = 0;
    auto pages_at = [&](int first) {
        const int i = first + lane * kADWarps;
        if (i < tile1)
            page_of = i < pre_tiles ? attn_page(a, a.prefix_pages, i * kAttnTile)
                                    : attn_page(a, own_pages, (i - pre_tiles) * kAttnTile);
    };
    // tile i (the n-th of this warp) into its ring stage
    auto fetch = [&](int i, int n) {
        if (n % 32 == 0) pages_at(i);
        const int64_t page = __shfl_sync(~0u, page_of, n % 32);
        if (i < tile1) {
            const bool pre = i < pre_tiles;
            const int j0 = (pre ? i : i - pre_tiles) * kAttnTile;
            const int live = (pre ? n_pre : own_seen) - j0;
            const int64_t off = j0 & ((1 << a.page_shift) - 1);
            const T *ks = kp + page * a.k_page + off * a.k_slot;
            const T *vs = vp + page * a.v_page + off * a.v_slot;
            const uint32_t dst = ring + (n % kADStages) * Lay::stage_bytes;
            constexpr int CH = D / 8;                   // 16-byte pieces of a row
#pragma unroll
            for (int c = lane; c < kAttnTile * CH; c += 32) {
                const int r = c / CH, p = c % CH;
                const uint32_t at = dst + r * Lay::row_bytes + ((p ^ (r & 7)) << 4);
                cp_async16_or_zero(at, ks + r * a.k_slot + p * 8, r < live);
                cp_async16_or_zero(at + Lay::tile_bytes, vs + r * a.v_slot + p * 8, r < live);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int n = 0; n < kADStages - 1; n++) fetch(tile0 + warp + n * kADWarps, n);

    // Q: the A operand, 16 rows x D
    uint32_t qf[D / 16][4];
    const int rlo = row0 + lane / 4, rhi = rlo + 8;
    {
        const T *qlo = nullptr, *qhi = nullptr;
        if (rlo < rows)
            qlo = (const T *)a.q + (int64_t)(rq.t0 + rlo / a.group) * a.q_token +
                  (int64_t)(kvh * a.group + rlo % a.group) * a.q_head;
        if (rhi < rows)
            qhi = (const T *)a.q + (int64_t)(rq.t0 + rhi / a.group) * a.q_token +
                  (int64_t)(kvh * a.group + rhi % a.group) * a.q_head;
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
            const int c = k * 16 + (lane % 4) * 2;
            qf[k][0] = qlo ? *(const uint32_t *)(qlo + c) : 0u;
            qf[k][1] = qhi ? *(const uint32_t *)(qhi + c) : 0u;
            qf[k][2] = qlo ? *(const uint32_t *)(qlo + c + 8) : 0u;
            qf[k][3] = qhi ? *(const uint32_t *)(qhi + c + 8) : 0u;
        }
    }
    // own keys that the thread's two rows and the tile's first row see
    int see_lo = own_seen, see_hi = own_seen, see_first = own_seen;
    if (!PACKED && a.causal) {
        see_first = rq.len - rq.n + row0 / a.group + 1;
        see_lo = rq.len - rq.n + rlo / a.group + 1;
        see_hi = rq.len - rq.n + rhi / a.group + 1;
    }

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    // the running maxima, lowered
    constexpr float lift = attn_lift<T>(0.f);
    float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;

    int n = 0;
    for (int i = tile0 + warp; i < tile1; i += kADWarps, n++) {
        fetch(i + (kADStages - 1) * kADWarps, n + kADStages - 1);
        cp_async_wait<kADStages - 1>();
        __syncwarp();
        const uint32_t kb = ring + (n % kADStages) * Lay::stage_bytes;
        const uint32_t vb = kb + Lay::tile_bytes;

        float s[2][4] = {};
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
            uint32_t b[4];
            const int r = (lane & 7) + (lane >> 4) * 8, p = k * 2 + ((lane >> 3) & 1);
            ldsm4(b, kb + r * Lay::row_bytes + ((p ^ (r & 7)) << 4));
            mma16816<T>(s[0], qf[k], b[0], b[1]);
            mma16816<T>(s[1], qf[k], b[2], b[3]);
        }
        const bool pre = i < pre_tiles;
        const int j0 = (pre ? i : i - pre_tiles) * kAttnTile;
        const int lim_lo = pre ? n_pre - j0 : min(see_lo, own_seen) - j0;
        const int lim_hi = pre ? n_pre - j0 : min(see_hi, own_seen) - j0;
        float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int j = t * 8 + (lane % 4) * 2 + e;
                s[t][e] = j < lim_lo ? s[t][e] * a.scale_log2 : -INFINITY;
                s[t][2 + e] = j < lim_hi ? s[t][2 + e] * a.scale_log2 : -INFINITY;
                mx_lo = fmaxf(mx_lo, s[t][e]);
                mx_hi = fmaxf(mx_hi, s[t][2 + e]);
            }
#pragma unroll
        for (int x = 1; x <= 2; x <<= 1) {
            mx_lo = fmaxf(mx_lo, __shfl_xor_sync(~0u, mx_lo, x));
            mx_hi = fmaxf(mx_hi, __shfl_xor_sync(~0u, mx_hi, x));
        }
        mx_lo = fmaxf(m_lo, mx_lo - lift);
        mx_hi = fmaxf(m_hi, mx_hi - lift);
        if (__any_sync(~0u, mx_lo > m_lo || mx_hi > m_hi)) {
            const float w_lo = mx_lo == -INFINITY ? 1.f : ex2(m_lo - mx_lo);
            const float w_hi = mx_hi == -INFINITY ? 1.f : ex2(m_hi - mx_hi);
            l_lo *= w_lo;
            l_hi *= w_hi;
#pragma unroll
            for (int d = 0; d < D / 8; d++) {
                o[d][0] *= w_lo;
                o[d][1] *= w_lo;
                o[d][2] *= w_hi;
                o[d][3] *= w_hi;
            }
            m_lo = mx_lo;
            m_hi = mx_hi;
        }
        const float z_lo = m_lo == -INFINITY ? 0.f : m_lo, z_hi = m_hi == -INFINITY ? 0.f : m_hi;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                s[t][e] = ex2(s[t][e] - z_lo);
                s[t][2 + e] = ex2(s[t][2 + e] - z_hi);
                l_lo += s[t][e];
                l_hi += s[t][2 + e];
            }
        uint32_t p[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]),
                         pack2<T>(s[1][0], s[1][1]), pack2<T>(s[1][2], s[1][3])};
        // a tile that some of the rows see only in part
        const bool cut = !PACKED && !pre && min(own_seen, j0 + kAttnTile) > see_first;
        uint32_t seen[4];
        if (cut) {
            const int c = (lane % 4) * 2;
            seen[0] = pack2<T>(c < lim_lo, c + 1 < lim_lo);
            seen[1] = pack2<T>(c < lim_hi, c + 1 < lim_hi);
            seen[2] = pack2<T>(c + 8 < lim_lo, c + 9 < lim_lo);
            seen[3] = pack2<T>(c + 8 < lim_hi, c + 9 < lim_hi);
        }
#pragma unroll
        for (int d = 0; d < D / 16; d++) {
            uint32_t b[4];
            const int r = (lane & 7) + ((lane >> 3) & 1) * 8, c = d * 2 + (lane >> 4);
            ldsm4t(b, vb + r * Lay::row_bytes + ((c ^ (r & 7)) << 4));
            if (cut) {
                mend_values<T>(b[0], b[1], seen, o[2 * d]);
                mend_values<T>(b[2], b[3], seen, o[2 * d + 1]);
            }
            mma16816<T>(o[2 * d], p, b[0], b[1]);
            mma16816<T>(o[2 * d + 1], p, b[2], b[3]);
        }
        __syncwarp();                       // the stage is free for the next fetch
    }
    cp_async_wait<0>();
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
        l_lo += __shfl_xor_sync(~0u, l_lo, x);
        l_hi += __shfl_xor_sync(~0u, l_hi, x);
    }
    __syncthreads();
    // join the warps
    float *so = (float *)smem;
    float *sm = so + kADWarps * kADRows * Lay::o_pitch, *sl = sm + kADWarps * kADRows;
    {
        float *mine = so + warp * kADRows * Lay::o_pitch;
        const int r = lane / 4;
#pragma unroll
        for (int d = 0; d < D / 8; d++) {
            const int c = d * 8 + (lane % 4) * 2;
            *(float2 *)(mine + r * Lay::o_pitch + c) = make_float2(o[d][0], o[d][1]);
            *(float2 *)(mine + (r + 8) * Lay::o_pitch + c) = make_float2(o[d][2], o[d][3]);
        }
        if (lane % 4 == 0) {
            sm[warp * kADRows + r] = m_lo;
            sm[warp * kADRows + r + 8] = m_hi;
            sl[warp * kADRows + r] = l_lo;
            sl[warp * kADRows + r + 8] = l_hi;
        }
    }
    __syncthreads();
    constexpr int TPR = D / 4;                          // threads a row, 4 values each
    const bool direct = !PACKED && !a.packed && parts == 1;
#pragma unroll
    for (int r = threadIdx.x / TPR; r < kADRows; r += kADWarps * 32 / TPR) {
        if (row0 + r >= rows) break;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kADWarps; w++) M = fmaxf(M, sm[w * kADRows + r]);
        const float z = M == -INFINITY ? 0.f : M;
        float l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        const int c = (threadIdx.x % TPR) * 4;
#pragma unroll
        for (int w = 0; w < kADWarps; w++) {
            const float f = ex2(sm[w * kADRows + r] - z);
            l += f * sl[w * kADRows + r];
            const float4 x = *(const float4 *)(so + (w * kADRows + r) * Lay::o_pitch + c);
            v.x += f * x.x;
            v.y += f * x.y;
            v.z += f * x.z;
            v.w += f * x.w;
        }
        const int64_t row = (int64_t)(rq.t0 + (row0 + r) / a.group) * a.q_heads +
                            kvh * a.group + (row0 + r) % a.group;
        if (direct) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            uint2 w;
            w.x = pack2<T>(v.x * inv, v.y * inv);
            w.y = pack2<T>(v.z * inv, v.w * inv);
            *(uint2 *)((T *)a.out + row * D + c) = w;
        } else {
            const int64_t slot = (int64_t)(PACKED ? part : a.prefix_parts + part) * a.tokens *
                                     a.q_heads + row;
            *(float4 *)(a.part_o + slot * D + c) = v;
            if (c == 0) a.part_ml[slot] = make_float2(M, l);
        }
    }
}

// The kernels of one call are launched so that each may start while the one
// before it runs (they read the same inputs and write different parts), and
// the last block of each waits for that one before it ends, so that the last
// one's end is the end of all.
// That one lets nothing start early: what follows the call may count on its
// results as soon as it runs.
template <typename T, int D, bool PACKED>
__global__ void __launch_bounds__(kADWarps * 32, 2)
attn_rows_kernel(const __grid_constant__ AttnArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    if (a.more) pdl_trigger();
    attn_rows<T, D, PACKED>(a, smem);
    attn_wait_last();
}

// Parts p0..p1-1 of one row, in order: the largest maximum M, the sum l and the
// lane's D / 32 values of o, both measured from M.  Each lane keeps the weight of
// one part in 32.
template <int D>
__device__ __forceinline__ void join_parts(const AttnArgs &a, int64_t row, int p0, int p1, float &M,
                                           float &l, float (&acc)[D / 32]) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x % 32;
    const int64_t rows = (int64_t)a.tokens * a.q_heads, stride = rows * D;
    const float *const src = a.part_o + row * D + lane * V;
    M = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0.f;
    for (; p0 < p1; p0 += 32) {
        const int p = p0 + lane, here = min(32, p1 - p0);
        const float2 ml = p < p1 ? a.part_ml[p * rows + row] : make_float2(-INFINITY, 0.f);
        float m = fmaxf(M, ml.x);
#pragma unroll
        for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, x));
        const float z = m == -INFINITY ? 0.f : m;
        const float keep = ex2(M - z), w = ex2(ml.x - z);
        l = l * keep + w * ml.y;            // a lane's own parts
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] *= keep;
        M = m;
        // eight parts' loads in flight
        for (int k0 = 0; k0 < here; k0 += 8) {
            float v[8][V];
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k0 + k < here) {
                    if (V == 4) *(float4 *)v[k] = *(const float4 *)(src + (p0 + k0 + k) * stride);
                    else *(float2 *)v[k] = *(const float2 *)(src + (p0 + k0 + k) * stride);
                }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float f = __shfl_sync(~0u, w, k0 + k);
                if (k0 + k < here)
#pragma unroll
                    for (int i = 0; i < V; i++) acc[i] += f * v[k][i];
            }
        }
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) l += __shfl_xor_sync(~0u, l, x);
}

template <typename T, int D>
__device__ __forceinline__ void join_store(const AttnArgs &a, int64_t row, float l,
                                           const float (&acc)[D / 32]) {
    constexpr int V = D / 32;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t o[V / 2];
#pragma unroll
    for (int i = 0; i < V; i += 2) o[i / 2] = pack2<T>(acc[i] * inv, acc[i + 1] * inv);
    T *const dst = (T *)a.out + row * D + threadIdx.x % 32 * V;
    if (V == 4) *(uint2 *)dst = *(uint2 *)o;
    else *(uint32_t *)dst = o[0];
}

// Joins the parts of each row.  Rows whose request has one part were written by
// their CTA.  A block has a token, or a share of its heads, and a warp of it a
// row; with SPREAD, where rows are few, a block has one row and its warps a share
// of the parts each (two streams of 131071 keys: 171.6 us in all against 175.1).
template <typename T, int D, bool SPREAD>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int V = D / 32;
    __shared__ float2 ml_of[8];
    __shared__ float o_of[8][D];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, t = blockIdx.x;
    int parts = 0;
    // the token's request: the last one that starts at or before it
    int b = -1;
    for (int i0 = 0; i0 < a.batch; i0 += 32) {
        const int i = i0 + lane;
        const unsigned hit = __ballot_sync(~0u, i < a.batch && a.q_start[i] <= t);
        if (hit) b = i0 + 31 - __clz(hit);
        if (hit != ~0u) break;
    }
    if (b >= 0) {
        const AttnReq rq = attn_req(a, b);
        const bool wide = rq.n * a.group > a.rows_small;
        const int tile = wide ? attn_wide(D) : kAttnTile;
        const int own = (a.packed ? 0 : (a.prefix_len + tile - 1) / tile) +
                        (rq.len + tile - 1) / tile;
        parts = max(1, attn_parts(own, wide ? a.wide_each : a.split_tiles));
        if ((!a.packed && parts == 1) || t >= rq.t0 + rq.n) parts = 0;
        else parts += a.prefix_parts;
    }
    pdl_wait();
    if (!parts) return;
    float M, l, acc[V];
    if (!SPREAD) {
        for (int head = blockIdx.y * 8 + warp; head < a.q_heads; head += gridDim.y * 8) {
            const int64_t row = (int64_t)t * a.q_heads + head;
            join_parts<D>(a, row, 0, parts, M, l, acc);
            join_store<T, D>(a, row, l, acc);
        }
        return;
    }
    const int64_t row = (int64_t)t * a.q_heads + blockIdx.y;
    const int each = (parts + 7) / 8;
    join_parts<D>(a, row, min(parts, warp * each), min(parts, (warp + 1) * each), M, l, acc);
    if (lane == 0) ml_of[warp] = make_float2(M, l);
#pragma unroll
    for (int i = 0; i < V; i++) o_of[warp][lane * V + i] = acc[i];
    __syncthreads();
    if (warp) return;
    M = -INFINITY;
    for (int w = 0; w < 8; w++) M = fmaxf(M, ml_of[w].x);
    const float z = M == -INFINITY ? 0.f : M;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0.f;
    for (int w = 0; w < 8; w++) {
        const float f = ex2(ml_of[w].x - z);
        l += f * ml_of[w].y;
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] += f * o_of[w][lane * V + i];
    }
    join_store<T, D>(a, row, l, acc);
}

// ------------------------------------------------------------ host side --

struct AttnPlan {
    int packed, packed_wide, prefix_parts, prefix_each;
    int rows_small;
    int each, parts;                        // own parts at most, attn_rows_kernel
    int wide_each, wide_parts;              // and attn_umma_kernel (0 parts: not run)
    int small_tiles;                        // row tiles a request, attn_rows_kernel (0: not run)
    int join;
    int64_t o_bytes, ml_bytes;
    int max_q, max_kv;                      // the host's bounds, no wider than tokens and pages
};

static int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Key tiles a part, for `ctas` CTAs of `tiles` tiles each: the split that takes
// the fewest microseconds by the measured time of a tile, of a CTA around its
// tiles and, if there are parts, of the join (its launch, and `rows` rows of
// fp32 parts written and read again).
static int pick_split(int64_t tiles, int64_t ctas, int64_t slots, double tile_us, double cta_us,
                      int64_t least, double rows, int D) {
    ctas = ctas < 1 ? 1 : ctas;
    int64_t best = tiles < 1 ? 1 : tiles;
    double least_us = 1e30;
    for (int64_t parts = 1; parts <= 128; parts++) {
        const int64_t each = up(tiles < 1 ? 1 : tiles, parts);
        if (parts > 1 && each < least) break;
        const int64_t n = up(tiles < 1 ? 1 : tiles, each);
        const double x = (double)ctas * n / slots;
        // Lengths are known on the device alone.  If they are all the same: whole
        // waves while there are few of them (many even out).  If they spread
        // from a fifth of the largest up: their mean's work evened out, and half
        // a CTA's time until the last one is done, but no less than the longest.
        const double one = each * tile_us, waves = x < 4 ? (double)up(ctas * n, slots) : x + 0.5;
        const double same = waves * (one + cta_us);
        const double mixed = 0.6 * x * one + 0.5 * one;
        double us = 0.5 * same + 0.5 * ((mixed > one ? mixed : one) + (x < 1 ? 1 : x) * cta_us);
        if (n > 1) us += 3 + rows * n * D * 8 / 4e6;
        if (us < least_us * 0.98) best = each, least_us = us;
    }
    return (int)best;
}

// attn_rows_kernel: two CTAs an SM; 16 keys of K and V of one head at an even
// share of the memory's rate, or at least what a CTA's own latency allows.
static int split_rows(int64_t tiles, int64_t ctas, double rows, int D) {
    const double tile_us = D == 128 ? 0.36 : 0.20;
    return pick_split(tiles, ctas, 2 * 148, tile_us, 3.0, 4, rows, D);
}

// attn_umma_kernel: one CTA an SM; 128 keys for 256 rows, and a CTA around them.
static double wide_tile_us(int D) { return D == 128 ? 1.55 : 1.25; }
constexpr double kWideCtaUs = 7.0;

static int split_wide(int64_t tiles, int64_t ctas, double rows, int D) {
    return pick_split(tiles, ctas, 148, wide_tile_us(D), kWideCtaUs, 2, rows, D);
}

// The same for a prefix, whose CTAs share the card with the requests' own keys
// (`bytes` of them, at the memory's rate if they had it alone): no SM idles, so
// what counts is the work in all, or one CTA's time where that is longer. More
// parts shorten the one and add to the other (64 streams behind 16001 keys: 66 us
// with 5 parts, 79 with 9, 107 with 32).
static int split_prefix(int64_t tiles, int64_t ctas, double bytes, double rows, int D) {
    const double tile_us = wide_tile_us(D), own = 148 * (bytes / 6.2e6 + 3.0);
    int64_t best = tiles;
    double least_us = 1e30;
    for (int64_t parts = 1; parts <= 128 && (parts == 1 || up(tiles, parts) >= 2); parts++) {
        const int64_t each = up(tiles, parts), n = up(tiles, each);
        const double one = each * tile_us + kWideCtaUs + 2.0, all = (ctas * n * one + own) / 148;
        const double us = (one > all ? one : all) + rows * n * D * 8 / 4e6;
        if (us < least_us * 0.98) best = each, least_us = us;
    }
    return (int)best;
}

static AttnPlan attn_plan(const warp_attn_desc *d, const warp_kv_pages *c) {
    AttnPlan p = {};
    p.max_q = d->max_q < d->tokens ? d->max_q : d->tokens;
    const int64_t held = (int64_t)d->pages_per_row * c->page_size;
    p.max_kv = d->max_kv < held ? d->max_kv : (int)held;
    const int64_t group = d->q_heads / d->kv_heads;
    const int keys = attn_wide(d->head_dim);
    const int64_t out = (int64_t)d->tokens * d->q_heads;        // rows of the result
    // The prefix apart, for all rows at once, where a request's rows alone
    // would leave a row tile mostly empty.
    p.packed = d->prefix_len > 0 && d->batch > 1 && d->tokens * group <= (int64_t)128 * d->batch;
    const int pre = p.packed ? 0 : d->prefix_len;
    const int64_t rows = p.max_q * group;
    // A single request's rows are known to be more than a few: all of them wide.
    p.rows_small = d->batch == 1 && rows > kADRows ? 0 : kADRows;
    if (rows > p.rows_small) {
        const int64_t pairs = up(rows, 256) * d->batch, by_tokens = up(d->tokens * group, 256);
        const int64_t ctas = pairs < by_tokens + d->batch - 1 ? pairs : by_tokens + d->batch - 1;
        const int64_t tiles = up(p.max_kv, keys) + up(pre, keys);
        p.wide_each = split_wide(tiles, ctas * d->kv_heads, out, d->head_dim);
        p.wide_parts = tiles ? (int)up(tiles, p.wide_each) : 1;
    }
    if (p.rows_small) {
        const int64_t tiles = up(p.max_kv, kAttnTile) + up(pre, kAttnTile);
        p.small_tiles = (int)up(rows < p.rows_small ? rows : p.rows_small, kADRows);
        p.each = split_rows(tiles, (int64_t)d->batch * d->kv_heads * p.small_tiles, out,
                            d->head_dim);
        p.parts = tiles ? (int)up(tiles, p.each) : 1;
    }
    if (p.packed) {
        const int64_t all = d->tokens * group;
        p.packed_wide = all > kADRows;
        const int64_t tiles = up(d->prefix_len, p.packed_wide ? keys : kAttnTile);
        p.prefix_each =
            p.packed_wide ? split_prefix(tiles, up(all, 256) * d->kv_heads,
                                         0.6 * d->batch * p.max_kv * d->kv_heads * d->head_dim * 4,
                                         out, d->head_dim)
                          : split_rows(tiles, up(all, kADRows) * d->kv_heads, out, d->head_dim);
        p.prefix_parts = (int)up(tiles, p.prefix_each);
    }
    const int own = p.parts > p.wide_parts ? p.parts : p.wide_parts;
    p.join = p.packed || own > 1;
    const int64_t all = p.join ? p.prefix_parts + own : 0;
    p.o_bytes = up(all * out * d->head_dim * 4, 256) * 256;
    p.ml_bytes = up(all * out * 8, 256) * 256;
    return p;
}

static int attn_check(const warp_attn_desc *d, const warp_kv_pages *c) {
    const char *who = "warp_paged_attention";
    WARP_ARG(d, "%s: NULL description", who);
    const int rc = kv_pages_check(c, who);
    if (rc) return rc;
    WARP_ARG(d->batch >= 0 && d->tokens >= 0 && d->max_q >= 0 && d->max_kv >= 0 &&
                 d->prefix_len >= 0 && d->pages_per_row >= 0 && d->pages_row >= 0,
             "%s: negative size", who);
    WARP_ARG(d->q_heads >= 1 && d->kv_heads >= 1 && d->q_heads % d->kv_heads == 0,
             "%s: %d query heads over %d kv heads", who, d->q_heads, d->kv_heads);
    WARP_ARG(d->q_heads <= 65536, "%s: %d query heads", who, d->q_heads);
    WARP_ARG(d->head_dim == 64 || d->head_dim == 128, "%s: head_dim %d is not 64 or 128", who,
             d->head_dim);
    WARP_ARG(c->kv_heads == d->kv_heads && c->head_dim == d->head_dim && c->type == d->type,
             "%s: the pages hold %d heads of %d (type %d), the queries want %d of %d (type %d)",
             who, c->kv_heads, c->head_dim, c->type, d->kv_heads, d->head_dim, d->type);
    WARP_ARG(d->scale > 0.f && isfinite(d->scale), "%s: scale %g is not positive", who,
             (double)d->scale);
    WARP_ARG(d->kv_heads <= 65535 && d->batch <= 65535, "%s: more than 65535 requests or kv heads",
             who);
    WARP_ARG(d->max_kv < (1 << 30) && d->prefix_len < (1 << 30), "%s: more than 2^30 keys", who);
    WARP_ARG((int64_t)d->tokens * d->q_heads < (int64_t)1 << 30, "%s: more than 2^30 rows", who);
    return WARP_OK;
}

template <typename T, int D>
static int attn_launch(AttnArgs a, const AttnPlan &p, bool first, cudaStream_t st) {
    using Lay = ADLay<D>;
    static std::atomic<uint64_t> done[2];
    cudaError_t e = attn_smem(attn_rows_kernel<T, D, false>, Lay::bytes, done[0]);
    if (e == cudaSuccess) e = attn_smem(attn_rows_kernel<T, D, true>, Lay::bytes, done[1]);
    if (e != cudaSuccess) return cuda_fail(e, "attention smem attribute");
    if (p.packed && !p.packed_wide) {
        a.more = 1;
        e = attn_start(attn_rows_kernel<T, D, true>,
                       dim3((unsigned)(up((int64_t)a.tokens * a.group, kADRows) * p.prefix_parts),
                            a.kv_heads, 1), kADWarps * 32, Lay::bytes, st, first, a);
        if (e != cudaSuccess) return cuda_fail(e, "attn_rows_kernel (prefix)");
        count_launch();
        first = false;
    }
    if (p.small_tiles) {
        a.more = p.join;
        e = attn_start(attn_rows_kernel<T, D, false>,
                       dim3(p.small_tiles * p.parts, a.kv_heads, a.batch), kADWarps * 32,
                       Lay::bytes, st, first, a);
        if (e != cudaSuccess) return cuda_fail(e, "attn_rows_kernel");
        count_launch();
        first = false;
    }
    if (p.join) {
        // a token's heads in one block, or shared out while the card has room, down
        // to a block a row
        const unsigned most = cdiv(a.q_heads, 8), room = cdiv(8 * 148, a.tokens);
        const bool spread = p.prefix_parts + (p.parts > p.wide_parts ? p.parts : p.wide_parts) > 8 &&
                            (int64_t)a.tokens * a.q_heads <= 8 * 148;
        e = spread ? attn_start(attn_join_kernel<T, D, true>, dim3(a.tokens, a.q_heads), 256, 0, st,
                                first, a)
                   : attn_start(attn_join_kernel<T, D, false>,
                                dim3(a.tokens, most < room ? most : room), 256, 0, st, first, a);
        if (e != cudaSuccess) return cuda_fail(e, "attn_join_kernel");
        count_launch();
    }
    return WARP_OK;
}

}  // namespace warp

extern "C" int64_t warp_attn_scratch(const warp_attn_desc *d, const warp_kv_pages *c) {
    const int rc = warp::attn_check(d, c);
    if (rc) return rc;
    const warp::AttnPlan p = warp::attn_plan(d, c);
    return p.o_bytes + p.ml_bytes;
}

extern "C" int warp_paged_attention(const warp_attn_desc *d, const warp_kv_pages *c, void *scratch,
                                    void *stream) {
    int rc = warp::attn_check(d, c);
    if (rc) return rc;
    if (d->tokens == 0 || d->batch == 0 || d->max_q == 0) return WARP_OK;
    const char *who = "warp_paged_attention";
    WARP_ARG(d->q && d->out && d->q_start && d->kv_len, "%s: NULL pointer", who);
    WARP_ARG(d->pages || d->pages_per_row == 0, "%s: NULL page table", who);
    WARP_ARG(d->prefix_pages || d->prefix_len == 0, "%s: NULL prefix page table", who);
    WARP_ARG(((uintptr_t)d->q & 15) == 0 && ((uintptr_t)d->out & 15) == 0 && d->q_token % 8 == 0 &&
                 d->q_head % 8 == 0,
             "%s: queries and results must be 16-byte aligned, strides multiples of 16 bytes", who);
    const warp::AttnPlan p = warp::attn_plan(d, c);
    WARP_ARG(p.o_bytes + p.ml_bytes == 0 || (scratch && ((uintptr_t)scratch & 255) == 0),
             "%s: scratch must be 256-byte aligned", who);
    warp::AttnArgs a = {};
    a.q = d->q, a.kp = c->k, a.vp = c->v, a.out = d->out;
    a.q_token = d->q_token, a.q_head = d->q_head;
    a.k_page = c->k_page, a.k_slot = c->k_slot, a.k_head = c->k_head;
    a.v_page = c->v_page, a.v_slot = c->v_slot, a.v_head = c->v_head;
    a.q_start = d->q_start, a.kv_len = d->kv_len;
    a.pages = d->pages, a.prefix_pages = d->prefix_pages, a.pages_row = d->pages_row;
    a.pages_per_row = d->pages_per_row, a.page_shift = __builtin_ctz(c->page_size);
    a.n_pages = (int)c->pages;
    a.batch = d->batch, a.tokens = d->tokens;
    a.q_heads = d->q_heads, a.kv_heads = d->kv_heads, a.group = d->q_heads / d->kv_heads;
    a.max_q = p.max_q, a.max_kv = p.max_kv, a.causal = d->causal != 0;
    a.prefix_len = d->prefix_len;
    a.scale_log2 = d->scale * 1.4426950408889634f;
    a.part_o = (float *)scratch;
    a.part_ml = (float2 *)((char *)scratch + p.o_bytes);
    a.packed = p.packed, a.prefix_parts = p.prefix_parts;
    a.rows_small = p.rows_small;
    a.split_tiles = p.each, a.wide_each = p.wide_each, a.wide_parts = p.wide_parts;
    a.prefix_split_tiles = a.prefix_wide_each = p.prefix_each;
    a.by_group = warp::attn_div(a.group);
    a.by_wide_parts = warp::attn_div(p.wide_parts), a.by_wide_each = warp::attn_div(p.wide_each);
    a.by_prefix_parts = warp::attn_div(p.prefix_parts);
    a.by_prefix_each = warp::attn_div(p.prefix_each);
    rc = warp::attn_err_word(&a.err);
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    bool first = true;
    if (p.packed_wide) {
        a.more = 1;
        rc = warp::attn_umma(a, c, true, first, st), first = false;
    }
    if (!rc && p.wide_parts) {
        a.more = p.small_tiles || p.join;
        rc = warp::attn_umma(a, c, false, first, st), first = false;
    }
    if (rc) return rc;
    if (d->type == WARP_T_F16)
        return d->head_dim == 64 ? warp::attn_launch<__half, 64>(a, p, first, st)
                                 : warp::attn_launch<__half, 128>(a, p, first, st);
    return d->head_dim == 64 ? warp::attn_launch<__nv_bfloat16, 64>(a, p, first, st)
                             : warp::attn_launch<__nv_bfloat16, 128>(a, p, first, st);
}
