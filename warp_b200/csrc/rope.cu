// rope.cu — per-head norm and rotary positions of queries and keys, with the
// keys and values written to a paged cache in the same pass.
//
// One row is the head_dim values of one (token, head).  With a the angle of
// pair i at the token's position,
//     (x0, x1) -> (x0 cos a - x1 sin a, x0 sin a + x1 cos a),
// after x -> x / sqrt(mean(x^2) + eps) * w where a norm is asked for.  Nothing
// is read twice, so the kernel is bound by memory: one read of q, k, v and one
// write of the results.
//
// A thread owns a "unit" of 2*VEC values of a row: the two VEC-wide vectors
// whose elements are each other's partners (half layout: VEC values of the
// first half and the VEC values rot_dim/2 further on; interleaved: 2*VEC
// neighbours), so that the rotation needs no exchange between threads.  A
// row's units sit on neighbouring lanes, and the norm's sum is a butterfly over them.
#include "attn.cuh"

#include <atomic>
#include <climits>

namespace warp {

__device__ unsigned g_attn_err;

// Takes off the bits that have been reported, and no other.
__global__ void attn_err_clear_kernel(unsigned bits) { atomicAnd(&g_attn_err, ~bits); }

// The word's address is fixed once its device is in use: looked up once for each.
int attn_err_word(unsigned **out) {
    constexpr int kDevices = 64;
    static std::atomic<unsigned *> known[kDevices];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && dev < kDevices && (*out = known[dev].load())) return WARP_OK;
    if (e == cudaSuccess) e = cudaGetSymbolAddress((void **)out, g_attn_err);
    if (e != cudaSuccess) return cuda_fail(e, "attention error word");
    if (dev < kDevices) known[dev].store(*out);
    return WARP_OK;
}

int kv_pages_check(const warp_kv_pages *c, const char *who) {
    WARP_ARG(c && c->k && c->v, "%s: NULL pages", who);
    WARP_ARG(c->type == WARP_T_F16 || c->type == WARP_T_BF16,
             "%s: pages must be fp16 or bf16 (type %d)", who, c->type);
    WARP_ARG(c->page_size >= 16 && c->page_size <= 4096 && !(c->page_size & (c->page_size - 1)),
             "%s: page_size %d is not a power of two in 16..4096", who, c->page_size);
    WARP_ARG(c->pages >= 1 && c->pages < ((int64_t)1 << 31), "%s: %lld pages", who,
             (long long)c->pages);
    WARP_ARG(c->kv_heads >= 1 && c->head_dim >= 2, "%s: kv_heads %d, head_dim %d", who,
             c->kv_heads, c->head_dim);
    WARP_ARG((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, "%s: pages must be 16-byte aligned",
             who);
    const int64_t st[6] = {c->k_page, c->k_slot, c->k_head, c->v_page, c->v_slot, c->v_head};
    const int64_t extent[3] = {c->pages, c->page_size, c->kv_heads};
    for (int i = 0; i < 6; i++)
        WARP_ARG(st[i] >= (extent[i % 3] > 1) && (st[i] & 7) == 0,
                 "%s: page strides must be positive multiples of 16 bytes (0 only on an axis of "
                 "one entry)", who);
    return WARP_OK;
}

struct RopeArgs {
    const void *q, *k, *v;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;
    void *q_out, *k_out;                    // contiguous [tokens][heads][D]
    const float *q_norm, *k_norm;
    const double *inv_freq;
    const int32_t *positions;
    const int64_t *slots;                   // non-NULL: append to the pages
    void *kp, *vp;
    int64_t k_page, k_slot, k_ph, v_page, v_slot, v_ph;
    int64_t n_slots;
    unsigned *err;
    float eps, rot_scale;
    int tokens, q_heads, kv_heads, D, rot, interleaved, page_shift;
    int rows;                               // rows a token: q, then k, then v (append)
    int shares, rows_per_share;             // of a token's rows, one share a warp
};

template <typename T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) RopeVec {
    T x[N];
};

constexpr int kRopeWarps = 4;
constexpr int kRopeCtas = 7;                // an SM: occupancy is what hides the latency here
constexpr int kRopeMaxPairs = 128;          // head_dim up to 256

template <int VEC> __device__ __forceinline__ void rope_f32(float (&x)[VEC], const float *p) {
    const RopeVec<float, VEC> v = *(const RopeVec<float, VEC> *)p;
#pragma unroll
    for (int i = 0; i < VEC; i++) x[i] = v.x[i];
}

// L lanes a row, UPL units a lane.
template <typename TI, typename TO, int VEC, int L, int UPL>
__global__ void __launch_bounds__(kRopeWarps * 32, kRopeCtas) rope_kernel(const RopeArgs a) {
    __shared__ alignas(16) float turns_of[kRopeWarps][2 * kRopeMaxPairs];
    constexpr int RPW = 32 / L;             // rows of a warp at a time
    const int warp = threadIdx.x / 32, lane = threadIdx.x % L;
    const int64_t id = (int64_t)blockIdx.x * kRopeWarps + warp;
    const int t = (int)(id / a.shares);
    if (t >= a.tokens) return;
    const int row0 = (int)(id - (int64_t)t * a.shares) * a.rows_per_share + threadIdx.x % 32 / L;
    const int row1 = min(a.rows, row0 - threadIdx.x % 32 / L + a.rows_per_share);
    const int half = a.rot / 2;
    const int units = a.D / (2 * VEC), rot_units = a.rot / (2 * VEC);
    const int k0 = a.q_heads, v0 = a.q_heads + a.kv_heads;      // first rows of k and v

    // Where unit n's two vectors start.  Half layout: the rotated units first,
    // behind them the rest of the row in two halves; interleaved: the whole row in
    // two halves, as pairs lie within a vector (but for single values).
    // Neighbouring lanes' vectors are neighbours either way.
    int at0[UPL], at1[UPL];
#pragma unroll
    for (int n = 0; n < UPL; n++) {
        const int u = lane + n * L;
        if (a.interleaved) {
            at0[n] = VEC > 1 ? u * VEC : 2 * u;
            at1[n] = VEC > 1 ? (units + u) * VEC : 2 * u + 1;
        } else {
            const bool turned = u < rot_units;
            at0[n] = turned ? u * VEC : a.rot + (u - rot_units) * VEC;
            at1[n] = turned ? half + u * VEC : at0[n] + (units - rot_units) * VEC;
        }
    }
    // The angle in turns, its two products with their rounding errors kept and
    // 1 / (2 pi) in two words, so that the fraction of a turn that is left is as
    // exact at position 2^31 (some 2^28 turns, of which one product alone would lose
    // 2^-25) as at 1: fp32 holds it to 2^-26.
    float *const cosines = turns_of[warp], *const sines = cosines + kRopeMaxPairs;
    if (half) {
        const double pos = (double)a.positions[t];
        for (int i = threadIdx.x % 32; i < half; i += 32) {
            constexpr double hi = 0.15915494309189533577, lo = -9.839338337591243e-18;
            const double f = a.inv_freq[i], x = pos * f, x_low = fma(pos, f, -x);
            const double whole = x * hi, low = fma(x, hi, -whole) + fma(x, lo, x_low * hi);
            const double turns = (whole - rint(whole)) + low;
            float si, co;
            sincospif(2.0f * (float)turns, &si, &co);
            cosines[i] = co * a.rot_scale;
            sines[i] = si * a.rot_scale;
        }
        __syncwarp();
    }
    int64_t slot = -1, page = 0, off = 0;
    if (a.slots) {
        slot = a.slots[t];
        if (slot >= a.n_slots) {
            if (threadIdx.x % 32 == 0) atomicOr(a.err, kAttnBadSlot);
            slot = -1;
        }
        page = slot >> a.page_shift, off = slot & ((1 << a.page_shift) - 1);
    }
    const float inv_d = 1.0f / (float)a.D;
    const bool norms = a.q_norm || a.k_norm;

    // Where the lane's row is read and written, and how far on its next one is, for
    // as long as it stays among q's, k's or v's rows (up to row `until`).
    const TI *src = nullptr;
    TO *dst = nullptr;
    const float *w = nullptr;
    int64_t src_step = 0, dst_step = 0;
    int until = 0;
    bool turned = false;
    auto enter = [&](int r) {
        if (r < k0) {
            src = (const TI *)a.q + t * a.q_token + r * a.q_head;
            src_step = RPW * a.q_head;
            dst = (TO *)a.q_out + ((int64_t)t * a.q_heads + r) * a.D;
            dst_step = RPW * a.D;
            w = a.q_norm;
            until = k0;
        } else if (r < v0) {
            const int h = r - k0;
            src = (const TI *)a.k + t * a.k_token + h * a.k_head;
            src_step = RPW * a.k_head;
            dst = a.slots ? (TO *)a.kp + page * a.k_page + off * a.k_slot + h * a.k_ph
                          : (TO *)a.k_out + ((int64_t)t * a.kv_heads + h) * a.D;
            dst_step = RPW * (a.slots ? a.k_ph : a.D);
            w = a.k_norm;
            until = v0;
        } else {
            const int h = r - v0;
            src = (const TI *)a.v + t * a.v_token + h * a.v_head;
            src_step = RPW * a.v_head;
            dst = (TO *)a.vp + page * a.v_page + off * a.v_slot + h * a.v_ph;
            dst_step = RPW * a.v_ph;
            w = nullptr;
            until = INT_MAX;
        }
        turned = half && r < v0;
    };

    // Every lane takes every step, for the sums across lanes.
    for (int r = row0; r - (int)(threadIdx.x % 32) / L < row1; r += RPW) {
        const bool live = r < row1;
        float x0[UPL][VEC], x1[UPL][VEC];
        if (r >= until && live) enter(r);
#pragma unroll
        for (int n = 0; n < UPL; n++) {
            RopeVec<TI, VEC> a0 = {}, a1 = {};
            if (live && lane + n * L < units) {
                a0 = *(const RopeVec<TI, VEC> *)(src + at0[n]);
                a1 = *(const RopeVec<TI, VEC> *)(src + at1[n]);
            }
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                x0[n][i] = AttnType<TI>::up(a0.x[i]);
                x1[n][i] = AttnType<TI>::up(a1.x[i]);
            }
        }
        if (norms) {
            float ss = 0.f;
#pragma unroll
            for (int n = 0; n < UPL; n++)
#pragma unroll
                for (int i = 0; i < VEC; i++) ss += x0[n][i] * x0[n][i] + x1[n][i] * x1[n][i];
#pragma unroll
            for (int o = L / 2; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
            if (w) {
                const float inv = rsqrtf(ss * inv_d + a.eps);
#pragma unroll
                for (int n = 0; n < UPL; n++) {
                    if (lane + n * L >= units) continue;
                    float w0[VEC], w1[VEC];
                    rope_f32<VEC>(w0, w + at0[n]);
                    rope_f32<VEC>(w1, w + at1[n]);
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        x0[n][i] *= inv * w0[i];
                        x1[n][i] *= inv * w1[i];
                    }
                }
            }
        }
        TO *const to = dst;
        src += src_step;
        dst += dst_step;
        if (!live || (slot < 0 && a.slots && r >= k0)) continue;
#pragma unroll
        for (int n = 0; n < UPL; n++) {
            if (lane + n * L >= units) continue;
            auto turn = [](float &x, float &y, float c, float s) {
                const float r0 = x * c - y * s, r1 = x * s + y * c;
                x = r0;
                y = r1;
            };
            if (!turned) {
                // passes through
            } else if (VEC > 1 && a.interleaved) {
                constexpr int P = (VEC + 1) / 2;
                float c[P], s[P];
                if (at0[n] < a.rot) {
                    rope_f32<P>(c, cosines + at0[n] / 2);
                    rope_f32<P>(s, sines + at0[n] / 2);
#pragma unroll
                    for (int i = 0; i < P; i++)
                        turn(x0[n][2 * i % VEC], x0[n][(2 * i + 1) % VEC], c[i], s[i]);
                }
                if (at1[n] < a.rot) {
                    rope_f32<P>(c, cosines + at1[n] / 2);
                    rope_f32<P>(s, sines + at1[n] / 2);
#pragma unroll
                    for (int i = 0; i < P; i++)
                        turn(x1[n][2 * i % VEC], x1[n][(2 * i + 1) % VEC], c[i], s[i]);
                }
            } else if (lane + n * L < rot_units) {
                float c[VEC], s[VEC];
                rope_f32<VEC>(c, cosines + (lane + n * L) * VEC);
                rope_f32<VEC>(s, sines + (lane + n * L) * VEC);
#pragma unroll
                for (int i = 0; i < VEC; i++) turn(x0[n][i], x1[n][i], c[i], s[i]);
            }
            RopeVec<TO, VEC> o0, o1;
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                o0.x[i] = AttnType<TO>::down(x0[n][i]);
                o1.x[i] = AttnType<TO>::down(x1[n][i]);
            }
            *(RopeVec<TO, VEC> *)(to + at0[n]) = o0;
            *(RopeVec<TO, VEC> *)(to + at1[n]) = o1;
        }
    }
}

template <typename TI, typename TO, int VEC, int L, int UPL>
static int rope_launch(RopeArgs &a, cudaStream_t st) {
    constexpr int RPW = 32 / L;
    // A token's rows are shared out among warps while there are fewer than
    // 32 an SM, down to one step of a warp each.
    const int64_t steps = (a.rows + RPW - 1) / RPW, want = (int64_t)32 * 148;
    int64_t shares = a.tokens < want ? want / a.tokens : 1;
    shares = shares < 1 ? 1 : shares > steps ? steps : shares;
    const int64_t each = (steps + shares - 1) / shares;
    a.rows_per_share = (int)(each * RPW);
    a.shares = (int)((steps + each - 1) / each);
    rope_kernel<TI, TO, VEC, L, UPL>
        <<<cdiv((size_t)a.tokens * a.shares, kRopeWarps), kRopeWarps * 32, 0, st>>>(a);
    WARP_CHECK_LAUNCH("rope_kernel");
    return WARP_OK;
}

// The widest vectors that the row's parts, addresses and strides allow.
template <typename TI, typename TO>
static int rope_vec(RopeArgs &a, cudaStream_t st) {
    auto fits = [&](int vec) {
        const uintptr_t ib = vec * sizeof(TI) < 16 ? vec * sizeof(TI) : 16;
        const uintptr_t ob = vec * sizeof(TO) < 16 ? vec * sizeof(TO) : 16;
        // half layout: whole vectors on both sides of a row's three boundaries;
        // interleaved: a vector is turned whole or not at all
        if (a.rot % (a.interleaved ? vec : 2 * vec) || a.D % (2 * vec)) return false;
        uintptr_t in = 0, out = (uintptr_t)a.q_out | (uintptr_t)a.k_out;
        const uintptr_t wb = vec * sizeof(float) < 16 ? vec * sizeof(float) : 16;
        if (((uintptr_t)a.q_norm | (uintptr_t)a.k_norm) % wb) return false;
        auto add = [&](const void *p, int64_t s0, int64_t s1) {
            if (p) in |= (uintptr_t)p | (uintptr_t)(s0 * sizeof(TI)) | (uintptr_t)(s1 * sizeof(TI));
        };
        add(a.q, a.q_token, a.q_head);
        add(a.k, a.k_token, a.k_head);
        if (a.slots) add(a.v, a.v_token, a.v_head);
        return in % ib == 0 && out % ob == 0;
    };
    // and the fewest lanes that hold a row (4922 tokens, 20 heads of 64, 52 of it
    // turned in halves: 28 us with 32 lanes and vectors of two, 8.4 with 16)
    if (fits(8)) {
        if (a.D <= 64) return rope_launch<TI, TO, 8, 4, 1>(a, st);
        if (a.D <= 128) return rope_launch<TI, TO, 8, 8, 1>(a, st);
        return rope_launch<TI, TO, 8, 16, 1>(a, st);
    }
    if (fits(4)) {
        if (a.D <= 64) return rope_launch<TI, TO, 4, 8, 1>(a, st);
        if (a.D <= 128) return rope_launch<TI, TO, 4, 16, 1>(a, st);
        return rope_launch<TI, TO, 4, 32, 1>(a, st);
    }
    if (fits(2)) {
        if (a.D <= 64) return rope_launch<TI, TO, 2, 16, 1>(a, st);
        if (a.D <= 128) return rope_launch<TI, TO, 2, 32, 1>(a, st);
        return rope_launch<TI, TO, 2, 32, 2>(a, st);
    }
    return rope_launch<TI, TO, 1, 32, 4>(a, st);
}

static int rope_run(const warp_rope_desc *d, const warp_kv_pages *c, const int64_t *slots,
                    const char *who, cudaStream_t st) {
    WARP_ARG(d, "%s: NULL description", who);
    WARP_ARG(d->tokens >= 0 && d->q_heads >= 0 && d->kv_heads >= 0, "%s: negative size", who);
    WARP_ARG(d->head_dim >= 2 && d->head_dim <= 256 && d->head_dim % 2 == 0,
             "%s: head_dim %d is not even in 2..256", who, d->head_dim);
    WARP_ARG(d->rot_dim >= 0 && d->rot_dim <= d->head_dim && d->rot_dim % 2 == 0,
             "%s: rot_dim %d is not even in 0..%d", who, d->rot_dim, d->head_dim);
    WARP_ARG(d->type >= WARP_T_F32 && d->type <= WARP_T_BF16 && d->out_type >= WARP_T_F32 &&
                 d->out_type <= WARP_T_BF16 && (d->type == d->out_type || d->type == WARP_T_F32),
             "%s: type %d to out_type %d (the same type, or from fp32)", who, d->type,
             d->out_type);
    const int rows = d->q_heads + (c ? 2 : 1) * d->kv_heads;
    WARP_ARG(rows <= 65536, "%s: %d heads", who, rows);
    if (d->tokens == 0 || rows == 0) return WARP_OK;
    WARP_ARG(d->positions || d->rot_dim == 0, "%s: NULL positions", who);
    WARP_ARG(d->inv_freq || d->rot_dim == 0, "%s: NULL inv_freq", who);
    WARP_ARG(!d->q_heads || (d->q && d->q_out), "%s: NULL queries", who);
    WARP_ARG(!d->kv_heads || (d->k && (c ? d->v != nullptr : d->k_out != nullptr)),
             "%s: NULL keys or values", who);
    RopeArgs a = {};
    a.q = d->q_heads ? d->q : nullptr;
    a.k = d->kv_heads ? d->k : nullptr;
    a.q_token = d->q_token, a.q_head = d->q_head;
    a.k_token = d->k_token, a.k_head = d->k_head;
    a.q_out = d->q_heads ? d->q_out : nullptr;
    a.q_norm = d->q_norm, a.k_norm = d->k_norm;
    a.inv_freq = d->inv_freq, a.positions = d->positions;
    a.eps = d->eps, a.rot_scale = d->rot_scale;
    a.tokens = d->tokens, a.q_heads = d->q_heads, a.kv_heads = d->kv_heads;
    a.D = d->head_dim, a.rot = d->rot_dim, a.interleaved = d->interleaved != 0;
    a.rows = rows;
    if (c) {
        const int rc = kv_pages_check(c, who);
        if (rc) return rc;
        WARP_ARG(slots, "%s: NULL slots", who);
        WARP_ARG(c->kv_heads == d->kv_heads && c->head_dim == d->head_dim,
                 "%s: the pages hold %d heads of %d, the keys are %d of %d", who, c->kv_heads,
                 c->head_dim, d->kv_heads, d->head_dim);
        WARP_ARG(c->type == d->out_type, "%s: out_type %d is not the pages' %d", who, d->out_type,
                 c->type);
        a.v = d->v, a.v_token = d->v_token, a.v_head = d->v_head;
        a.slots = slots;
        a.kp = c->k, a.vp = c->v;
        a.k_page = c->k_page, a.k_slot = c->k_slot, a.k_ph = c->k_head;
        a.v_page = c->v_page, a.v_slot = c->v_slot, a.v_ph = c->v_head;
        a.n_slots = c->pages * c->page_size;
        a.page_shift = __builtin_ctz(c->page_size);
        const int er = attn_err_word(&a.err);
        if (er) return er;
    } else {
        a.k_out = d->kv_heads ? d->k_out : nullptr;
    }
    if (d->type == WARP_T_F16) return rope_vec<__half, __half>(a, st);
    if (d->type == WARP_T_BF16) return rope_vec<__nv_bfloat16, __nv_bfloat16>(a, st);
    return d->out_type == WARP_T_F16    ? rope_vec<float, __half>(a, st)
           : d->out_type == WARP_T_BF16 ? rope_vec<float, __nv_bfloat16>(a, st)
                                        : rope_vec<float, float>(a, st);
}

// One thread a token; its request by bisection of q_start.  A few microseconds
// once a step, for all layers.
__global__ void kv_slots_kernel(const int32_t *__restrict__ q_start,
                                const int32_t *__restrict__ kv_len, int batch, int tokens,
                                const int32_t *__restrict__ pages, int64_t pages_row,
                                int pages_per_row, int page_shift, int base,
                                int32_t *__restrict__ positions, int64_t *__restrict__ slots) {
    const int t = blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= tokens) return;
    int lo = 0, hi = batch;                 // the last b with q_start[b] <= t
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (q_start[mid] <= t) lo = mid; else hi = mid;
    }
    const int first = q_start[lo], end = q_start[lo + 1];
    int64_t slot = -1;
    int32_t pos = 0;
    if (t >= first && t < end) {
        const int64_t j = (int64_t)kv_len[lo] - end + t;
        pos = (int32_t)(base + j);
        if ((j >> page_shift) >= pages_per_row) {
            atomicOr(&g_attn_err, kAttnBadLen);
        } else if (j >= 0) {
            const int page = pages[lo * pages_row + (j >> page_shift)];
            // a negative slot would pass for a token that is not to be stored
            if (page < 0) atomicOr(&g_attn_err, kAttnBadPage);
            else slot = ((int64_t)page << page_shift) + (j & ((1 << page_shift) - 1));
        }
    }
    positions[t] = pos;
    slots[t] = slot;
}

}  // namespace warp

extern "C" int warp_qk_norm_rope(const warp_rope_desc *d, void *stream) {
    return warp::rope_run(d, nullptr, nullptr, "warp_qk_norm_rope", (cudaStream_t)stream);
}

extern "C" int warp_kv_append(const warp_rope_desc *d, const warp_kv_pages *c,
                              const int64_t *slots, void *stream) {
    WARP_ARG(c, "warp_kv_append: NULL pages");
    return warp::rope_run(d, c, slots, "warp_kv_append", (cudaStream_t)stream);
}

extern "C" int warp_kv_slots(const int32_t *q_start, const int32_t *kv_len, int batch, int tokens,
                             const int32_t *pages, int64_t pages_row, int pages_per_row,
                             int page_size, int base, int32_t *positions, int64_t *slots,
                             void *stream) {
    WARP_ARG(batch >= 0 && tokens >= 0 && pages_per_row >= 0 && pages_row >= 0 && base >= 0,
             "warp_kv_slots: negative size");
    WARP_ARG(page_size >= 16 && page_size <= 4096 && !(page_size & (page_size - 1)),
             "warp_kv_slots: page_size %d is not a power of two in 16..4096", page_size);
    if (tokens == 0) return WARP_OK;
    WARP_ARG(batch >= 1 && q_start && kv_len && positions && slots && (pages || !pages_per_row),
             "warp_kv_slots: NULL pointer or no request");
    warp::kv_slots_kernel<<<warp::cdiv(tokens, 256), 256, 0, (cudaStream_t)stream>>>(
        q_start, kv_len, batch, tokens, pages, pages_row, pages_per_row,
        __builtin_ctz(page_size), base, positions, slots);
    WARP_CHECK_LAUNCH("kv_slots_kernel");
    return WARP_OK;
}

extern "C" int warp_attn_status(int clear) {
    unsigned v = 0;
    // a copy by itself does not wait for streams that do not block the default one
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, warp::g_attn_err, sizeof(v));
    if (e != cudaSuccess) return warp::cuda_fail(e, "warp_attn_status");
    if (clear && v) {
        warp::attn_err_clear_kernel<<<1, 1>>>(v);
        WARP_CHECK_LAUNCH("attn_err_clear_kernel");
        e = cudaDeviceSynchronize();        // before anything that may report anew
        if (e != cudaSuccess) return warp::cuda_fail(e, "warp_attn_status");
    }
    if (v & warp::kAttnTimeout) {
        warp::set_error("attention: a tensor-core wait gave up (flags 0x%x)", v);
        return WARP_E_TIMEOUT;
    }
    if (v) {
        warp::set_error("attention:%s%s%s%s%s",
                        v & warp::kAttnBadSlot ? " a slot outside the pages;" : "",
                        v & warp::kAttnBadPage ? " a page number outside the pages;" : "",
                        v & warp::kAttnNoPage ? " no page left in the pool;" : "",
                        v & warp::kAttnBadTree ? " a parent behind its node;" : "",
                        v & warp::kAttnBadLen ? " a length over its bound" : "");
        return WARP_E_ARG;
    }
    return WARP_OK;
}
