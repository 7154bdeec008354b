// The paged 4-bit key/value cache: appending a step's keys and values with
// the rotary embedding (and the per-head RMSNorm of q and k) on the way, and
// reading rows back as the values they stand for.
//
// Arithmetic: fp32 with every operation rounded by itself (__fmul_rn and the
// like keep the compiler from contracting a product and a sum), sums of squares in
// halving order, so that the codes, which hang on the last bit where a value
// lies between two of them, are the same on every run.
#include "kv4.cuh"

namespace dm {
namespace {

struct AppendArgs {
    KvView kv;
    const void *q, *k, *v;
    int64_t qs, ks, vs;
    int32_t nh, rot, interleaved;
    const uint16_t *qn, *kn;
    const float *cosv, *sinv;
    int64_t positions;
    float eps;
    uint16_t *q_out;
};

__device__ __forceinline__ void unpack8(uint4 w, float x[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ uint4 pack8(const float x[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        u[i] = (uint32_t)f32_to_bf16_bits(x[2 * i]) | ((uint32_t)f32_to_bf16_bits(x[2 * i + 1]) << 16);
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// Eight elements of a row from element `at` on, by 16-byte loads.
template <bool F32>
__device__ __forceinline__ void load8(const void *p, int64_t at, float x[8]) {
    if (F32) {
        const float *f = (const float *)p + at;
        const float4 a = *(const float4 *)f, b = *(const float4 *)(f + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        unpack8(*(const uint4 *)((const uint16_t *)p + at), x);
    }
}

// How a row lies over its L = HD / 8 lanes: eight neighbours a lane, or (PAIRED: the whole head
// turns, pairs (i, i + HD / 2)) four of each half, so that a pair is one lane's.
template <bool F32, bool VEC, bool PAIRED, int HD>
__device__ __forceinline__ void load_row(const void *p, int64_t at, int l, float (&x)[8]) {
    static_assert(VEC || !PAIRED, "pairs are read by vectors");
    if (!PAIRED && VEC) {
        load8<F32>(p, at + 8 * l, x);
    } else if (!PAIRED) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            x[e] = F32 ? ((const float *)p)[at + 8 * l + e] : bf16_bits_to_f32(((const uint16_t *)p)[at + 8 * l + e]);
    } else if (F32) {
        const float4 u = *(const float4 *)((const float *)p + at + 4 * l), v = *(const float4 *)((const float *)p + at + HD / 2 + 4 * l);
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else {
        const uint2 u = *(const uint2 *)((const uint16_t *)p + at + 4 * l), v = *(const uint2 *)((const uint16_t *)p + at + HD / 2 + 4 * l);
        unpack8(make_uint4(u.x, u.y, v.x, v.y), x);
    }
}

// The sum of a row's squares in halving order: element i with i + HD / 2, then with
// + HD / 4, and so on. Where a level pairs lanes, of what two lanes would both compute each
// keeps one half and gives the other away; the levels within a lane come last, as exchanges
// between the classes that the lanes then hold: 11 exchanges (head_dim 128) in
// place of 32, or 7 where a lane holds pairs of the first level.
template <int L, bool PAIRED>
__device__ __forceinline__ float halving_sum(const float (&x)[8], int l, uint32_t mask) {
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = __fmul_rn(x[e], x[e]);
    constexpr int HELD = PAIRED ? 4 : 8;  // neighbours that a lane holds
    if (PAIRED)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = __fadd_rn(s[e], s[e + 4]);
#pragma unroll
    for (int o = L / 2, n = HELD / 2; o > 0; o >>= 1, n >>= 1) {
        if (n > 0) {  // n values are kept
            const bool up = l & o;
#pragma unroll
            for (int e = 0; e < n; ++e) {
                const float mine = up ? s[e + n] : s[e], theirs = up ? s[e] : s[e + n];
                s[e] = __fadd_rn(mine, __shfl_xor_sync(mask, theirs, o));
            }
        } else {
            s[0] = __fadd_rn(s[0], __shfl_xor_sync(mask, s[0], o));
        }
    }
#pragma unroll
    for (int o = L / 2, n = HELD / 2; n > 0; o >>= 1, n >>= 1) s[0] = __fadd_rn(s[0], __shfl_xor_sync(mask, s[0], o));
    return s[0];
}

// HD / 8 lanes per head row, eight elements a lane. A block takes one token and every
// gridDim.y-th group of 256 / (HD / 8) of its rows (the q heads, then, in groups of
// their own, the keys and values): the token's sequence, position and rotary row are looked up
// once, the next group's row is on its way while one is computed.
//
// Bound: the rows in and out. 3781 tokens of 64 + 2 x 8 heads (head_dim 128): 165 MB with their
// reading back, 25 us at 6.57 TB/s; measured 52 us and 8.3 for the reading (2.7 TB/s). The instructions
// limit it, issued at 68 % of what the schedulers can: about 130 per two rows of a warp for
// the norm and the rotation, one element at a time and none contracted, and 70 to
// load, pack and place them. One token takes 4.6 us with its reading back, two launches' time.
// Rows held as pairs against eight neighbours a lane (us): 3781 tokens 61 and 80, 512 tokens 9.1 and 11.8.
template <int HD, bool F32, bool VEC, bool PAIRED>
__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int L = HD / 8, RB = 256 / L;
    pdl_launch_dependents();
    pdl_wait();
    const KvView &kv = a.kv;
    const int t = blockIdx.x, lane = threadIdx.x & 31, l = threadIdx.x & (L - 1), in = threadIdx.x / L;
    const uint32_t mine = ((1u << L) - 1u) << (lane & ~(L - 1));  // the row's lanes
    const int qg = (a.nh + RB - 1) / RB, groups = qg + (2 * kv.nkv + RB - 1) / RB;
    const int64_t qrow = (int64_t)t * a.qs, krow = (int64_t)t * a.ks, vrow = (int64_t)t * a.vs;
    float nx[8];
    auto fetch = [&](int g) {
        const int r = (g < qg ? g : g - qg) * RB + in;
#pragma unroll
        for (int e = 0; e < 8; ++e) nx[e] = 0.f;
        if (g < qg) {
            if (r < a.nh) load_row<F32, VEC, PAIRED, HD>(a.q, qrow + r * HD, l, nx);
        } else if (r < kv.nkv) {
            load_row<F32, VEC, PAIRED, HD>(a.k, krow + r * HD, l, nx);
        } else if (r < 2 * kv.nkv) {
            load_row<F32, VEC, PAIRED, HD>(a.v, vrow + (r - kv.nkv) * HD, l, nx);
        }
    };
    int g = blockIdx.y;
    fetch(g);
    const int b = kv_sequence(kv, t, lane);
    const bool none = b >= kv.seqs || t < kv.q_start[b];
    const int64_t p = none ? -1 : (int64_t)kv.kv_len[b] - (kv.q_start[b + 1] - t);
    const bool bad = a.rot && p >= a.positions, turns = a.rot && p >= 0 && !bad;
    if (bad && threadIdx.x == 0) atomicExch(kv.err, kKvErrRange);
    const bool rows = p >= 0 && !bad;  // there are rows to write
    // the angles of this lane's elements
    const int hl = a.rot / 16;          // lanes of half the rotated part
    const bool first = l < hl, turn = turns && (PAIRED || 8 * l < a.rot);
    constexpr int NC = PAIRED ? 4 : 8;
    float c[NC], s[NC];
#pragma unroll
    for (int e = 0; e < NC; ++e) c[e] = s[e] = 0.f;
    if (turn) {
        const float *cp = a.cosv + p * (a.rot / 2), *sp = a.sinv + p * (a.rot / 2);
        if (PAIRED || a.interleaved) {
            const float4 c4 = *(const float4 *)(cp + 4 * l), s4 = *(const float4 *)(sp + 4 * l);
            c[0] = c4.x, c[1] = c4.y, c[2] = c4.z, c[3] = c4.w, s[0] = s4.x, s[1] = s4.y, s[2] = s4.z, s[3] = s4.w;
        } else if constexpr (!PAIRED) {
            const int i0 = 8 * (first ? l : l - hl);
            load8<true>(cp, i0, c);
            load8<true>(sp, i0, s);
            if (first)  // u - o s = u + o (-s)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[e] = -s[e];
        }
    }
    auto norm = [&](float (&x)[8], const float (&w)[8]) {
        const float ss = halving_sum<L, PAIRED>(x, l, mine);
        const float r = __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(ss, 1.0f / HD), a.eps)));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(__fmul_rn(x[e], r), w[e]);
    };
    auto rotate = [&](float (&x)[8], bool now) {  // the row's lanes together
        if constexpr (PAIRED) {
            if (now)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y1 = x[e], y2 = x[e + 4];
                    x[e] = __fsub_rn(__fmul_rn(y1, c[e]), __fmul_rn(y2, s[e]));
                    x[e + 4] = __fadd_rn(__fmul_rn(y2, c[e]), __fmul_rn(y1, s[e]));
                }
        } else if (a.interleaved) {
            if (now && turn)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y1 = x[2 * i], y2 = x[2 * i + 1];
                    x[2 * i] = __fsub_rn(__fmul_rn(y1, c[i]), __fmul_rn(y2, s[i]));
                    x[2 * i + 1] = __fadd_rn(__fmul_rn(y2, c[i]), __fmul_rn(y1, s[i]));
                }
        } else {
            const int from = (lane & ~(L - 1)) + (turn ? (first ? l + hl : l - hl) : l);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float o = __shfl_sync(0xffffffffu, x[e], from);
                const float y = __fadd_rn(__fmul_rn(x[e], c[e]), __fmul_rn(o, s[e]));
                if (now && turn) x[e] = y;
            }
        }
    };
    auto next = [&](float (&x)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = nx[e];
        if (g + (int)gridDim.y < groups) fetch(g + gridDim.y);
    };

    if (g < qg) {
        float w[8];
        if (a.qn) load_row<false, VEC, PAIRED, HD>(a.qn, 0, l, w);
        uint16_t *out = a.q_out + (int64_t)t * a.nh * HD + (PAIRED ? 4 : 8) * l;
        for (; g < qg; g += gridDim.y) {
            float x[8];
            next(x);
            if (a.qn) norm(x, w);
            if (turns) rotate(x, true);  // the whole block: p is its token's
            const int r = g * RB + in;
            if (r >= a.nh) continue;
            uint4 y = pack8(x);
            if (!rows) y = make_uint4(0u, 0u, 0u, 0u);
            if (PAIRED) {
                *(uint2 *)(out + r * HD) = make_uint2(y.x, y.y);
                *(uint2 *)(out + r * HD + HD / 2) = make_uint2(y.z, y.w);
            } else {
                *(uint4 *)(out + r * HD) = y;
            }
        }
    }
    if (g >= groups) return;
    const int64_t page = rows ? kv_page(kv, b, p) : -1;
    const int slot = (int)(p & (kv.ps - 1));
    for (; g < groups; g += gridDim.y) {
        float x[8];
        next(x);
        const int r = (g - qg) * RB + in;
        const bool key = r < kv.nkv, row = r < 2 * kv.nkv;
        if (a.kn && key) {  // not uniform over a warp: the exchanges are among the row's own lanes
            float w[8];
            load_row<false, VEC, PAIRED, HD>(a.kn, 0, l, w);
            norm(x, w);
        }
        __syncwarp();
        if (turns) rotate(x, key);
        float lo = x[0], hi = x[0];
        bool fin = true;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            lo = fminf(lo, x[e]);
            hi = fmaxf(hi, x[e]);
            fin = fin && isfinite(x[e]);
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const uint32_t finite = __ballot_sync(0xffffffffu, fin);
        if (!row || page < 0) continue;
        uint16_t mb = f32_to_bf16_bits(lo), sb = f32_to_bf16_bits(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
        const float m = bf16_bits_to_f32(mb), sc = bf16_bits_to_f32(sb);
        uint32_t word = 0;
        if ((finite & mine) != mine || !isfinite(sc) || !isfinite(m)) {
            mb = sb = 0x7fc0;  // NaN
        } else if (sc < 1.17549435e-38f) {
            sb = 0;
        } else {
            const float inv = __frcp_rn(sc);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float k = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[e], m), inv)), 0.f), 15.f);
                word |= (uint32_t)(int)k << (4 * e);
            }
        }
        const int part = key ? 0 : 1;
        const int64_t at = page * kv.nkv + (key ? r : r - kv.nkv);
        uint8_t *dst = kv.codes + ((at * 2 + part) * kv.ps + slot) * (HD / 2);
        if (PAIRED) {
            *(uint16_t *)(dst + 2 * l) = (uint16_t)word;
            *(uint16_t *)(dst + HD / 4 + 2 * l) = (uint16_t)(word >> 16);
        } else {
            *(uint32_t *)(dst + 4 * l) = word;
        }
        if (l == 0) *(uint32_t *)(kv.scales + (at * kv.ps + slot) * 4 + 2 * part) = (uint32_t)sb | ((uint32_t)mb << 16);
    }
}

// A block per token and 256 / (HD / 8) rows (key and value of each kv head). Bound by
// what it reads and writes: 3781 tokens of 8 kv heads of 128, 19.6 MB, in 8.3 us (2.4 TB/s; 1.9 us are a launch's).
template <int HD, bool F32>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ KvView kv, void *k_out, void *v_out) {
    constexpr int L = HD / 8;
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, lane = threadIdx.x & 31, l = threadIdx.x & (L - 1);
    const int r = blockIdx.y * (256 / L) + threadIdx.x / L;
    const int b = kv_sequence(kv, t, lane);
    if (r >= 2 * kv.nkv) return;
    const int h = r >> 1, part = r & 1;
    void *out = part ? v_out : k_out;
    if (!out) return;
    const bool none = b >= kv.seqs || t < kv.q_start[b];
    const int64_t p = none ? -1 : (int64_t)kv.kv_len[b] - (kv.q_start[b + 1] - t);
    const int64_t page = p < 0 ? -1 : kv_page(kv, b, p);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (page >= 0) {
        const int slot = (int)(p & (kv.ps - 1));
        const int64_t at = page * kv.nkv + h;
        const uint32_t word = *(const uint32_t *)(kv.codes + ((at * 2 + part) * kv.ps + slot) * (HD / 2) + 4 * l);
        const uint32_t sm = *(const uint32_t *)(kv.scales + (at * kv.ps + slot) * 4 + 2 * part);
        const float s = __uint_as_float(sm << 16), m = __uint_as_float(sm & 0xffff0000u);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(__fmul_rn((float)((word >> (4 * e)) & 15u), s), m);
    }
    const int64_t o = ((int64_t)t * kv.nkv + h) * HD + 8 * l;
    if (F32) {
        float4 *f = (float4 *)((float *)out + o);
        f[0] = make_float4(x[0], x[1], x[2], x[3]);
        f[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *(uint4 *)((uint16_t *)out + o) = pack8(x);
    }
}

template <int HD, bool F32>
cudaError_t launch_append(const AppendArgs &a, bool vec, dim3 grid, void *stream) {
    if (!vec) return launch_pdl(kv4_append_kernel<HD, F32, false, false>, grid, dim3(256), 0, stream, a);
    return a.rot == HD && !a.interleaved ? launch_pdl(kv4_append_kernel<HD, F32, true, true>, grid, dim3(256), 0, stream, a)
                                         : launch_pdl(kv4_append_kernel<HD, F32, true, false>, grid, dim3(256), 0, stream, a);
}

}  // namespace
}  // namespace dm

extern "C" int dm_kv4_append(const dm_kv4_cache *c, const dm_kv4_batch *b, const dm_kv4_append_args *a, void *stream,
                             char *err, size_t err_len) {
    using namespace dm;
    const char *who = "dm_kv4_append";
    if (int rc = kv_check_args(who, c, b, err, err_len)) return rc;
    if (!a || !a->k || !a->v) return kv_refuse(err, err_len, "%s: null keys or values", who);
    const int heads = a->q ? a->heads : 0;
    if (a->q && (heads < 1 || heads > 65536 || !a->q_out || !kv_aligned(a->q_out, 16)))
        return kv_refuse(err, err_len, "%s: q needs heads and a 16-byte aligned q_out", who);
    if (a->in_dtype != DM_BF16 && a->in_dtype != DM_F32)
        return kv_refuse(err, err_len, "%s: the inputs must be bf16 or fp32", who);
    if (a->rot < 0 || a->rot > c->head_dim || a->rot % 16)
        return kv_refuse(err, err_len, "%s: rot must be a multiple of 16 up to head_dim, not %d", who, a->rot);
    if (a->rot && (!a->cos_table || !a->sin_table || a->positions < 1 || !kv_aligned(a->cos_table, 16) ||
                   !kv_aligned(a->sin_table, 16)))
        return kv_refuse(err, err_len, "%s: the rotary tables must be given, 16-byte aligned", who);
    if (a->k_stride < 0 || a->v_stride < 0 || a->q_stride < 0)
        return kv_refuse(err, err_len, "%s: negative stride", who);
    if (b->tokens == 0) return DM_OK;
    const bool f32 = a->in_dtype == DM_F32;
    const int64_t step = f32 ? 4 : 8;  // elements of 16 bytes
    const bool vec = kv_aligned(a->q_norm, 16) && kv_aligned(a->k_norm, 16) && kv_aligned(a->k, 16) && kv_aligned(a->v, 16) && a->k_stride % step == 0 &&
                     a->v_stride % step == 0 && (!a->q || (kv_aligned(a->q, 16) && a->q_stride % step == 0));
    AppendArgs g;
    g.kv = kv_view(c, b);
    g.q = a->q, g.k = a->k, g.v = a->v;
    g.qs = a->q_stride, g.ks = a->k_stride, g.vs = a->v_stride;
    g.nh = heads, g.rot = a->rot, g.interleaved = a->interleaved;
    g.qn = (const uint16_t *)a->q_norm, g.kn = (const uint16_t *)a->k_norm;
    g.cosv = a->cos_table, g.sinv = a->sin_table, g.positions = a->positions;
    g.eps = a->eps;
    g.q_out = (uint16_t *)a->q_out;
    const int per = 256 / (c->head_dim / 8);
    // blocks a token: as many as fill the GPU (four an SM), one for prompts. With the reading back (us),
    // as chosen, one a token, one a group of rows: 64 tokens 5.6, 7.0, 5.6; 3781 tokens 61, 61, 80
    const int64_t groups = (heads + per - 1) / per + (2 * c->kv_heads + per - 1) / per, fill = (4 * 148 + b->tokens - 1) / b->tokens;
    const dim3 grid((unsigned)b->tokens, (unsigned)(fill < groups ? fill : groups));
    const cudaError_t e = c->head_dim == 64 ? (f32 ? launch_append<64, true>(g, vec, grid, stream) : launch_append<64, false>(g, vec, grid, stream))
                                            : (f32 ? launch_append<128, true>(g, vec, grid, stream) : launch_append<128, false>(g, vec, grid, stream));
    return kv_launched("kv4_append_kernel", e, err, err_len);
}

extern "C" int dm_kv4_read(const dm_kv4_cache *c, const dm_kv4_batch *b, void *k_out, void *v_out, int32_t out_dtype,
                           void *stream, char *err, size_t err_len) {
    using namespace dm;
    const char *who = "dm_kv4_read";
    if (int rc = kv_check_args(who, c, b, err, err_len)) return rc;
    if (!k_out && !v_out) return kv_refuse(err, err_len, "%s: no output", who);
    if (!kv_aligned(k_out, 16) || !kv_aligned(v_out, 16))
        return kv_refuse(err, err_len, "%s: the outputs must be 16-byte aligned", who);
    if (out_dtype != DM_BF16 && out_dtype != DM_F32)
        return kv_refuse(err, err_len, "%s: the outputs must be bf16 or fp32", who);
    if (b->tokens == 0) return DM_OK;
    const KvView v = kv_view(c, b);
    const int per = 256 / (c->head_dim / 8);
    const dim3 grid((unsigned)b->tokens, (unsigned)((2 * c->kv_heads + per - 1) / per));
    cudaError_t e;
    if (c->head_dim == 64)
        e = out_dtype == DM_F32 ? launch_pdl(kv4_read_kernel<64, true>, grid, dim3(256), 0, stream, v, k_out, v_out)
                                : launch_pdl(kv4_read_kernel<64, false>, grid, dim3(256), 0, stream, v, k_out, v_out);
    else
        e = out_dtype == DM_F32 ? launch_pdl(kv4_read_kernel<128, true>, grid, dim3(256), 0, stream, v, k_out, v_out)
                                : launch_pdl(kv4_read_kernel<128, false>, grid, dim3(256), 0, stream, v, k_out, v_out);
    return kv_launched("kv4_read_kernel", e, err, err_len);
}

extern "C" int dm_kv4_check(int32_t *error, int32_t *device_error, void *stream, char *err, size_t err_len) {
    using namespace dm;
    if (!error || !device_error) return kv_refuse(err, err_len, "dm_kv4_check: null pointer");
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e = cudaMemcpyAsync(device_error, error, 4, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(error, 0, 4, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    return kv_launched("dm_kv4_check", e, err, err_len);
}
