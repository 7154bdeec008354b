// Grouped-query attention over the paged 4-bit cache for few query rows per kv
// head: single tokens and verify batches.
//
// Mathematics. A key row stands for m + s c (c: its codes), so
// q . K = s (q . c) + m sum(q): the product runs on the codes, which bf16 holds
// exactly, and the scale is applied to the fp32 result. In the same way
// sum_j p_j V_j = sum_j (p_j s_j) (c_j - 8) + sum_j p_j (m_j + 8 s_j). The weights
// p_j s_j are the one thing rounded to bf16 (for the tensor core); the second
// sum takes p_j in fp32. c - 8 keeps what the rounding multiplies as small
// as the values themselves. Softmax in base 2 with a running maximum and sum.
//
// Layout of the products: a warp takes 16 positions at a time (a UNIT), the
// positions are the 16 rows of the m16n8k16 MMA and the query rows (8 a
// column block) its columns, so a kv head's few query rows fill the narrow
// side. S^T = K q^T takes the codes straight from global memory: lane (g, t)
// loads 16 bytes of position g's row and of position g + 8's, and the k order that
// this gives is matched when q is packed. P^T goes from the accumulator layout to the
// B operand by movmatrix. O^T = V^T P^T needs pairs of positions for one element:
// the 16-bit halves of two rows' words are put together (prmt) before the
// nibbles are taken apart, so no transposition of V is ever stored. A nibble
// becomes bf16 128 + c by one mask-and-or (0x4300 is 128, whose last mantissa
// bit is 1).
//
// Work split: stream-K. The units of all (sequence, kv head) pairs, in order,
// are cut into equal ranges, one a CTA, whatever the lengths are; the cut is
// computed on the device from the lengths, so one captured graph serves every
// step. A CTA's eight warps take its range's units in turn and are joined in
// shared memory; a pair that spans CTAs is joined by the last of them to
// finish, in CTA order, so that the result does not depend on the timing.
//
// Bound: the codes are read once, 136 bytes a position and kv head (head_dim
// 128). About 230 instructions a warp and unit of 2176 bytes.
#include <algorithm>

#include "kv4.cuh"

namespace dm {
namespace {

constexpr int kWarps = 8;
constexpr int kUnit = 16;          // positions a warp takes at a time
constexpr int kMinUnits = kWarps;  // units a CTA takes at least, where there are that many
constexpr float kLog2e = 1.4426950408889634f;
// A weight may exceed 1 by this power of two before the running maximum is
// raised: one vote a unit instead of a reduction over its positions.
constexpr float kSlack = 8.f;

struct AttnArgs {
    KvView kv;
    const uint16_t *q;
    int64_t qs;
    void *out;
    int32_t nh, grp, out_f32, max_q, nrb;
    float scale;
    int64_t window;
    uint32_t *count;  // [seqs][nkv][nrb] arrivals, zero between launches
    float *part;      // [gridDim.x][2][8 NT][HD + 2]: a CTA's shared first and last pair
};

template <int HD>
struct Unit {
    uint32_t k[2][HD / 32];  // rows g and g + 8, HD / 8 bytes each
    uint32_t v[4][HD / 64];  // positions 2t, 2t + 1, 2t + 8, 2t + 9, HD / 16 bytes each
    uint2 s[2];              // key s, m, value s, m of rows g and g + 8
};

template <int N>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t (&w)[N]) {
    if (N == 4) {
        const uint4 x = __ldg((const uint4 *)p);
        w[0] = x.x, w[1 % N] = x.y, w[2 % N] = x.z, w[3 % N] = x.w;
    } else if (N == 2) {
        const uint2 x = __ldg((const uint2 *)p);
        w[0] = x.x, w[1 % N] = x.y;
    } else {
        w[0] = __ldg((const uint32_t *)p);
    }
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// bf16 pair 128 + c of the nibbles at bits 0-3 and 16-19
__device__ __forceinline__ uint32_t codes128(uint32_t w) { return lop3<0xEA>(w, 0x000F000Fu, 0x43004300u); }
// bf16 pair minus 136: c - 8 (exact)
__device__ __forceinline__ uint32_t less136(uint32_t x) {
    uint32_t y;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x43084308u));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float bf_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf_hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// A sequence as the split sees it.
struct Seq {
    int32_t t0, n, len;  // first token, new tokens, rows
    int32_t u0, units;   // first unit and units (0: no tokens; at least 1 otherwise)
};
__device__ __forceinline__ Seq seq_of(const AttnArgs &a, int b) {
    Seq s;
    s.t0 = a.kv.q_start[b];
    s.n = a.kv.q_start[b + 1] - s.t0;
    s.len = max(a.kv.kv_len[b], 0);
    if (s.t0 < 0 || s.n < 0 || s.n > a.max_q || s.t0 + s.n > a.kv.tokens) {
        if (s.n != 0) atomicExch(a.kv.err, kKvErrRange);
        s.n = 0;
    }
    int64_t lo = 0;
    if (a.window > 0) lo = max((int64_t)0, (int64_t)s.len - s.n - a.window + 1);
    s.u0 = (int32_t)(lo / kUnit);
    s.units = s.n == 0 ? 0 : max(1, (s.len + kUnit - 1) / kUnit - s.u0);
    return s;
}

template <int HD, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 2 : 1) kv4_attn_split_kernel(AttnArgs a) {
    constexpr int R = 8 * NT;        // query rows
    constexpr int KS = HD / 16;      // k steps of S, and element blocks of O
    constexpr int KW = HD / 32, VW = HD / 64;
    constexpr int LD = HD + 4;       // a row of the joined sums (padded)
    extern __shared__ float smem[];
    float *s_o = smem;                       // [kWarps][R][LD]
    float *s_m = s_o + kWarps * R * LD;      // [kWarps][R]
    float *s_l = s_m + kWarps * R;           // [kWarps][R]
    float *s_f = s_l + kWarps * R;           // [kWarps][R]
    int32_t *s_base = (int32_t *)(s_f + kWarps * R);  // [256 + 1] units before a thread's sequences
    __shared__ int s_warp[kWarps];
    __shared__ int s_last;

    pdl_launch_dependents();
    pdl_wait();
    const KvView &kv = a.kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

    // units of the sequences before each thread's, by a scan over the block
    const int per = (kv.seqs + 255) / 256;
    {
        int mine = 0;
        for (int b = tid * per; b < min(kv.seqs, (tid + 1) * per); ++b) mine += seq_of(a, b).units;
        int x = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) s_warp[warp] = x;
        __syncthreads();
        int before = 0;
        for (int w = 0; w < warp; ++w) before += s_warp[w];
        s_base[tid + 1] = before + x;
        if (tid == 0) s_base[0] = 0;
        __syncthreads();
    }
    const int64_t heads = (int64_t)kv.nkv * a.nrb, W = heads * s_base[256];
    if (W == 0) return;
    const int64_t G = min((int64_t)gridDim.x, (W + kMinUnits - 1) / kMinUnits);
    if (blockIdx.x >= G) return;
    int64_t x = blockIdx.x * W / G;
    const int64_t x1 = (blockIdx.x + 1) * W / G;
    int b = 0;
    int64_t seq_x = 0;  // the sequence's first unit in the whole order
    {
        int lo = 0, hi = 256;  // the last thread whose sequences begin at or before x
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (heads * s_base[mid] <= x) lo = mid;
            else hi = mid;
        }
        b = lo * per;
        seq_x = heads * s_base[lo];
    }
    Seq sq = seq_of(a, b);
    const float sl = a.scale * kLog2e;

    while (x < x1) {
        while (x >= seq_x + heads * sq.units) {
            seq_x += heads * sq.units;
            sq = seq_of(a, ++b);
        }
        const int pair = (int)((x - seq_x) / sq.units);  // kv head and row block
        const int h = pair / a.nrb, rb = pair - h * a.nrb;
        const int64_t pair_x = seq_x + (int64_t)pair * sq.units;
        const int u0 = (int)(x - pair_x), u1 = (int)(min(x1, pair_x + sq.units) - pair_x);
        x += u1 - u0;
        const int rows = min(R, sq.n * a.grp - rb * R);  // may be 0 or less: a short sequence of the batch
        const int p0 = sq.len - sq.n;                    // the position of the first new token

        // q as the B operand, and its sums over the head
        uint32_t qf[NT][KS][2];
        float qsum[NT][2];
        int last[NT][2], first[NT][2];  // what columns 2t, 2t + 1 see
        int p_min = INT32_MAX, lo_max = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = rb * R + 8 * n + g, i = r / a.grp;
            const bool live = 8 * n + g < rows;
            const uint16_t *src = a.q + (int64_t)(sq.t0 + (live ? i : 0)) * a.qs +
                                  (int64_t)(h * a.grp + (live ? r - i * a.grp : 0)) * HD + t * (HD / 4);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < KW; ++j) {
                uint4 w = live ? *(const uint4 *)(src + 8 * j) : make_uint4(0, 0, 0, 0);
                sum += ((bf_lo(w.x) + bf_hi(w.x)) + (bf_lo(w.y) + bf_hi(w.y))) +
                       ((bf_lo(w.z) + bf_hi(w.z)) + (bf_lo(w.w) + bf_hi(w.w)));
                qf[n][2 * j][0] = __byte_perm(w.x, w.z, 0x5410);
                qf[n][2 * j][1] = __byte_perm(w.x, w.z, 0x7632);
                qf[n][2 * j + 1][0] = __byte_perm(w.y, w.w, 0x5410);
                qf[n][2 * j + 1][1] = __byte_perm(w.y, w.w, 0x7632);
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                qsum[n][e] = __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4);
                const int p = p0 + (rb * R + 8 * n + 2 * t + e) / a.grp;
                last[n][e] = p;
                first[n][e] = a.window > 0 ? (int)max((int64_t)0, p - a.window + 1) : 0;
            }
        }
        if (rows > 0) {
            p_min = p0 + rb * R / a.grp;
            const int p_max = p0 + (rb * R + rows - 1) / a.grp;
            lo_max = a.window > 0 ? (int)max((int64_t)0, p_max - a.window + 1) : 0;
        }

        float o[KS][NT][4], m[NT][2], l[NT][2], rs[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) m[n][e] = -INFINITY, l[n][e] = 0.f, rs[n][e] = 0.f;
        }

        // this warp's units, the next one's rows in flight while one is computed
        auto page_of = [&](int u) -> int64_t {
            const int64_t p = (int64_t)(sq.u0 + u) * kUnit;
            if (u >= u1 || p >= sq.len || rows <= 0) return -1;
            return kv_page(kv, b, p);
        };
        auto load = [&](Unit<HD> &w, int u, int64_t page) {
            const int slot = ((sq.u0 + u) * kUnit) & (kv.ps - 1);
            const int64_t at = page * kv.nkv + h;
            const uint8_t *k = kv.codes + (at * 2 * kv.ps + slot) * (HD / 2);
            const uint8_t *v = k + (int64_t)kv.ps * (HD / 2);
            const uint2 *s = (const uint2 *)(kv.scales + (at * kv.ps + slot) * 4);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                load_words<KW>(k + (g + 8 * i) * (HD / 2) + t * (HD / 8), w.k[i]);
                w.s[i] = __ldg(s + g + 8 * i);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                load_words<VW>(v + (2 * t + (i & 1) + 8 * (i >> 1)) * (HD / 2) + g * (HD / 16), w.v[i]);
        };
        int u = u0 + warp;
        int64_t page = page_of(u), page_next = page_of(u + kWarps);
        Unit<HD> cur;
        if (page >= 0) load(cur, u, page);
        for (; u < u1; u += kWarps) {
            Unit<HD> nxt;
            const int64_t page2 = page_of(u + 2 * kWarps);
            if (page_next >= 0) load(nxt, u + kWarps, page_next);
            if (page >= 0) {
                const int j0 = (sq.u0 + u) * kUnit;
                float c[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[n][e] = 0.f;
#pragma unroll
                for (int j = 0; j < KW; ++j) {
                    const uint32_t w0 = cur.k[0][j], w1 = cur.k[1][j];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t a0 = codes128(w0 >> (8 * i)), a1 = codes128(w1 >> (8 * i)),
                                       a2 = codes128(w0 >> (8 * i + 4)), a3 = codes128(w1 >> (8 * i + 4));
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            mma_bf16_16816(c[n][0], c[n][1], c[n][2], c[n][3], a0, a1, a2, a3, qf[n][2 * j + i][0],
                                           qf[n][2 * j + i][1]);
                    }
                }
                const bool edge = j0 + kUnit - 1 > p_min || j0 < lo_max;
                float ka[2], kb[2], vs[2], vr[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float ks = bf_lo(cur.s[i].x), km = bf_hi(cur.s[i].x), s = bf_lo(cur.s[i].y);
                    ka[i] = ks * sl;
                    kb[i] = fmaf(-128.f, ks, km) * sl;
                    vs[i] = s;
                    vr[i] = fmaf(8.f, s, bf_hi(cur.s[i].y));
                }
                bool raise = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float s = fmaf(ka[e >> 1], c[n][e], kb[e >> 1] * qsum[n][e & 1]);
                        if (edge) {
                            const int j = j0 + g + 8 * (e >> 1);
                            if (j > last[n][e & 1] || j < first[n][e & 1]) s = -INFINITY;
                        }
                        c[n][e] = s;
                        raise = raise || s > m[n][e & 1] + kSlack;
                    }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float f[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = fmaxf(c[n][e], c[n][e + 2]);
                            for (int k = 4; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
                            top = fmaxf(m[n][e], top);
                            f[e] = m[n][e] == top ? 1.f : exp2_approx(m[n][e] - top);
                            m[n][e] = top;
                            l[n][e] *= f[e];
                            rs[n][e] *= f[e];
                        }
#pragma unroll
                        for (int i = 0; i < KS; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[i][n][e] *= f[e & 1];
                    }
                }
                uint32_t pb[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float wgt[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float top = m[n][e & 1];
                        const float p = exp2_approx(c[n][e] - (top == -INFINITY ? 0.f : top));
                        // a masked row's scales may be anything: they are not multiplied
                        const bool none = edge && c[n][e] == -INFINITY;
                        wgt[e] = none ? 0.f : p * vs[e >> 1];
                        l[n][e & 1] += p;
                        rs[n][e & 1] = none ? rs[n][e & 1] : fmaf(p, vr[e >> 1], rs[n][e & 1]);
                    }
                    pb[n][0] = movmatrix(pack_bf16(wgt[0], wgt[1]));
                    pb[n][1] = movmatrix(pack_bf16(wgt[2], wgt[3]));
                }
#pragma unroll
                for (int j = 0; j < VW; ++j) {
                    const uint32_t lo0 = __byte_perm(cur.v[0][j], cur.v[1][j], 0x5410),
                                   hi0 = __byte_perm(cur.v[0][j], cur.v[1][j], 0x7632),
                                   lo1 = __byte_perm(cur.v[2][j], cur.v[3][j], 0x5410),
                                   hi1 = __byte_perm(cur.v[2][j], cur.v[3][j], 0x7632);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t a0 = less136(codes128(lo0 >> (4 * i))), a1 = less136(codes128(hi0 >> (4 * i))),
                                       a2 = less136(codes128(lo1 >> (4 * i))), a3 = less136(codes128(hi1 >> (4 * i)));
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            mma_bf16_16816(o[4 * j + i][n][0], o[4 * j + i][n][1], o[4 * j + i][n][2],
                                           o[4 * j + i][n][3], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                    }
                }
            }
            cur = nxt;
            page = page_next;
            page_next = page2;
        }

        // the warps' sums into shared memory: element (HD / 8) g + 8 j + i (+ 4), rows 2t, 2t + 1
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                for (int k = 4; k < 32; k <<= 1) {
                    l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], k);
                    rs[n][e] += __shfl_xor_sync(0xffffffffu, rs[n][e], k);
                }
                const int r = 8 * n + 2 * t + e;
                if (g == 0) {
                    s_m[warp * R + r] = m[n][e];
                    s_l[warp * R + r] = l[n][e];
                }
                float *d = s_o + (warp * R + r) * LD + g * (HD / 8);
#pragma unroll
                for (int j = 0; j < VW; ++j) {
                    *(float4 *)(d + 8 * j) =
                        make_float4(o[4 * j][n][e] + rs[n][e], o[4 * j + 1][n][e] + rs[n][e],
                                    o[4 * j + 2][n][e] + rs[n][e], o[4 * j + 3][n][e] + rs[n][e]);
                    *(float4 *)(d + 8 * j + 4) =
                        make_float4(o[4 * j][n][e + 2] + rs[n][e], o[4 * j + 1][n][e + 2] + rs[n][e],
                                    o[4 * j + 2][n][e + 2] + rs[n][e], o[4 * j + 3][n][e + 2] + rs[n][e]);
                }
            }
        __syncthreads();
        // the whole pair: the result. A part of it: {maximum, sum, O} of the rows to
        // the workspace, and the last CTA of the pair joins them.
        const bool whole = u0 == 0 && u1 == sq.units;
        float *mine = a.part + ((int64_t)blockIdx.x * 2 + (u0 == 0 ? 1 : 0)) * (R * (HD + 2));
        auto store = [&](int r, int d4, float4 v) {
            const int rr = rb * R + r, i = rr / a.grp;
            const int64_t at = ((int64_t)(sq.t0 + i) * a.nh + h * a.grp + (rr - i * a.grp)) * HD + 4 * d4;
            if (a.out_f32)
                *(float4 *)((float *)a.out + at) = v;
            else
                *(uint2 *)((uint16_t *)a.out + at) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
        };
        for (int i = tid; i < R * (HD / 4); i += kWarps * 32) {
            const int r = i / (HD / 4), d4 = i % (HD / 4);
            if (r >= rows) break;
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * R + r]);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float mw = s_m[w * R + r], f = mw == top ? 1.f : exp2_approx(mw - top);
                const float4 y = *(const float4 *)(s_o + (w * R + r) * LD + 4 * d4);
                sum = fmaf(f, s_l[w * R + r], sum);
                v.x = fmaf(f, y.x, v.x), v.y = fmaf(f, y.y, v.y), v.z = fmaf(f, y.z, v.z), v.w = fmaf(f, y.w, v.w);
            }
            if (whole) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                store(r, d4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            } else {
                float *dst = mine + r * (HD + 2);
                if (d4 == 0) dst[HD] = top, dst[HD + 1] = sum;
                *(float2 *)(dst + 4 * d4) = make_float2(v.x, v.y);
                *(float2 *)(dst + 4 * d4 + 2) = make_float2(v.z, v.w);
            }
        }
        if (!whole) {
            const int64_t c0 = ((pair_x + 1) * G - 1) / W, c1 = ((pair_x + sq.units) * G - 1) / W;
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                uint32_t *cnt = a.count + ((int64_t)b * kv.nkv + h) * a.nrb + rb;
                s_last = atom_add_acq_rel_gpu(cnt, 1u) == (uint32_t)(c1 - c0);
                if (s_last) *cnt = 0u;  // for the next launch
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                for (int i = tid; i < R * (HD / 4); i += kWarps * 32) {
                    const int r = i / (HD / 4), d4 = i % (HD / 4);
                    if (r >= rows) break;
                    float top = -INFINITY, sum = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (int64_t cc = c0; cc <= c1; ++cc) {
                        const float *src = a.part + (cc * 2 + (cc == c0 ? 1 : 0)) * (R * (HD + 2)) + r * (HD + 2);
                        const float2 ml = __ldcg((const float2 *)(src + HD)), ya = __ldcg((const float2 *)(src + 4 * d4)),
                                     yb = __ldcg((const float2 *)(src + 4 * d4 + 2));
                        const float now = fmaxf(top, ml.x);
                        const float fo = top == now ? 1.f : exp2_approx(top - now),
                                    fn = ml.x == now ? 1.f : exp2_approx(ml.x - now);
                        sum = sum * fo + ml.y * fn;
                        v.x = v.x * fo + ya.x * fn, v.y = v.y * fo + ya.y * fn;
                        v.z = v.z * fo + yb.x * fn, v.w = v.w * fo + yb.y * fn;
                        top = now;
                    }
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    store(r, d4, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                }
            }
        }
        __syncthreads();  // shared memory is written again by the next pair
    }
}

constexpr int split_smem(int hd, int nt) {
    return (kWarps * 8 * nt * (hd + 4) + 3 * kWarps * 8 * nt + 257) * 4;
}

// Column blocks of eight query rows a kernel takes at once, and its CTAs: two
// an SM with one block (registers), one with more.
int split_nt(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }
int split_grid(int nt) { return nt == 1 ? 296 : 148; }

int64_t count_bytes(int64_t seqs, int64_t nkv, int64_t nrb) { return (seqs * nkv * nrb * 4 + 255) / 256 * 256; }

template <int HD, int NT>
cudaError_t launch_split(const AttnArgs &g, void *stream) {
    constexpr int smem = split_smem(HD, NT);
    static bool ready[64];  // the attribute is per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (smem > 48 * 1024 && (dev >= 64 || !ready[dev])) {
        e = cudaFuncSetAttribute(kv4_attn_split_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready[dev] = true;
    }
    return launch_pdl(kv4_attn_split_kernel<HD, NT>, dim3(split_grid(NT)), dim3(kWarps * 32), smem, stream, g);
}

}  // namespace
}  // namespace dm

extern "C" int64_t dm_kv4_workspace_bytes(const dm_kv4_cache *c, int32_t seqs, int32_t max_q, int32_t heads) {
    if (!c || seqs < 1 || max_q < 1 || heads < 1 || c->kv_heads < 1 || heads % c->kv_heads) return -1;
    const int64_t rows = (int64_t)max_q * (heads / c->kv_heads);
    const int nt = dm::split_nt(rows);
    const int64_t nrb = (rows + 8 * nt - 1) / (8 * nt);
    return dm::kKvHead + dm::count_bytes(seqs, c->kv_heads, nrb) +
           (int64_t)dm::split_grid(nt) * 2 * 8 * nt * (c->head_dim + 2) * 4;
}

extern "C" int dm_kv4_attention(const dm_kv4_cache *c, const dm_kv4_batch *b, const void *q, int64_t q_stride,
                                int32_t heads, float scale, int64_t window, void *out, int32_t out_dtype,
                                void *stream, char *err, size_t err_len) {
    using namespace dm;
    const char *who = "dm_kv4_attention";
    if (int rc = kv_check_args(who, c, b, err, err_len)) return rc;
    if (heads < 1 || heads % c->kv_heads || heads > 65536)
        return kv_refuse(err, err_len, "%s: %d heads are no multiple of %d kv heads", who, heads, c->kv_heads);
    if (!q || !out || !kv_aligned(q, 16) || !kv_aligned(out, 16) || q_stride < 0 || q_stride % 8)
        return kv_refuse(err, err_len, "%s: q and out must be 16-byte aligned, q's stride a multiple of 8", who);
    if (out_dtype != DM_BF16 && out_dtype != DM_F32)
        return kv_refuse(err, err_len, "%s: the output must be bf16 or fp32", who);
    if (window < 0) return kv_refuse(err, err_len, "%s: negative window", who);
    if (b->work_bytes < dm_kv4_workspace_bytes(c, b->seqs, b->max_q, heads))
        return kv_refuse(err, err_len, "%s: the workspace is smaller than dm_kv4_workspace_bytes", who);
    if (b->tokens == 0) return DM_OK;
    AttnArgs g;
    g.kv = kv_view(c, b);
    g.q = (const uint16_t *)q;
    g.qs = q_stride;
    g.out = out;
    g.nh = heads;
    g.grp = heads / c->kv_heads;
    g.out_f32 = out_dtype == DM_F32;
    g.max_q = b->max_q;
    g.scale = scale;
    g.window = window;
    const int64_t rows = (int64_t)b->max_q * g.grp;
    const int nt = split_nt(rows);
    g.nrb = (int)((rows + 8 * nt - 1) / (8 * nt));
    g.count = (uint32_t *)((uint8_t *)b->work + kKvHead);
    g.part = (float *)((uint8_t *)b->work + kKvHead + count_bytes(b->seqs, c->kv_heads, g.nrb));
    cudaError_t e;
    if (c->head_dim == 64)
        e = nt == 1 ? launch_split<64, 1>(g, stream) : nt == 2 ? launch_split<64, 2>(g, stream)
                                                               : launch_split<64, 4>(g, stream);
    else
        e = nt == 1 ? launch_split<128, 1>(g, stream) : nt == 2 ? launch_split<128, 2>(g, stream)
                                                                : launch_split<128, 4>(g, stream);
    return kv_launched("kv4_attn_split_kernel", e, err, err_len);
}
