// Grouped-query attention over the paged 4-bit cache for few query rows per kv
// head: single tokens and verify batches.
//
// Mathematics. A key row stands for m + s c (c: its codes), so
// q . K = s (q . c) + m sum(q): the product runs on the codes and the scale is
// applied afterwards in fp32. The codes go to the integer tensor core as bytes (a
// word of eight needs two masks and a shift); q becomes 16-bit integers by a
// power of two per row (exact for elements down to 2^-7 of the row's largest,
// within 2^-16 of it below; sum(q) is that of the integers, so what is
// rounded away meets the key values and not their codes), as a signed high and an
// unsigned low byte, and the sums are exact. For the values, sum_j p_j V_j = sum_j (p_j s_j) (c_j - 8) + sum_j p_j (m_j + 8 s_j):
// the weights p_j s_j are rounded to bf16 (for the tensor core), the second
// sum takes p_j in fp32, and c - 8 keeps what the rounding multiplies as small
// as the values themselves. A nibble becomes bf16 128 + c by one mask-and-or
// (0x4300 is 128, whose last mantissa bit is 1); the 136 too much is taken off every 16
// positions, by a second MMA with -136 in every place or from the operand itself, so the
// fp32 sums stay as small as the result. Softmax in base 2 with a running
// maximum and sum.
//
// Layout of the products: a warp takes 16 positions at a time (a UNIT), the
// positions are the 16 rows of the MMA and the query rows (8 a column block)
// its columns, so a kv head's few query rows fill the narrow side. S^T = K q^T:
// lane (g, t) reads 16 bytes of position g's row and of position g + 8's,
// and the k order that this gives is matched when q is packed. P^T goes from
// the accumulator layout to the B operand by movmatrix. O^T = V^T P^T needs pairs
// of positions for one element: the 16-bit halves of two rows' words are put together
// (prmt) before the nibbles are taken apart, so no transposition of V is ever stored.
//
// Each warp streams its units through a ring of its own in shared memory
// (cp.async, three units ahead), value rows with their 16-byte pieces
// exchanged so that the reads of four positions fall on different banks.
//
// Work split: the units of all (sequence, kv head) pairs, in order, are cut
// into equal ranges, one a CTA (stream-K), or, while every pair's pieces of
// eight units fit the grid, into those pieces (one unit a warp: the shortest
// chain). The cut is computed on the device from the lengths, so one captured
// graph serves every step. A CTA's eight warps take its units in turn and are joined in
// shared memory; a pair that spans CTAs is joined by the last of them to finish, in CTA
// order, so the result does not depend on the timing.
//
// Bound: the codes are read once, 136 bytes a position and kv head (head_dim 128).
#include <type_traits>

#include "kv4.cuh"

namespace dm {
namespace {

constexpr int kWarps = 8;
constexpr int kUnit = 16;  // positions a warp takes at a time
constexpr int kRing = 4;   // units a warp holds in shared memory
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

constexpr int unit_bytes(int hd) { return 2 * kUnit * (hd / 2) + kUnit * 8; }

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// D += A (16 x 32 unsigned bytes, row) * B (32 x 8 bytes, col), int32
template <bool SIGNED>
__device__ __forceinline__ void mma_u8_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    if (SIGNED)
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// Byte `i` of four integers
template <int I>
__device__ __forceinline__ uint32_t bytes_of(int a, int b, int c, int d) {
    const uint32_t ab = __byte_perm(a, b, I | ((4 + I) << 4)), cd = __byte_perm(c, d, I | ((4 + I) << 4));
    return __byte_perm(ab, cd, 0x5410);
}

__device__ __forceinline__ void ring_copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ring_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void lds(uint32_t at, uint32_t (&w)[N]) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
    else
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at));
}

// Byte of 16-byte piece `c` of value row r in a unit's copy: pieces exchanged
// so that rows 2t (t = 0 .. 3) fall on different banks.
template <int HD>
__device__ __forceinline__ uint32_t value_piece(int r, int c) {
    if (HD == 128) return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
    return (uint32_t)((r >> 2) * 128 + ((((r & 3) * 2 + c) ^ (((r >> 2) & 1) << 1)) << 4));
}

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
constexpr int region_bytes() {  // a warp's shared memory: its ring, and its sums when it is done
    constexpr int sums = 8 * NT * (HD + 4) * 4, ring = kRing * unit_bytes(HD);
    return ((sums > ring ? sums : ring) + 127) / 128 * 128;
}
template <int HD, int NT>
constexpr int split_smem() {
    return kWarps * region_bytes<HD, NT>() + NT * (HD / 32) * 512 + 2 * 8 * NT * 4 + 2 * kWarps * 8 * NT * 4 + 257 * 4;
}

template <int HD, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 2 : 1) kv4_attn_split_kernel(AttnArgs a) {
    constexpr int R = 8 * NT;        // query rows
    constexpr int KS = HD / 16;      // element blocks of O
    constexpr int KW = HD / 32, VW = HD / 64;
    constexpr int LD = HD + 4;       // a row of a warp's sums (padded)
    constexpr int UB = unit_bytes(HD), KB = kUnit * (HD / 2);
    constexpr bool kLess = NT > 1;   // 136 off the operand (once a unit) or by an MMA (once a column block)
    constexpr int RB = region_bytes<HD, NT>();
    extern __shared__ __align__(128) uint8_t smem[];
    uint4 *s_q = (uint4 *)(smem + kWarps * RB);       // [NT][KW][32]: B operands, first and rest
    float *s_qs = (float *)(s_q + NT * KW * 32);      // [R] sums of q
    float *s_qf = s_qs + R;                           // [R] what undoes the row's power of two
    float *s_m = s_qf + R;                            // [kWarps][R]
    float *s_l = s_m + kWarps * R;                    // [kWarps][R]
    int32_t *s_base = (int32_t *)(s_l + kWarps * R);  // [256 + 1] cells before a thread's sequences
    __shared__ int2 s_warp[kWarps];
    __shared__ int s_last;

    pdl_launch_dependents();
    pdl_wait();
    const KvView &kv = a.kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

    // cells (units, or pieces of eight) of the sequences before each thread's
    const int per = (kv.seqs + 255) / 256;
    const int64_t heads = (int64_t)kv.nkv * a.nrb;
    bool pieces;
    {
        int units = 0, eights = 0;
        for (int b = tid * per; b < min(kv.seqs, (tid + 1) * per); ++b) {
            const int n = seq_of(a, b).units;
            units += n;
            eights += (n + kWarps - 1) / kWarps;
        }
        int x = units, y = eights;
        for (int o = 1; o < 32; o <<= 1) {
            const int xu = __shfl_up_sync(0xffffffffu, x, o), yu = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) x += xu, y += yu;
        }
        if (lane == 31) s_warp[warp] = make_int2(x, y);
        __syncthreads();
        int all = 0, before_x = 0, before_y = 0;
        for (int w = 0; w < kWarps; ++w) {
            const int2 v = s_warp[w];
            if (w < warp) before_x += v.x, before_y += v.y;
            all += v.y;
        }
        pieces = heads * all <= gridDim.x;
        s_base[tid + 1] = pieces ? before_y + y : before_x + x;
        if (tid == 0) s_base[0] = 0;
        __syncthreads();
    }
    const int64_t W = heads * s_base[256], G = min((int64_t)gridDim.x, W);
    if (blockIdx.x >= G) return;
    int64_t x = blockIdx.x * W / G;
    const int64_t x1 = (blockIdx.x + 1) * W / G;
    int b = 0;
    int64_t seq_x = 0;  // the sequence's first cell in the whole order
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
    auto cells_of = [&](const Seq &s) { return pieces ? (s.units + kWarps - 1) / kWarps : s.units; };
    int cells = cells_of(sq);
    const float sl = a.scale * kLog2e;
    const uint32_t ring = smem_addr(smem + warp * RB);
    float *const s_o = (float *)(smem + warp * RB);
    // where this lane's copies go and its reads are, in a unit's copy
    constexpr int PR = HD / 32;  // 16-byte pieces of a row
    const uint32_t v_dst = KB + value_piece<HD>(lane / PR, lane % PR);
    const uint32_t k_src = ring + g * (HD / 2) + t * (HD / 8);
    uint32_t v_src[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        v_src[i] = ring + KB + value_piece<HD>(2 * t + i, g * (HD / 16) / 16) + (g * (HD / 16)) % 16;

    while (x < x1) {
        while (x >= seq_x + heads * cells) {
            seq_x += heads * cells;
            sq = seq_of(a, ++b);
            cells = cells_of(sq);
        }
        const int pair = (int)((x - seq_x) / cells);  // kv head and row block
        const int h = pair / a.nrb, rb = pair - h * a.nrb;
        const int64_t pair_x = seq_x + (int64_t)pair * cells;
        int u0 = (int)(x - pair_x), u1 = (int)(min(x1, pair_x + cells) - pair_x);
        x += u1 - u0;
        if (pieces) {  // even pieces of the pair's units
            u0 = (int)((int64_t)u0 * sq.units / cells);
            u1 = (int)((int64_t)u1 * sq.units / cells);
        }
        const int rows = min(R, sq.n * a.grp - rb * R);  // may be 0 or less: a short sequence of the batch
        const int p0 = sq.len - sq.n;                    // the position of the first new token

        // the warp's units u0 + warp, + 8, ...: pages are looked up 32 units at
        // a time, a lane each, one batch ahead
        auto pages_of = [&](int u) -> int {
            u += kWarps * lane;
            const int64_t p = (int64_t)(sq.u0 + u) * kUnit;
            return u >= u1 || p >= sq.len || rows <= 0 ? -1 : (int)kv_page(kv, b, p);
        };
        int u_ahead = u0 + warp, batch_ahead = 0;  // the next unit to copy, its place in the batch of pages
        int pages = pages_of(u_ahead), pages_next = pages_of(u_ahead + 32 * kWarps);
        uint32_t fill = 0;     // ring slot of the next copy
        uint32_t have = 0;     // bit i: the unit copied i units ago has rows
        auto copy = [&]() {
            const int page = __shfl_sync(0xffffffffu, pages, batch_ahead);
            if (page >= 0) {
                const int slot = ((sq.u0 + u_ahead) * kUnit) & (kv.ps - 1);
                const int64_t at = (int64_t)page * kv.nkv + h;
                const uint8_t *k = kv.codes + (at * 2 * kv.ps + slot) * (HD / 2) + lane * 16;
                const uint8_t *v = k + kv.ps * (HD / 2);
                const uint32_t dst = ring + fill * UB;
                ring_copy16(dst + lane * 16, k);
                ring_copy16(dst + v_dst, v);
                if (HD == 128) {
                    ring_copy16(dst + lane * 16 + 512, k + 512);
                    ring_copy16(dst + v_dst + 512, v + 512);
                }
                if (lane < 8)
                    ring_copy16(dst + 2 * KB + lane * 16, (const uint8_t *)(kv.scales + (at * kv.ps + slot) * 4) + lane * 16);
            }
            ring_commit();
            have = (have << 1) | (page >= 0 ? 1u : 0u);
            fill = fill + 1 == kRing ? 0 : fill + 1;
            u_ahead += kWarps;
            if (++batch_ahead == 32) {
                batch_ahead = 0;
                pages = pages_next;
                pages_next = pages_of(u_ahead + 32 * kWarps);
            }
        };
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) copy();

        // q as the B operand: its two parts, its sum and its power of two; warp n
        // takes column block n
        if (warp < NT) {
            const int n = warp, r = rb * R + 8 * n + g, i = r / a.grp;
            const bool live = 8 * n + g < rows;
            const uint16_t *src = a.q + (int64_t)(sq.t0 + (live ? i : 0)) * a.qs +
                                  (int64_t)(h * a.grp + (live ? r - i * a.grp : 0)) * HD + t * (HD / 4);
            uint4 w[KW];
            float top = 0.f;
            bool fin = true;
#pragma unroll
            for (int j = 0; j < KW; ++j) {
                w[j] = live ? *(const uint4 *)(src + 8 * j) : make_uint4(0, 0, 0, 0);
                const uint32_t u[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    top = fmaxf(top, fmaxf(fabsf(bf_lo(u[k])), fabsf(bf_hi(u[k]))));
                    fin = fin && isfinite(bf_lo(u[k])) && isfinite(bf_hi(u[k]));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            fin = (__ballot_sync(0xffffffffu, fin) >> (lane & ~3) & 15u) == 15u;
            // 2^(14 - floor(log2 top)), kept where its inverse is a normal number
            const int e = fin ? min(268 - (int)(__float_as_uint(top) >> 23), 253) : 127;
            const float up = __uint_as_float((uint32_t)e << 23);
            int sum = 0;
#pragma unroll
            for (int j = 0; j < KW; ++j) {
                // word j of the lane's part of a row: codes 0, 2, 4, 6 are operand register 0, the odd ones 1
                int v[8];
                const uint32_t u[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[2 * k] = __float2int_rn(bf_lo(u[k]) * up);
                    v[2 * k + 1] = __float2int_rn(bf_hi(u[k]) * up);
                    sum += v[2 * k] + v[2 * k + 1];
                }
                s_q[(n * KW + j) * 32 + lane] =
                    make_uint4(bytes_of<1>(v[0], v[2], v[4], v[6]), bytes_of<1>(v[1], v[3], v[5], v[7]),
                               bytes_of<0>(v[0], v[2], v[4], v[6]), bytes_of<0>(v[1], v[3], v[5], v[7]));
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (t == 0) {
                const float down = __uint_as_float((uint32_t)(254 - e) << 23) * sl;
                s_qs[8 * n + g] = fin ? (float)sum * down : NAN;  // a row that is not finite stays so
                s_qf[8 * n + g] = down;
            }
        }
        int p_min = INT32_MAX, lo_max = 0;
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
        __syncthreads();
        uint4 qreg[KW];
        float qs_[NT][2], qf_[NT][2];
        if (NT == 1) {
#pragma unroll
            for (int j = 0; j < KW; ++j) qreg[j] = s_q[j * 32 + lane];
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) qs_[n][e] = s_qs[8 * n + 2 * t + e], qf_[n][e] = s_qf[8 * n + 2 * t + e];

        // one unit out of ring slot `at`; EDGE: some of its positions are hidden
        // from some rows
        auto compute = [&](uint32_t at, int j0, auto edge_tag) {
            constexpr bool EDGE = decltype(edge_tag)::value;
            float c[NT][4];
            int hi[NT][4], lo[NT][4];
            uint32_t k0[KW], k1[KW], sc0[2], sc1[2];
            lds(k_src + at, k0);
            lds(k_src + at + 8 * (HD / 2), k1);
            lds(ring + at + 2 * KB + g * 8, sc0);
            lds(ring + at + 2 * KB + g * 8 + 64, sc1);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) hi[n][e] = lo[n][e] = 0;
#pragma unroll
            for (int j = 0; j < KW; ++j) {
                const uint32_t a0 = k0[j] & 0x0f0f0f0fu, a1 = k1[j] & 0x0f0f0f0fu, a2 = (k0[j] >> 4) & 0x0f0f0f0fu,
                               a3 = (k1[j] >> 4) & 0x0f0f0f0fu;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint4 qb = NT == 1 ? qreg[j] : s_q[(n * KW + j) * 32 + lane];
                    mma_u8_16832<true>(hi[n], a0, a1, a2, a3, qb.x, qb.y);
                    mma_u8_16832<false>(lo[n], a0, a1, a2, a3, qb.z, qb.w);
                }
            }
            const float ks[2] = {bf_lo(sc0[0]), bf_lo(sc1[0])}, km[2] = {bf_hi(sc0[0]), bf_hi(sc1[0])};
            const float vs[2] = {bf_lo(sc0[1]), bf_lo(sc1[1])};
            const float vr[2] = {fmaf(8.f, vs[0], bf_hi(sc0[1])), fmaf(8.f, vs[1], bf_hi(sc1[1]))};
            bool raise = false, hide[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float s = fmaf(ks[e >> 1] * (float)(hi[n][e] * 256 + lo[n][e]), qf_[n][e & 1], km[e >> 1] * qs_[n][e & 1]);
                    if (EDGE) {
                        const int j = j0 + g + 8 * (e >> 1), p = p0 + (rb * R + 8 * n + 2 * t + (e & 1)) / a.grp;
                        hide[n][e] = j > p || j >= sq.len || (a.window > 0 && j <= p - a.window);
                        if (hide[n][e]) s = -INFINITY;
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
                    float p = exp2_approx(c[n][e] - m[n][e & 1]);
                    float r = p * vr[e >> 1];
                    wgt[e] = p * vs[e >> 1];
                    // a hidden row's scales may be anything, and a maximum may not be there yet
                    if (EDGE && hide[n][e]) p = 0.f, r = 0.f, wgt[e] = 0.f;
                    l[n][e & 1] += p;
                    rs[n][e & 1] += r;
                }
                pb[n][0] = movmatrix(pack_bf16(wgt[0], wgt[1]));
                pb[n][1] = movmatrix(pack_bf16(wgt[2], wgt[3]));
            }
            uint32_t v[4][VW];
            lds(v_src[0] + at, v[0]);
            lds(v_src[1] + at, v[1]);
            lds(v_src[0] + at + 8 * (HD / 2), v[2]);
            lds(v_src[1] + at + 8 * (HD / 2), v[3]);
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const uint32_t lo0 = __byte_perm(v[0][j], v[1][j], 0x5410), hi0 = __byte_perm(v[0][j], v[1][j], 0x7632),
                               lo1 = __byte_perm(v[2][j], v[3][j], 0x5410), hi1 = __byte_perm(v[2][j], v[3][j], 0x7632);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t a0 = codes128(lo0 >> (4 * i)), a1 = codes128(hi0 >> (4 * i)), a2 = codes128(lo1 >> (4 * i)),
                             a3 = codes128(hi1 >> (4 * i));
                    if (kLess) a0 = less136(a0), a1 = less136(a1), a2 = less136(a2), a3 = less136(a3);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float(&d)[4] = o[4 * j + i][n];
                        mma_bf16_16816(d[0], d[1], d[2], d[3], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                        if (!kLess)  // -136 in every place
                            mma_bf16_16816(d[0], d[1], d[2], d[3], 0xC308C308u, 0xC308C308u, 0xC308C308u, 0xC308C308u,
                                           pb[n][0], pb[n][1]);
                    }
                }
            }
        };
        uint32_t at = 0;
        for (int u = u0 + warp; u < u1; u += kWarps) {
            ring_wait<kRing - 2>();
            __syncwarp();  // the unit's copies are everyone's, and the slot filled next has been read
            copy();
            const int j0 = (sq.u0 + u) * kUnit;
            if ((have >> (kRing - 1)) & 1) {
                if (j0 + kUnit - 1 > p_min || j0 < lo_max)
                    compute(at, j0, std::true_type{});
                else
                    compute(at, j0, std::false_type{});
            }
            at = at + UB == kRing * UB ? 0 : at + UB;
        }
        ring_wait<0>();
        __syncwarp();

        // the warp's sums into its shared memory: element (HD / 8) g + 8 j + i (+ 4), rows 2t, 2t + 1
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
                float *d = s_o + r * LD + g * (HD / 8);
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
            const int64_t to = ((int64_t)(sq.t0 + i) * a.nh + h * a.grp + (rr - i * a.grp)) * HD + 4 * d4;
            if (a.out_f32)
                *(float4 *)((float *)a.out + to) = v;
            else
                *(uint2 *)((uint16_t *)a.out + to) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
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
                const float4 y = *(const float4 *)((const float *)(smem + w * RB) + r * LD + 4 * d4);
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
            const int64_t c0 = ((pair_x + 1) * G - 1) / W, c1 = ((pair_x + cells) * G - 1) / W;
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
        __syncthreads();  // shared memory is written again for the next pair
    }
}

// Column blocks of eight query rows a kernel takes at once, and its CTAs: two
// an SM with one block (registers), one with more.
int split_nt(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }
int split_grid(int nt) { return nt == 1 ? 296 : 148; }

int64_t count_bytes(int64_t seqs, int64_t nkv, int64_t nrb) { return (seqs * nkv * nrb * 4 + 255) / 256 * 256; }

template <int HD, int NT>
cudaError_t launch_split(const AttnArgs &g, void *stream) {
    constexpr int smem = split_smem<HD, NT>();
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
