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
// Layout of the products: a warp takes 32 positions at a time (a UNIT), 16 are
// the rows of an MMA and the query rows (8 a column block) its columns, so a kv head's few query rows fill the narrow side. S^T = K q^T:
// lane (g, t) reads 16 bytes of position g's row and of position g + 8's,
// and the k order that this gives is matched when q is packed. P^T goes from
// the accumulator layout to the B operand by movmatrix. O^T = V^T P^T needs pairs
// of positions for one element: the 16-bit halves of two rows' words are put together
// (prmt) before the nibbles are taken apart, so no transposition of V is ever stored.
//
// Each warp streams its units through three slots of its own in shared memory
// (cp.async, two units in flight while one is computed), value rows with their 16-byte pieces
// exchanged so that the reads of four positions fall on different banks.
//
// Work split: the units of all (sequence, kv head) pairs, in order, are cut
// into equal ranges, one a CTA (stream-K). While it fits the grid, a pair's cut
// is its own instead: one CTA up to 1024 positions, pieces of 256 above, or of
// 512 where only those fit. The cut is computed on the device
// from the lengths, so one captured graph serves every step. A CTA's eight
// warps take its units in turn and are joined in shared memory; a pair that
// spans CTAs is joined by the last of them to finish, in CTA order, so the
// result does not depend on the timing.
//
// In the figures B x L is B sequences, the first of L positions, the others spread down
// to a quarter of it. Both sides of the split's rules, measured with 32 heads on 8 kv
// heads, one token (us, each pair together, before rows of no sequence were looked for: 0.1
// to 0.2 more since): one CTA for 1000 positions 10.0, pieces of 256 12.4 (joining costs more
// than the warps' four units each), one CTA for 4000 25.7, pieces 12.6; pieces of 256 for 4000
// 12.6, of 512 13.7, of 128 13.5; 16000 in pieces of 512 16.2, cut evenly 17.0.
//
// Bound: the codes are read once, 136 bytes a position and kv head (head_dim 128): 32 x 8192
// is 182 MB, 27.7 us at 6.57 TB/s. Measured 58.5 us (3.1 TB/s), and 49.8 for one of 131071 with
// 64 heads (143 MB, 2.9 TB/s). What limits it is not the memory but issue: about 650 instructions a
// unit (300 of them on the ALU: codes to operands, weights, the layout's changes), at 0.54 a cycle and
// scheduler; 16 warps an SM are what the registers allow. Short calls (10 us for 1000 positions) are a chain of
// waits: 4.5 us from the launch to the first product (lengths, the cut, q, the first rows), then the units, then
// 2 to 7 us for the warps' and the CTAs' join.
#include <type_traits>

#include "kv4_attention.cuh"

namespace dm {
namespace {

constexpr int kWarps = 8;        // of a CTA
constexpr int kUnit = 32;  // positions a warp takes at a time
constexpr int kHalf = 16;  // ... and an MMA has rows
constexpr int kWhole = 32; // units of a pair that one CTA takes without a cut
constexpr int kFine = 8, kCoarse = 16;  // units of a piece of a longer pair
constexpr int kMostCtas = 296;  // two an SM
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
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same, D = A * B
template <bool SIGNED>
__device__ __forceinline__ void mma_u8_16832_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                   uint32_t b0, uint32_t b1) {
    if (SIGNED)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}

// D += A (16 x 16 bf16, row) * B (16 x 8 bf16, col), fp32
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Byte `i` of four integers
template <int I>
__device__ __forceinline__ uint32_t bytes_of(int a, int b, int c, int d) {
    const uint32_t ab = __byte_perm(a, b, I | ((4 + I) << 4)), cd = __byte_perm(c, d, I | ((4 + I) << 4));
    return __byte_perm(ab, cd, 0x5410);
}

// N words of shared memory (a plain load: the compiler may move it among the arithmetic)
template <int N>
__device__ __forceinline__ void lds(const uint8_t *at, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 x = *(const uint4 *)at;
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (N == 2) {
        const uint2 x = *(const uint2 *)at;
        w[0] = x.x, w[1] = x.y;
    } else {
        w[0] = *(const uint32_t *)at;
    }
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
__device__ __forceinline__ Seq seq_of(const AttnArgs &a, int b, const Tokens &q) {
    Seq s;
    s.t0 = q.t0, s.n = q.n;
    s.len = max(a.kv.kv_len[b], 0);
    if (s.n * (int64_t)a.grp > a.few) s.n = 0;  // the prompt kernel's
    int64_t lo = 0;
    if (a.window > 0) lo = max((int64_t)0, (int64_t)s.len - s.n - a.window + 1);
    s.u0 = (int32_t)(lo / kUnit);
    // (rows past what the table covers are not there)
    const int64_t covered = (int64_t)a.kv.cols << a.kv.pshift;
    if (s.len > covered && s.n > 0) atomicExch(a.kv.err, kKvErrRange);
    s.units = s.n == 0 ? 0 : max(1, (int)((min((int64_t)s.len, covered) + kUnit - 1) / kUnit) - s.u0);
    return s;
}
__device__ __forceinline__ Seq seq_of(const AttnArgs &a, int b) { return seq_of(a, b, tokens_of(a, b)); }

// A warp's shared memory: three units; its sums lie in the third when its units are done.
template <int HD, int NT>
constexpr int region_bytes() {
    constexpr int sums = 8 * NT * (HD + 4) * 4;
    return 2 * unit_bytes(HD) + (sums > unit_bytes(HD) ? sums : unit_bytes(HD));
}
template <int HD, int NT>
constexpr int split_smem() {  // ... the operands of q, maxima and sums, the CTAs' factors
    return kWarps * region_bytes<HD, NT>() + NT * (HD / 32) * 512 + 2 * 8 * NT * 4 + 2 * kWarps * 8 * NT * 4;
}

// A pair's units [u0, u1) for this CTA, and where it stands in the order of
// cells. Each warp keeps its own in shared memory: nothing of it is needed
// from register to register in the loop over the units.
struct Segment {
    Seq sq;
    int b, h, u0, u1, cells, rows, p0;
    int64_t pair_x, seq_x, x, x1;  // first cells of the pair and the sequence, the next cell, the CTA's last
    int64_t W, G;                  // all cells, and the CTAs that take some
    int piece;                     // units of a piece, 0 where a cell is a unit
};

// Four elements of row r of a pair, divided by the row's sum (0: nothing was seen).
template <int HD>
__device__ __forceinline__ void store_out(const AttnArgs &a, int r, int h, int t0, int d4, float sum, float4 v) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    v.x *= inv, v.y *= inv, v.z *= inv, v.w *= inv;
    const int i = r / a.grp;
    const int64_t to = ((int64_t)(t0 + i) * a.nh + h * a.grp + (r - i * a.grp)) * HD + 4 * d4;
    if (a.out_f32)
        *(float4 *)((float *)a.out + to) = v;
    else
        *(uint2 *)((uint16_t *)a.out + to) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

// The parts of a pair that CTAs c0 .. c0 + nc - 1 left in the workspace, joined
// in their order by the whole CTA. The factors [nc][R] lie in the warps' places for sums
// (`place`, `stride` floats apart). A function of its own: its registers are not the loop's.
template <int HD, int NT>
__device__ __noinline__ void join_parts(const AttnArgs &a, int c0, int nc, int rows, int h, int t0, float *place,
                                        int stride, float *sums) {
    constexpr int R = 8 * NT, RP = HD + 4;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // CTA c0 + c's part: its second slot for the first CTA, its first for the others
    auto part_of = [&](int c, int r) {
        return a.part + ((int64_t)(c0 + c) * 2 + (c == 0 ? 1 : 0)) * (R * RP) + r * RP;
    };
    auto fac = [&](int c, int r) -> float & { return place[(c / HD) * stride + (c % HD) * R + r]; };
    __threadfence();
    for (int r = warp; r < rows; r += kWarps) {  // a warp a row
        constexpr int MOST = (kMostCtas + 31) / 32;
        float2 ml[MOST];
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < MOST; ++i)
            ml[i] = lane + 32 * i < nc ? __ldcg((const float2 *)(part_of(lane + 32 * i, r) + HD)) : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int i = 0; i < MOST; ++i) top = fmaxf(top, ml[i].x);
        for (int k = 1; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
            const float f = ml[i].x == top ? 1.f : exp2_approx(ml[i].x - top);
            if (lane + 32 * i < nc) fac(lane + 32 * i, r) = f;
            sum = fmaf(f, ml[i].y, sum);
        }
        for (int k = 1; k < 32; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        if (lane == 0) sums[r] = sum;
    }
    __syncthreads();
    for (int i = tid; i < rows * (HD / 4); i += kWarps * 32) {
        const int r = i / (HD / 4), d4 = i % (HD / 4);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < nc; c += 16) {  // sixteen parts in flight
            float4 y[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) y[k] = __ldcg((const float4 *)(part_of(min(c + k, nc - 1), r) + 4 * d4));
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const float f = c + k < nc ? fac(c + k, r) : 0.f;
                if (c + k < nc) {
                    v.x = fmaf(f, y[k].x, v.x), v.y = fmaf(f, y[k].y, v.y);
                    v.z = fmaf(f, y[k].z, v.z), v.w = fmaf(f, y[k].w, v.w);
                }
            }
        }
        store_out<HD>(a, r, h, t0, d4, sums[r], v);
    }
}

template <int HD, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 2 : 1) kv4_attn_split_kernel(const __grid_constant__ AttnArgs a) {
    constexpr int R = 8 * NT;        // query rows
    constexpr int KS = HD / 16;      // element blocks of O
    constexpr int KW = HD / 32, VW = HD / 64;
    constexpr int LD = HD + 4;       // a row of a warp's sums (padded)
    constexpr int UB = unit_bytes(HD), KB = kUnit * (HD / 2), HB = kHalf * (HD / 2);
    constexpr bool kLess = NT > 1;   // 136 off the operand (once a unit) or by an MMA (once a column block)
    constexpr int RP = HD + 4;       // floats of a row in the workspace: O, maximum, sum (16-byte aligned)
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int RB = region_bytes<HD, NT>();
    auto sums_of = [&](int w) { return (float *)(smem + w * RB + 2 * UB); };  // [R][LD]
    uint4 *s_q = (uint4 *)(smem + kWarps * RB);        // [NT][KW][32]: B operands, high and low bytes
    float *s_qs = (float *)(s_q + NT * KW * 32);       // [R] sums of q
    float *s_qf = s_qs + R;                            // [R] what undoes the row's power of two
    float *s_m = s_qf + R;                             // [kWarps][R]
    float *s_l = s_m + kWarps * R;                     // [kWarps][R]
    __shared__ int4 s_warp[kWarps];
    __shared__ Segment s_seg[kWarps], s_begin;
    __shared__ int s_last, s_rest;

    pdl_launch_dependents();
    pdl_wait();
    const KvView &kv = a.kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

    // cells (units, or pieces) of the sequences before each thread's
    const int per = (kv.seqs + 255) / 256;
    const int64_t heads = kv.nkv;
    auto pieces_of = [](int units, int piece) { return units <= kWhole ? min(units, 1) : (units + piece - 1) / piece; };
    auto cells_of = [&](int units, int piece) { return piece ? pieces_of(units, piece) : units; };
    {
        int units = 0, fine = 0, coarse = 0;
        bool rest = false;
        Seq mine{};
        for (int b = tid * per; b < min(kv.seqs, (tid + 1) * per); ++b) {
            const Tokens q = tokens_of(a, b);
            mine = seq_of(a, b, q);
            rest = rest || q.rest;
            units += mine.units;
            fine += pieces_of(mine.units, kFine), coarse += pieces_of(mine.units, kCoarse);
        }
        int u = units, f = fine, c = coarse;
        for (int o = 1; o < 32; o <<= 1) {
            const int ou = __shfl_up_sync(0xffffffffu, u, o), of = __shfl_up_sync(0xffffffffu, f, o),
                      oc = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) u += ou, f += of, c += oc;
        }
        if (lane == 31) s_warp[warp] = make_int4(u, f, c, 0);
        rest = __syncthreads_or(rest);
        int all_u = 0, all_f = 0, all_c = 0, before_u = 0, before_f = 0, before_c = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const int4 v = s_warp[w];
            if (w < warp) before_u += v.x, before_f += v.y, before_c += v.z;
            all_u += v.x, all_f += v.y, all_c += v.z;
        }
        if (tid == 0) s_rest = rest;
        const int piece = heads * all_f <= gridDim.x ? kFine : heads * all_c <= gridDim.x ? kCoarse : 0;
        const int all = piece == kFine ? all_f : piece ? all_c : all_u;
        const int here = piece == kFine ? fine : piece ? coarse : units;  // this thread's cells
        const int upto = piece == kFine ? before_f + f : piece ? before_c + c : before_u + u;
        const int64_t W = heads * all, G = min((int64_t)gridDim.x, W);
        if (blockIdx.x >= G) {
            if (rest) zero_rest<HD>(a);
            return;
        }
        const int64_t x = blockIdx.x * W / G;
        // the thread whose sequences hold x finds the one
        const int64_t end = heads * upto;
        int64_t begin = end - heads * here;
        if (begin <= x && x < end) {
            int b = tid * per;
            if (per > 1)
                for (;; ++b) {
                    mine = seq_of(a, b);
                    const int64_t n = heads * cells_of(mine.units, piece);
                    if (x < begin + n) break;
                    begin += n;
                }
            Segment w{};
            w.sq = mine, w.b = b, w.seq_x = begin, w.x = x, w.x1 = (blockIdx.x + 1) * W / G;
            w.W = W, w.G = G, w.piece = piece;
            s_begin = w;
        }
        __syncthreads();
    }
    Segment &sg = s_seg[warp];
    auto next_segment = [&](const Segment &from) {
        Segment w = from;
        __syncwarp();
        for (;;) {
            w.cells = cells_of(w.sq.units, w.piece);
            if (w.x < w.seq_x + heads * w.cells) break;
            w.seq_x += heads * w.cells;
            w.sq = seq_of(a, ++w.b);
        }
        w.h = (int)((w.x - w.seq_x) / w.cells);
        w.pair_x = w.seq_x + (int64_t)w.h * w.cells;
        w.u0 = (int)(w.x - w.pair_x);
        w.u1 = (int)(min(w.x1, w.pair_x + w.cells) - w.pair_x);
        w.x += w.u1 - w.u0;
        if (w.piece) {  // even pieces of the pair's units
            w.u0 = (int)((int64_t)w.u0 * w.sq.units / w.cells);
            w.u1 = (int)((int64_t)w.u1 * w.sq.units / w.cells);
        }
        w.rows = min(R, w.sq.n * a.grp);
        w.p0 = w.sq.len - w.sq.n;  // the position of the first new token
        if (lane == 0) sg = w;
        __syncwarp();
    };

    const float sl = a.scale * kLog2e;
    const uint32_t ring = smem_addr(smem + warp * RB);
    float *const my_o = sums_of(warp);
    // where this lane's copies go and its reads are, in a unit's copy
    constexpr int PR = HD / 32;  // 16-byte pieces of a row
    const uint32_t v_dst = KB + value_piece<HD>(lane / PR, lane % PR);
    const uint8_t *const slots = smem + warp * RB;
    const uint8_t *const k_src = slots + g * (HD / 2) + t * (HD / 8);
    const uint8_t *v_src[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        v_src[i] = slots + KB + value_piece<HD>(2 * t + i, g * (HD / 16) / 16) + (g * (HD / 16)) % 16;

    // The warp's units of a segment: u0 + warp, + 8, ... Pages are looked up 16
    // units at a time, a lane each half of a unit, one batch ahead.
    int u_ahead = 0, at_batch = 0, pages = -1, pages_next = -1;
    uint32_t have = 0;  // bits 1, 0: whether the halves of the unit copied last have rows; two more for each before it
    auto pages_of = [&](int u) -> int {
        u += kWarps * (lane & 15);
        const int64_t p = (int64_t)(sg.sq.u0 + u) * kUnit + kHalf * (lane >> 4);
        return u >= sg.u1 || p >= sg.sq.len ? -1 : (int)kv_page(kv, sg.b, p, first_seen(a, sg.p0) - (kHalf - 1));
    };
    auto copy = [&](uint32_t to) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int page = __shfl_sync(0xffffffffu, pages, at_batch + 16 * half);
            have = (have << 1) | (page >= 0 ? 1u : 0u);
            if (page < 0) continue;
            const int slot = ((sg.sq.u0 + u_ahead) * kUnit + kHalf * half) & (kv.ps - 1);
            const int64_t at = (int64_t)page * kv.nkv + sg.h;
            const uint8_t *k = kv.codes + (at * 2 * kv.ps + slot) * (HD / 2) + lane * 16;
            const uint8_t *v = k + kv.ps * (HD / 2);
            const uint32_t dst = ring + to + half * HB;
            ring_copy16(dst + lane * 16, k);
            ring_copy16(dst + v_dst, v);
            if (HD == 128) {
                ring_copy16(dst + lane * 16 + 512, k + 512);
                ring_copy16(dst + v_dst + 512, v + 512);
            }
            if (lane < 8)
                ring_copy16(ring + to + 2 * KB + half * (kHalf * 8) + lane * 16,
                            (const uint8_t *)(kv.scales + (at * kv.ps + slot) * 4) + lane * 16);
        }
        ring_commit();
        u_ahead += kWarps;
        if (++at_batch == 16) {
            at_batch = 0;
            pages = pages_next;
            pages_next = pages_of(u_ahead + 16 * kWarps);
        }
    };
    auto begin_segment = [&]() {
        u_ahead = sg.u0 + warp;
        at_batch = 0;
        pages = pages_of(u_ahead);
        pages_next = pages_of(u_ahead + 16 * kWarps);
        copy(0);
        copy(UB);
    };
    // q's rows for the B operand: warp n takes column block n
    uint4 qw[KW];
    auto load_q = [&]() {
        if (warp >= NT) return;
        const int r = 8 * warp + g, i = r / a.grp;
        const bool live = r < sg.rows;
        const uint16_t *src = a.q + (int64_t)(sg.sq.t0 + (live ? i : 0)) * a.qs +
                              (int64_t)(sg.h * a.grp + (live ? r - i * a.grp : 0)) * HD + t * (HD / 4);
#pragma unroll
        for (int j = 0; j < KW; ++j) qw[j] = live ? *(const uint4 *)(src + 8 * j) : make_uint4(0, 0, 0, 0);
    };

    next_segment(s_begin);
    load_q();
    begin_segment();
    for (;;) {
        // q as the B operand: its two bytes, its sum and its power of two
        if (warp < NT) {
            const int n = warp;
            float top = 0.f;
            bool fin = true;
#pragma unroll
            for (int j = 0; j < KW; ++j) {
                const uint32_t u[4] = {qw[j].x, qw[j].y, qw[j].z, qw[j].w};
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
                const uint32_t u[4] = {qw[j].x, qw[j].y, qw[j].z, qw[j].w};
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
        // units [in0, in1) are whole and in every row's sight: row 0's last position, the last row's first
        const int lo_max = a.window > 0 ? (int)max((int64_t)0, (int64_t)sg.p0 + (sg.rows - 1) / a.grp - a.window + 1) : 0;
        const int in0 = (lo_max + kUnit - 1) / kUnit - sg.sq.u0, in1 = max(0, sg.p0 + 1) / kUnit - sg.sq.u0;
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
        if (NT == 1) {
#pragma unroll
            for (int j = 0; j < KW; ++j) qreg[j] = s_q[j * 32 + lane];
        }
        const float2 qs1 = *(const float2 *)(s_qs + 2 * t), qf1 = *(const float2 *)(s_qf + 2 * t);
        auto qs_ = [&](int n, int e) { return NT == 1 ? (e ? qs1.y : qs1.x) : s_qs[8 * n + 2 * t + e]; };
        auto qf_ = [&](int n, int e) { return NT == 1 ? (e ? qf1.y : qf1.x) : s_qf[8 * n + 2 * t + e]; };

        // one unit out of the slot at `at`; EDGE: some of its positions are hidden
        // from some rows (live: its halves that have rows)
        auto compute = [&](uint32_t at, int u, uint32_t live, auto edge_tag) {
            constexpr bool EDGE = decltype(edge_tag)::value;
            const int j0 = EDGE ? (sg.sq.u0 + u) * kUnit : 0;
            // halves together (more in flight), or one after the other (fewer registers)
            constexpr int TOG = NT == 1 ? 2 : 1;
#pragma unroll
            for (int h0 = 0; h0 < 2; h0 += TOG) {
                float c[TOG][NT][4];
                bool raise = false, hide[TOG][NT][4];
#pragma unroll
                for (int i = 0; i < TOG; ++i) {
                    const int hf = h0 + i;
                    uint32_t k0[KW], k1[KW], sm[2][1];  // sm: key s, m of rows g and g + 8
                    int acc[NT][4];
                    lds(k_src + at + hf * HB, k0);
                    lds(k_src + at + hf * HB + 8 * (HD / 2), k1);
                    lds(slots + at + 2 * KB + hf * (kHalf * 8) + g * 8, sm[0]);
                    lds(slots + at + 2 * KB + hf * (kHalf * 8) + g * 8 + 64, sm[1]);
                    // the high bytes' sums, times 256, plus the low bytes': one chain with few
                    // registers, two with one column block
                    int low[NT == 3 ? 1 : NT][4];
#pragma unroll
                    for (int pass = 0; pass < (NT == 3 ? 2 : 1); ++pass) {
#pragma unroll
                        for (int j = 0; j < KW; ++j) {
                            const uint32_t a0 = k0[j] & 0x0f0f0f0fu, a1 = k1[j] & 0x0f0f0f0fu,
                                           a2 = (k0[j] >> 4) & 0x0f0f0f0fu, a3 = (k1[j] >> 4) & 0x0f0f0f0fu;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const uint4 qb = NT == 1 ? qreg[j] : s_q[(n * KW + j) * 32 + lane];
                                if (NT == 3) {
                                    if (pass == 0 && j == 0) mma_u8_16832_first<true>(acc[n], a0, a1, a2, a3, qb.x, qb.y);
                                    else if (pass == 0) mma_u8_16832<true>(acc[n], a0, a1, a2, a3, qb.x, qb.y);
                                    else mma_u8_16832<false>(acc[n], a0, a1, a2, a3, qb.z, qb.w);
                                } else if (j == 0) {
                                    mma_u8_16832_first<true>(acc[n], a0, a1, a2, a3, qb.x, qb.y);
                                    mma_u8_16832_first<false>(low[n], a0, a1, a2, a3, qb.z, qb.w);
                                } else {
                                    mma_u8_16832<true>(acc[n], a0, a1, a2, a3, qb.x, qb.y);
                                    mma_u8_16832<false>(low[n], a0, a1, a2, a3, qb.z, qb.w);
                                }
                            }
                        }
                        if (NT == 3 && pass == 0)
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[n][e] *= 256;
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int dot = NT == 3 ? acc[n][e] : acc[n][e] * 256 + low[n][e];
                            float s = fmaf(bf_lo(sm[e >> 1][0]) * (float)dot, qf_(n, e & 1),
                                           bf_hi(sm[e >> 1][0]) * qs_(n, e & 1));
                            if (EDGE) {
                                const int j = j0 + kHalf * hf + g + 8 * (e >> 1),
                                          p = sg.p0 + (8 * n + 2 * t + (e & 1)) / a.grp;
                                hide[i][n][e] = j > p || j >= sg.sq.len || (a.window > 0 && j <= p - a.window) ||
                                                !((live >> (1 - hf)) & 1);
                                if (hide[i][n][e]) s = -INFINITY;
                            }
                            c[i][n][e] = s;
                            raise = raise || s > m[n][e & 1] + kSlack;
                        }
                }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float f[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = m[n][e];
#pragma unroll
                            for (int i = 0; i < TOG; ++i) top = fmaxf(top, fmaxf(c[i][n][e], c[i][n][e + 2]));
                            for (int k = 4; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
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
#pragma unroll
                for (int i = 0; i < TOG; ++i) {
                    const int hf = h0 + i;
                    uint32_t pb[NT][2], sm[2][1];  // value s, m
                    lds(slots + at + 2 * KB + hf * (kHalf * 8) + g * 8 + 4, sm[0]);
                    lds(slots + at + 2 * KB + hf * (kHalf * 8) + g * 8 + 68, sm[1]);
                    const float vs[2] = {bf_lo(sm[0][0]), bf_lo(sm[1][0])};
                    const float vr[2] = {fmaf(8.f, vs[0], bf_hi(sm[0][0])), fmaf(8.f, vs[1], bf_hi(sm[1][0]))};
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float wgt[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float p = exp2_approx(c[i][n][e] - m[n][e & 1]);
                            wgt[e] = p * vs[e >> 1];
                            // a hidden row's scales may be anything, and a maximum may not be there yet
                            if (EDGE && hide[i][n][e]) p = 0.f, wgt[e] = 0.f;
                            l[n][e & 1] += p;
                            rs[n][e & 1] = EDGE && hide[i][n][e] ? rs[n][e & 1] : fmaf(p, vr[e >> 1], rs[n][e & 1]);
                        }
                        pb[n][0] = movmatrix(pack_bf16(wgt[0], wgt[1]));
                        pb[n][1] = movmatrix(pack_bf16(wgt[2], wgt[3]));
                    }
                    uint32_t v[4][VW];
                    lds(v_src[0] + at + hf * HB, v[0]);
                    lds(v_src[1] + at + hf * HB, v[1]);
                    lds(v_src[0] + at + hf * HB + 8 * (HD / 2), v[2]);
                    lds(v_src[1] + at + hf * HB + 8 * (HD / 2), v[3]);
#pragma unroll
                    for (int j = 0; j < VW; ++j) {
                        const uint32_t lo0 = __byte_perm(v[0][j], v[1][j], 0x5410),
                                       hi0 = __byte_perm(v[0][j], v[1][j], 0x7632),
                                       lo1 = __byte_perm(v[2][j], v[3][j], 0x5410),
                                       hi1 = __byte_perm(v[2][j], v[3][j], 0x7632);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t a0 = codes128(lo0 >> (4 * k)), a1 = codes128(hi0 >> (4 * k)),
                                     a2 = codes128(lo1 >> (4 * k)), a3 = codes128(hi1 >> (4 * k));
                            if (kLess) a0 = less136(a0), a1 = less136(a1), a2 = less136(a2), a3 = less136(a3);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                mma_bf16(o[4 * j + k][n], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                                if (!kLess)  // -136 in every place
                                    mma_bf16(o[4 * j + k][n], 0xC308C308u, 0xC308C308u, 0xC308C308u, 0xC308C308u,
                                             pb[n][0], pb[n][1]);
                            }
                        }
                    }
                }
            }
        };
        uint32_t at = 0, to = 2 * UB;
        const int u1 = sg.u1;
        for (int u = sg.u0 + warp; u < u1; u += kWarps) {
            copy(to);  // the slot read in the last turn
            ring_wait<2>();
            __syncwarp();  // the unit's copies are everyone's
            const uint32_t live = (have >> 4) & 3u;
            if (live) {
                if (live != 3u || u < in0 || u >= in1)
                    compute(at, u, live, std::true_type{});
                else
                    compute(at, u, live, std::false_type{});
            }
            to = at;
            at = at == 2 * UB ? 0 : at + UB;
            __syncwarp();  // the slot has been read
        }
        ring_wait<0>();

        // the warp's sums into shared memory: element (HD / 8) g + 8 j + i (+ 4), rows 2t, 2t + 1
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
                float *d = my_o + r * LD + g * (HD / 8);
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
        const Segment was = sg;
        const int rows = was.rows;
        const bool more = was.x < was.x1;
        if (more) {  // the next pair's first rows are on their way while this one is joined
            next_segment(sg);
            load_q();
            begin_segment();
        }
        __syncthreads();
        // the whole pair: the result. A part of it: {maximum, sum, O} of the rows to
        // the workspace, and the last CTA of the pair joins them.
        const bool whole = was.u0 == 0 && was.u1 == was.sq.units;
        float *mine = a.part + ((int64_t)blockIdx.x * 2 + (was.u0 == 0 ? 1 : 0)) * (R * RP);
        for (int i = tid; i < rows * (HD / 4); i += kWarps * 32) {
            const int r = i / (HD / 4), d4 = i % (HD / 4);
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * R + r]);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float mw = s_m[w * R + r], f = mw == top ? 1.f : exp2_approx(mw - top);
                const float4 y = *(const float4 *)(sums_of(w) + r * LD + 4 * d4);
                sum = fmaf(f, s_l[w * R + r], sum);
                v.x = fmaf(f, y.x, v.x), v.y = fmaf(f, y.y, v.y), v.z = fmaf(f, y.z, v.z), v.w = fmaf(f, y.w, v.w);
            }
            if (whole) {
                store_out<HD>(a, r, was.h, was.sq.t0, d4, sum, v);
            } else {
                float *dst = mine + r * RP;
                if (d4 == 0) *(float2 *)(dst + HD) = make_float2(top, sum);
                *(float4 *)(dst + 4 * d4) = v;
            }
        }
        if (!whole) {
            const int64_t c0 = ((was.pair_x + 1) * was.G - 1) / was.W;
            const int nc = (int)(((was.pair_x + was.cells) * was.G - 1) / was.W - c0) + 1;
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                uint32_t *cnt = a.count + (int64_t)was.b * kv.nkv + was.h;
                s_last = atom_add_acq_rel_gpu(cnt, 1u) == (uint32_t)(nc - 1);
                if (s_last) *cnt = 0u;  // for the next launch
            }
            __syncthreads();
            if (s_last)
                join_parts<HD, NT>(a, (int)c0, nc, rows, was.h, was.sq.t0, sums_of(0), RB / 4, s_m);
        }
        if (!more) break;
        __syncthreads();  // shared memory is written again for the next pair
    }
    if (s_rest) zero_rest<HD>(a);
}

// Column blocks of eight query rows that the kernel takes at once, and its CTAs: two
// an SM with one block (registers), one with more. Measured (us), blocks as needed against
// more: 4 rows, 32 x 8192 58 (one), 82 (two), 106 (three); 16 rows, 64 x 1000 63 (two), 81 (three).
// Three blocks fill the registers (head_dim 128 spills 40 bytes; four spilled more than
// they gained), and from 25 rows on the prompt kernel takes over, at its own price: 24 rows, 8 x 4000 34
// here and 74 there, 1 x 1000 15 and 33; 28 rows 75 and 34 there. Two passes of this kernel over
// such rows were not tried.
constexpr int kFewRows = 24;
int split_nt(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 3; }
int split_grid(int nt) { return nt == 1 ? kMostCtas : kMostCtas / 2; }

// The workspace: the arrival counters of both kernels, then the parts, which they
// use one after the other.
struct Plan {
    int nt;
    bool few, prompt;  // which kernels run
    int64_t pairs, counts_few, counts_prompt, bytes;
};
Plan plan_of(const dm_kv4_cache *c, int64_t seqs, int64_t max_q, int64_t heads) {
    Plan p;
    const int64_t rows = max_q * (heads / c->kv_heads);
    p.prompt = rows > kFewRows;
    p.few = !p.prompt || seqs > 1;  // a long sequence alone leaves nothing for the other kernel
    p.nt = split_nt(rows);
    p.pairs = prompt_pairs(rows);
    p.counts_few = (seqs * c->kv_heads * 4 + 255) / 256 * 256;
    p.counts_prompt = p.prompt ? (seqs * c->kv_heads * p.pairs * 4 + 255) / 256 * 256 : 0;
    int64_t parts = (int64_t)split_grid(p.nt) * 2 * 8 * p.nt * (c->head_dim + 4) * 4;
    if (p.prompt) parts = parts > prompt_part_bytes(c->head_dim) ? parts : prompt_part_bytes(c->head_dim);
    p.bytes = p.counts_few + p.counts_prompt + parts;
    return p;
}

template <int HD, int NT>
cudaError_t launch_split(const AttnArgs &g, void *stream) {
    constexpr int smem = split_smem<HD, NT>();
    static bool ready[64];  // the attribute is per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(kv4_attn_split_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready[dev] = true;
    }
    return launch_pdl(kv4_attn_split_kernel<HD, NT>, dim3(split_grid(NT)), dim3(kWarps * 32), smem, stream, g);
}

template <int HD>
cudaError_t launch_split_nt(const AttnArgs &g, int nt, void *stream) {
    return nt == 1 ? launch_split<HD, 1>(g, stream) : nt == 2 ? launch_split<HD, 2>(g, stream) : launch_split<HD, 3>(g, stream);
}

}  // namespace
}  // namespace dm

extern "C" int64_t dm_kv4_workspace_bytes(const dm_kv4_cache *c, int32_t seqs, int32_t max_q, int32_t heads) {
    if (!c || seqs < 1 || max_q < 1 || heads < 1 || c->kv_heads < 1 || heads % c->kv_heads ||
        (c->head_dim != 64 && c->head_dim != 128))
        return -1;
    return dm::plan_of(c, seqs, max_q, heads).bytes;
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
    if ((int64_t)b->max_q * heads > INT32_MAX / 2)
        return kv_refuse(err, err_len, "%s: %d new tokens of %d heads are too many rows", who, b->max_q, heads);
    const Plan p = plan_of(c, b->seqs, b->max_q, heads);
    if (!b->work || !kv_aligned(b->work, 16) || b->work_bytes < p.bytes)
        return kv_refuse(err, err_len, "%s: the workspace must be 16-byte aligned and hold dm_kv4_workspace_bytes", who);
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
    uint8_t *work = (uint8_t *)b->work;
    g.part = (float *)(work + p.counts_few + p.counts_prompt);
    g.rest = !p.few;
    cudaError_t e = cudaSuccess;
    if (p.few) {
        g.few = p.prompt ? kFewRows : INT32_MAX;
        g.nrb = 0;
        g.count = (uint32_t *)work;
        e = c->head_dim == 64 ? launch_split_nt<64>(g, p.nt, stream) : launch_split_nt<128>(g, p.nt, stream);
    }
    if (e == cudaSuccess && p.prompt) {
        g.few = p.few ? kFewRows : -1;
        g.nrb = (int)p.pairs;
        g.count = (uint32_t *)(work + p.counts_few);
        e = launch_prompt(g, c->head_dim, stream);
    }
    return kv_launched("kv4 attention kernels", e, err, err_len);
}
