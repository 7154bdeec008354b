// Grouped-query attention over the paged 4-bit cache for many query rows per kv
// head (prompt chunks), on the 5th-generation tensor cores.
//
// A CTA takes two tiles of 128 query rows (row = new token x head of the kv
// head's group) against blocks of 128 positions. Per tile S = Q K^T and
// O += P V are tcgen05.mma with fp32 accumulators in tensor memory (two S of 128
// columns, two O of head_dim: all 512 columns); P replaces the first half of its S.
//
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread a row, no shuffles
//   warps 8-11      codes to bf16 operands in shared memory, scales to fp32
//   warp 12         issues the MMAs (one thread) and owns the tensor memory
//
// Mathematics: the scores' product runs on the key codes, which bf16 holds
// exactly, and the rows' scales are applied in fp32, the row's maximum taken off in
// the same instruction: s_ij - M_i = k_j (q_i . (128 + c_j)) + ((m_j - 128 k_j) sum(q_i) - M_i).
// (Keys rounded to bf16 would put 2^-9 of a score's size into it.) Values the same way:
// O = sum_j bf16(p_j v_j) (c_j - 8) + sum_j p_j (m_j + 8 v_j), the second sum a number a row, in fp32.
// The weights' rounding is then the only one; values made whole and rounded, bf16(m_j + v_j c_j),
// were faster (420 us where this takes 479) but their rounding is as large as the weights' (relative error of
// the output 0.0027 against 0.0023, 0.0017 of it the output's own bf16). Exponentials
// are taken against the row's last maximum, 32 columns at a time; only when a score
// passes it by more than 2^8 is it raised (and O, and what is there of P, rescaled in
// tensor memory). A value row that is NaN is a zero operand whose key scale is NaN: it
// reaches the rows that see it, and no weight of 0 meets a NaN in the product.
//
// Order of elements: a word's eight codes come apart as pairs (i, i + 4); q is
// stored in the same order, so K needs no shuffling. V is stored transposed, eight
// positions of one element a 16-byte piece: the halves of two positions' words are put
// together first.
//
// Work split: the blocks of all (sequence, kv head, pair of tiles) in order,
// cut into equal ranges, one a CTA; a pair cut in two leaves its parts {O, maximum, sum}
// in the workspace and the last CTA to finish joins them in order. A part is 128 KB, about
// a block's time to write and read again: ranges have at least four blocks (64 tokens after 3936
// rows: 53 us, with one block 64, with eight 64), and
// where every pair can have a CTA of its own and none is longer than an equal
// range by more than four blocks, none is cut (512 tokens alone: 33 us, cut 52; 33 tokens after
// 967 rows, eight blocks: 39 us cut, 53 not).
//
// Bound: per block and pair of tiles the MMAs take 2048 cycles of the tensor core
// (head_dim 128), the exponentials 2048 of the MUFU. Measured: 2048 tokens after 6144 rows, 32 heads
// on 8, 479 us (502 TF/s of 1640), 1024 after 15360 with 64 heads 982 us (542 TF/s). With the values
// made whole (420 us) a pair of tiles took 6700 cycles a block: for each tile one chain of the
// softmax (4500), the last product and the next scores (2200: P lies where the next S will, so they
// wait for one another), while the operand warps work 4900; the scales in the weights put 900 more on the
// softmax. All roles share the schedulers and shared
// memory. P in shared memory with the next S ahead of P V takes the chain apart, but its
// stores and the product's reads of it cost more (474 us for 420); blocks of half the width with two
// S in turn 486, more warps for the operands 487, chunks of 16 columns pipelined 439. Scores two at
// a time in fp32 pairs took 430 to 420. Weights split in two bf16 (values whole) 496, as exact as
// this.
#include <type_traits>

#include "kv4.cuh"
#include "kv4_attention.cuh"

namespace dm {
namespace {

constexpr int kTile = 128;    // query rows of a tile, positions of a block
constexpr int kSoft = 8;      // softmax warps
constexpr int kDeq = 4;       // warps that make operands
constexpr int kMmaWarp = kSoft + kDeq;
constexpr int kThreads = 16 * 32;  // four warpgroups; warps 13-15 only fill the last
constexpr int kGrid = 148;    // one CTA an SM
constexpr int kLeast = 4;     // blocks of a range that may cut pairs, at least
constexpr int kSpare = 4;     // blocks that a pair may be longer than an equal range before it is cut
constexpr int kBars = 22;  // the last only keeps what follows on 16 bytes

template <int HD>
struct Smem {
    static constexpr int PANEL = kTile * 128;         // 128 rows x 64 bf16, 128-byte swizzle
    static constexpr int Q = 0;                       // [2 tiles][HD / 64 panels]
    static constexpr int K = Q + 2 * (HD / 64) * PANEL;  // [2 stages][HD / 64 panels]
    static constexpr int VPANEL = HD * 128;           // HD rows x 64 positions
    static constexpr int V = K + 2 * (HD / 64) * PANEL;  // [2 stages][2 panels]
    static constexpr int RAW = V + 2 * 2 * VPANEL;    // [2][128 rows of codes, 16 bytes between groups of eight]
    static constexpr int RAWB = kTile * (HD / 2) + 16 * 16;
    static constexpr int SC = RAW + 2 * RAWB;         // [2 stages][64 pairs of positions] key s, s, m, m, value s, s, m, m
    static constexpr int ROW = SC + 2 * kTile * 16;   // [2][128] int64 rows of the cache (-1: none)
    static constexpr int BAR = ROW + 2 * kTile * 8;
    static constexpr int LIVE = BAR + kBars * 8;      // [2 stages][4] which positions have rows
    static constexpr int MISC = LIVE + 32;
    static constexpr int BYTES = MISC + 32 + 1024;    // and room to align the tiles
};

// Issued by the lane with `lead` of a converged warp (so that the operands stay
// in uniform registers)
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
        "r"(lead)
        : "memory");
}
__device__ __forceinline__ uint32_t elect() {
    uint32_t lead;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(lead));
    return lead;
}
// Two fp32 values in a pair of registers: one instruction for both
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}
__device__ __forceinline__ void pair_to(uint64_t d, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(d)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void tmem_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Registers of a warpgroup's threads: 144 + 144 + 136 + 88 of the launch's 4 x 128.
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void group_sync(int id) {  // N threads on named barrier id
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}

// A sequence as this kernel sees it: blocks of 128 positions for each pair of row tiles.
struct PSeq {
    int32_t t0, n, len, pairs, all, longest;  // of one kv head: its pairs, all their blocks, the longest's
};
// The blocks [first, end) that pair `rp` of a sequence needs (at least one).
__device__ __forceinline__ void pair_blocks(const AttnArgs &a, const PSeq &s, int rp, int &first, int &end) {
    const int i0 = rp * (2 * kTile) / a.grp, i1 = min(s.n * a.grp - 1, (rp + 1) * (2 * kTile) - 1) / a.grp;
    const int p0 = s.len - s.n;  // the first new token's position
    first = (int)(first_seen(a, (int64_t)p0 + i0) / kTile);
    const int64_t covered = (int64_t)a.kv.cols << a.kv.pshift;  // rows past it are not there
    end = max(first + 1, (int)((min((int64_t)max(0, p0 + i1 + 1), covered) + kTile - 1) / kTile));
}
__device__ __forceinline__ PSeq pseq_of(const AttnArgs &a, int b, const Tokens &q) {
    PSeq s;
    s.t0 = q.t0, s.n = q.n;
    s.len = max(a.kv.kv_len[b], 0);
    if (s.n * (int64_t)a.grp <= a.few) s.n = 0;  // the other kernel's
    if (s.n > 0 && s.len > (int64_t)a.kv.cols << a.kv.pshift) atomicExch(a.kv.err, kKvErrRange);
    s.pairs = (int)(((int64_t)s.n * a.grp + 2 * kTile - 1) / (2 * kTile));
    s.all = s.longest = 0;
    for (int rp = 0; rp < s.pairs; ++rp) {
        int f, e;
        pair_blocks(a, s, rp, f, e);
        s.all += e - f;
        s.longest = max(s.longest, e - f);
    }
    return s;
}
__device__ __forceinline__ PSeq pseq_of(const AttnArgs &a, int b) { return pseq_of(a, b, tokens_of(a, b)); }

// One piece of work: blocks [j0, j1) of a pair of tiles; `first`, `end` are the pair's.
struct Piece {
    int b, h, rp, j0, j1, first, end, t0, n, len, rows;  // rows of the two tiles
    int low;                                             // the first position that any of them sees
    int64_t x, pair_x;
};

// The CTA's pieces in order, the same for every role.
struct Walk {
    int64_t x, x1, seq_x;
    int b;
    bool whole;  // a cell is a pair; otherwise a block
    PSeq s;
    __device__ int cells(int blocks) const { return whole ? 1 : blocks; }
    __device__ int all() const { return whole ? s.pairs : s.all; }
    __device__ bool next(const AttnArgs &a, Piece &p) {
        if (x >= x1) return false;
        while (x >= seq_x + (int64_t)a.kv.nkv * all()) {
            seq_x += (int64_t)a.kv.nkv * all();
            s = pseq_of(a, ++b);
        }
        const int64_t in = x - seq_x;
        p.h = (int)(in / all());
        int left = (int)(in - (int64_t)p.h * all()), first = 0, end = 0;
        p.pair_x = x - left;
        p.rp = 0;
        for (;; ++p.rp) {
            pair_blocks(a, s, p.rp, first, end);
            const int n = cells(end - first);
            if (left < n) break;
            left -= n;
            p.pair_x += n;
        }
        p.b = b, p.first = first, p.end = end;
        p.j0 = first + left;
        p.j1 = whole ? end : (int)min((int64_t)end, p.j0 + (x1 - x));
        p.t0 = s.t0, p.n = s.n, p.len = s.len;
        p.rows = min(2 * kTile, s.n * a.grp - p.rp * 2 * kTile);
        p.low = (int)first_seen(a, (int64_t)s.len - s.n + p.rp * (2 * kTile) / a.grp);
        p.x = x;
        x += cells(p.j1 - p.j0);
        return true;
    }
};

// The next piece of a warp's walk (both in shared memory: the roles' registers
// are for their loops).
__device__ __forceinline__ bool next_piece(const AttnArgs &a, Walk &walk, Piece &piece) {
    Walk w = walk;
    Piece p;
    __syncwarp();
    const bool more = w.next(a, p);
    if (more && (threadIdx.x & 31) == 0) {
        walk = w;
        piece = p;
    }
    __syncwarp();
    return more;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) kv4_prompt_kernel(const __grid_constant__ AttnArgs a) {
    using M = Smem<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *bar = (uint64_t *)(smem + M::BAR);
    uint64_t *k_full = bar, *k_empty = bar + 2, *v_full = bar + 4, *v_empty = bar + 6, *sc_full = bar + 8,
             *sc_empty = bar + 10, *s_full = bar + 12, *p_ready = bar + 14, *pv_done = bar + 16, *q_ready = bar + 18, *drain = bar + 20;
    // o_free (the tile's O has been read) is q_ready of the next piece: Q is written after O is read
    uint32_t *live = (uint32_t *)(smem + M::LIVE);
    uint32_t *misc = (uint32_t *)(smem + M::MISC);
    __shared__ int4 s_scan[kThreads / 32];  // blocks and pairs up to a warp's sequences, the longest pair
    __shared__ Walk s_walk[kMmaWarp + 1];
    __shared__ Piece s_piece[kMmaWarp + 1][2];
    __shared__ int64_t s_total, s_ctas;  // cells, CTAs that take some

    pdl_launch_dependents();
    pdl_wait();
    const KvView &kv = a.kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int *err = kv.err;

    // the cut
    const int per = (kv.seqs + kThreads - 1) / kThreads;
    {
        int blocks = 0, pairs = 0, longest = 0;
        bool rest = false;
        for (int b = tid * per; b < min(kv.seqs, (tid + 1) * per); ++b) {
            const Tokens k = tokens_of(a, b);
            const PSeq q = pseq_of(a, b, k);
            rest = rest || k.rest;
            blocks += q.all, pairs += q.pairs, longest = max(longest, q.longest);
        }
        int ub = blocks, up = pairs;
        for (int o = 1; o < 32; o <<= 1) {
            const int vb = __shfl_up_sync(0xffffffffu, ub, o), vp = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) ub += vb, up += vp;
            longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
        }
        if (lane == 31) s_scan[warp] = make_int4(ub, up, longest, 0);
        if (tid == 0) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&k_full[i], kDeq), mbar_init(&k_empty[i], 1);
                mbar_init(&v_full[i], kDeq), mbar_init(&v_empty[i], 1);
                mbar_init(&sc_full[i], kDeq), mbar_init(&sc_empty[i], kSoft);
                mbar_init(&s_full[i], 1), mbar_init(&p_ready[i], 4), mbar_init(&pv_done[i], 1), mbar_init(&q_ready[i], 4);
            }
            mbar_init(drain, 1);
            mbar_fence_init();
        }
        rest = __syncthreads_or(rest);
        int all_b = 0, all_p = 0, before_b = 0, before_p = 0, most = 0;
        for (int w = 0; w < kThreads / 32; ++w) {
            const int4 v = s_scan[w];
            if (w < warp) before_b += v.x, before_p += v.y;
            all_b += v.x, all_p += v.y, most = max(most, v.z);
        }
        if (rest && a.rest) zero_rest<HD>(a);
        const int64_t Wb = (int64_t)all_b * kv.nkv, Wp = (int64_t)all_p * kv.nkv;
        const bool whole = Wp <= gridDim.x && most <= (Wb + gridDim.x - 1) / gridDim.x + kSpare;
        const int64_t W = whole ? Wp : Wb, G = whole ? Wp : min((int64_t)gridDim.x, (Wb + kLeast - 1) / kLeast);
        if (blockIdx.x >= G) return;
        const int64_t x = blockIdx.x * W / G, end = (int64_t)(whole ? before_p + up : before_b + ub) * kv.nkv;
        int64_t begin = end - (int64_t)(whole ? pairs : blocks) * kv.nkv;
        if (begin <= x && x < end) {
            Walk w;
            w.x = x, w.x1 = (blockIdx.x + 1) * W / G, w.b = tid * per, w.whole = whole;
            for (;; ++w.b) {
                w.s = pseq_of(a, w.b);
                if (x < begin + (int64_t)w.all() * kv.nkv) break;
                begin += (int64_t)w.all() * kv.nkv;
            }
            w.seq_x = begin;
            for (int i = 0; i <= kMmaWarp; ++i) s_walk[i] = w;
            s_total = W;
            s_ctas = G;
        }
        if (warp == kMmaWarp) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(misc)), "r"(512)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        tmem_before();
        __syncthreads();
        tmem_after();
    }
    const uint32_t tmem = *misc;
    const int role = min(warp, kMmaWarp);
    Walk &walk = s_walk[role];
    bool ok = true;
    const float sl = a.scale * kLog2e;

    if (warp < kSoft) {
        // ------------------------------------------------------ softmax --
        regs_up<144>();
        const int tile = warp >> 2, row = tid & (kTile - 1);
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t ts = lanes + tile * kTile, to = lanes + 2 * kTile + tile * HD;
        uint8_t *qs = smem + M::Q + tile * (HD / 64) * M::PANEL;
        uint32_t blk = 0, use = 0;  // blocks of the CTA so far, and of this tile
        auto wait = [&](uint64_t *b, uint32_t parity) {
            if (ok) ok = mbar_wait(b, parity, err, kKvErrWait);
            __syncwarp();
        };
        const Piece &pc = s_piece[role][0];
        while (next_piece(a, walk, s_piece[role][0])) {
            const bool active = tile * kTile < pc.rows;
            const int rr = pc.rp * 2 * kTile + tile * kTile + row, tok = rr / a.grp, head = pc.h * a.grp + rr % a.grp;
            const bool mine = tile * kTile + row < pc.rows;
            float qsum = 0.f;
            if (active) {
                // q's row in the order of the codes: 16 bytes hold elements 0 4 1 5 2 6 3 7 of eight
                const uint4 *src = (const uint4 *)(a.q + (int64_t)(pc.t0 + (mine ? tok : 0)) * a.qs + (int64_t)(mine ? head : 0) * HD);
#pragma unroll
                for (int c0 = 0; c0 < HD / 8; c0 += 8) {  // eight loads on their way before the first store
                    uint4 q8[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) q8[k] = mine ? src[c0 + k] : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int c = c0 + k;
                        const uint4 w = q8[k];
                        qsum += ((bf_lo(w.x) + bf_hi(w.x)) + (bf_lo(w.y) + bf_hi(w.y))) +
                                ((bf_lo(w.z) + bf_hi(w.z)) + (bf_lo(w.w) + bf_hi(w.w)));
                        *(uint4 *)(qs + (c >> 3) * M::PANEL + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
                            make_uint4(__byte_perm(w.x, w.z, 0x5410), __byte_perm(w.x, w.z, 0x7632),
                                       __byte_perm(w.y, w.w, 0x5410), __byte_perm(w.y, w.w, 0x7632));
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_ready[tile]);
            }
            float m = -INFINITY;
            uint64_t l[2] = {0, 0};  // sums of every fourth position, two and two
            uint64_t base = 0;       // what the rows' values have in common: sums of p (m + 8 s)
            const uint64_t qsum2 = pair_of(qsum, qsum);
            const int p = pc.len - pc.n + tok;  // the row's position
            const int see0 = (int)first_seen(a, p);
            const int j0 = pc.j0, j1 = pc.j1;
            for (int j = j0; j < j1; ++j, ++blk) {
                const uint32_t st = blk & 1;
                wait(&sc_full[st], (blk >> 1) & 1);
                if (active) {
                    wait(&s_full[tile], use & 1);
                    tmem_after();
                    const ulonglong2 *sck = (const ulonglong2 *)(smem + M::SC + st * kTile * 16);  // keys' and values' of two positions
                    const int hi = p - j * kTile, lo = see0 - j * kTile;  // columns lo .. hi are seen
                    const uint32_t *lv = live + st * 4;
                    const bool inside = mine && hi >= kTile - 1 && lo <= 0 && (lv[0] & lv[1] & lv[2] & lv[3]) == 0xffffffffu;
                    const bool edge = !__all_sync(0xffffffffu, inside);
                    auto block = [&](auto edge_tag) {
                        constexpr bool EDGE = decltype(edge_tag)::value;
                        uint32_t r[32];
                        tmem_ld32(ts, r);
#pragma unroll 1
                        for (int c0 = 0; c0 < kTile; c0 += 32) {
                            const bool none = m == -INFINITY;  // no maximum yet: taken as 0
                            const float off = none ? 0.f : -m;
                            const uint64_t off2 = pair_of(off, off);
                            float t[32], tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const ulonglong2 k = sck[c0 + i];
                                pair_to(fma_pair(pair_of(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), k.x,
                                                 fma_pair(k.y, qsum2, off2)),
                                        t[i], t[i + 1]);
                            }
                            if (c0 + 32 < kTile) tmem_ld32(ts + c0 + 32, r);  // on its way meanwhile
                            if (EDGE) {
                                const uint32_t w = mine ? lv[c0 >> 5] : 0u;
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                    if (c0 + i > hi || c0 + i < lo || !((w >> i) & 1)) t[i] = -INFINITY;
                            }
#pragma unroll
                            for (int i = 0; i < 32; i += 2) tops[(i >> 1) & 3] = fmaxf(tops[(i >> 1) & 3], fmaxf(t[i], t[i + 1]));
                            const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                            if (__any_sync(0xffffffffu, top > (none ? -INFINITY : kSlack))) {
                                const float up = none ? (top == -INFINITY ? 0.f : top) : fmaxf(top, 0.f);
                                const float f = none ? 1.f : exp2_approx(-up);  // nothing is summed without a maximum
                                m = none ? top : m + up;
#pragma unroll
                                for (int i = 0; i < 32; ++i) t[i] -= up;
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    float x, y;
                                    pair_to(l[i], x, y);
                                    l[i] = pair_of(x * f, y * f);
                                }
                                {
                                    float x, y;
                                    pair_to(base, x, y);
                                    base = pair_of(x * f, y * f);
                                }
                                if (j > j0) {  // O, once the last product has been added to it
                                    wait(&pv_done[tile], (use - 1) & 1);
                                    tmem_after();
#pragma unroll 1
                                    for (int d = 0; d < HD; d += 16) {
                                        uint32_t o[16];
                                        tmem_ld16(to + d, o);
                                        tmem_wait_ld();
#pragma unroll
                                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                        tmem_st16(to + d, o);
                                    }
                                }
                                tmem_wait_st();
#pragma unroll 1
                                for (int d = 0; d < c0 / 2; d += 16) {  // this block's weights so far
                                    uint32_t o[16];
                                    tmem_ld16(ts + d, o);
                                    tmem_wait_ld();
#pragma unroll
                                    for (int i = 0; i < 16; ++i) o[i] = pack_bf16(bf_lo(o[i]) * f, bf_hi(o[i]) * f);
                                    tmem_st16(ts + d, o);
                                }
                            }
                            uint32_t pk[16];
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float p0 = exp2_approx(t[i]), p1 = exp2_approx(t[i + 1]);
                                const uint64_t p2 = pair_of(p0, p1);
                                const ulonglong2 v = sck[c0 + i + 1];
                                l[(i >> 1) & 1] = add_pair(l[(i >> 1) & 1], p2);
                                base = fma_pair(p2, v.y, base);
                                float w0, w1;
                                pair_to(mul_pair(p2, v.x), w0, w1);
                                pk[i >> 1] = pack_bf16(w0, w1);
                            }
                            // over scores that have been read: columns c0 / 2 .. + 16
                            tmem_st16(ts + (c0 >> 1), pk);
                        }
                    };
                    if (edge) block(std::true_type{});
                    else block(std::false_type{});
                    tmem_wait_st();
                    tmem_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_ready[tile]);
                    ++use;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sc_empty[st]);
            }
            // the rows' results, or this CTA's part of them
            float l0, l1, l2, l3;
            pair_to(l[0], l0, l1), pair_to(l[1], l2, l3);
            float b0, b1;
            pair_to(base, b0, b1);
            const float bsum = b0 + b1;
            const float lsum = (l0 + l1) + (l2 + l3);
            const bool whole = pc.j0 == pc.first && pc.j1 == pc.end;
            const int slot = pc.j0 == pc.first ? 1 : 0;
            if (active) {
                wait(&pv_done[tile], (use - 1) & 1);
                tmem_after();
                const float inv = whole ? (lsum == 0.f ? 0.f : 1.f / lsum) : 1.f;
                // parts lie [HD / 4][128 rows][4], so that a warp's pieces are together
                float *part = a.part + (((int64_t)blockIdx.x * 2 + slot) * 2 + tile) * (kTile * (HD + 4));
                const int64_t at = ((int64_t)(pc.t0 + tok) * a.nh + head) * HD;
#pragma unroll 1
                for (int c0 = 0; c0 < HD; c0 += 32) {
                    uint32_t r[32];
                    tmem_ld32(to + c0, r);
                    tmem_wait_ld();
                    if (!mine) continue;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float y[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = (__uint_as_float(r[i + e]) + bsum) * inv;
                        if (!whole) {
                            *(float4 *)(part + ((c0 + i) * kTile + row * 4)) = make_float4(y[0], y[1], y[2], y[3]);
                            *(float4 *)(part + ((c0 + i + 4) * kTile + row * 4)) = make_float4(y[4], y[5], y[6], y[7]);
                        } else if (a.out_f32) {
                            float4 *o = (float4 *)((float *)a.out + at + c0 + i);
                            o[0] = make_float4(y[0], y[1], y[2], y[3]);
                            o[1] = make_float4(y[4], y[5], y[6], y[7]);
                        } else {
                            *(uint4 *)((uint16_t *)a.out + at + c0 + i) =
                                make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]),
                                           pack_bf16(y[6], y[7]));
                        }
                    }
                }
                if (!whole && mine) *(float2 *)(part + HD * kTile + row * 4) = make_float2(m, lsum);
                tmem_before();
            }
            if (!whole) {
                const int64_t W = s_total, G = s_ctas;
                const int64_t c0 = ((pc.pair_x + 1) * G - 1) / W;
                const int nc = (int)(((pc.pair_x + pc.end - pc.first) * G - 1) / W - c0) + 1;
                __threadfence();
                group_sync<kSoft * 32>(1);
                if (tid == 0) {
                    uint32_t *cnt = a.count + ((int64_t)pc.b * kv.nkv + pc.h) * a.nrb + pc.rp;
                    const bool last = atom_add_acq_rel_gpu(cnt, 1u) == (uint32_t)(nc - 1);
                    if (last) *cnt = 0u;  // for the next launch
                    misc[1] = last;
                }
                group_sync<kSoft * 32>(1);
                if (misc[1] && mine) {
                    __threadfence();
                    auto part_of = [&](int c) {
                        return a.part + (((c0 + c) * 2 + (c == 0 ? 1 : 0)) * 2 + tile) * (int64_t)(kTile * (HD + 4)) + row * 4;
                    };
                    float top = -INFINITY, sum = 0.f;
                    for (int c = 0; c < nc; ++c) top = fmaxf(top, __ldcg(part_of(c) + HD * kTile));
                    for (int c = 0; c < nc; ++c) {
                        const float2 ml = __ldcg((const float2 *)(part_of(c) + HD * kTile));
                        sum = fmaf(ml.x == top ? 1.f : exp2_approx(ml.x - top), ml.y, sum);
                    }
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    const int64_t at = ((int64_t)(pc.t0 + tok) * a.nh + head) * HD;
#pragma unroll 1
                    for (int d = 0; d < HD; d += 32) {
                        float4 y[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (int c = 0; c < nc; ++c) {
                            const float *src = part_of(c);
                            const float mc = __ldcg(src + HD * kTile), f = mc == top ? 1.f : exp2_approx(mc - top);
                            float4 z[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) z[i] = __ldcg((const float4 *)(src + (d + 4 * i) * kTile));
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                y[i].x = fmaf(f, z[i].x, y[i].x), y[i].y = fmaf(f, z[i].y, y[i].y);
                                y[i].z = fmaf(f, z[i].z, y[i].z), y[i].w = fmaf(f, z[i].w, y[i].w);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            y[i].x *= inv, y[i].y *= inv, y[i].z *= inv, y[i].w *= inv;
                            if (a.out_f32)
                                *(float4 *)((float *)a.out + at + d + 4 * i) = y[i];
                            else
                                *(uint2 *)((uint16_t *)a.out + at + d + 4 * i) =
                                    make_uint2(pack_bf16(y[i].x, y[i].y), pack_bf16(y[i].z, y[i].w));
                        }
                    }
                }
                group_sync<kSoft * 32>(1);  // misc[1] is written again
            }
        }
    } else if (warp < kMmaWarp) {
        // ----------------------------------------------------- operands --
        regs_up<136>();
        const int d = tid - kSoft * 32;  // 0 .. 127: the key row, and a piece of the values
        const int dw = warp - kSoft;
        constexpr int RW = HD / 8;       // words of a row
        int64_t *s_row = (int64_t *)(smem + M::ROW);
        uint32_t blk = 0;
        auto wait = [&](uint64_t *b, uint32_t parity) {
            if (ok) ok = mbar_wait(b, parity, err, kKvErrWait);
            __syncwarp();
        };
        // what is in flight for the next block: the key row's codes, its
        // scales; the value rows go to shared memory
        uint32_t kw[RW];
        uint2 sc;
        bool have;
        // the page table's entry for this thread's position of a block
        auto entry_of = [&](const Piece &p, int j) -> int {
            const int64_t pos = (int64_t)j * kTile + d, col = pos >> kv.pshift;
            return pos < p.len && col < kv.cols ? __ldcg(kv.table + (int64_t)p.b * kv.tstride + col) : -1;
        };
        int entry = -1;  // for the next block, looked up a block ahead
        auto fetch = [&](const Piece &p, int j, uint32_t buf) {
            const int64_t pos = (int64_t)j * kTile + d;
            have = pos < p.len && entry >= 0 && entry < kv.pages;
            // (a page that lies before every row's window need not be there)
            if (pos < p.len && !have && pos >= p.low) atomicExch(err, kKvErrRange);
            const int64_t r = have ? ((int64_t)entry * kv.nkv + p.h) * 2 * kv.ps + (pos & (kv.ps - 1)) : -1;
            s_row[buf * kTile + d] = r;
            group_sync<kDeq * 32>(2);
            if (j + 1 < p.j1) entry = entry_of(p, j + 1);
            const uint4 *k = (const uint4 *)(kv.codes + (have ? r : 0) * (HD / 2));
#pragma unroll
            for (int i = 0; i < RW / 4; ++i) {
                const uint4 w = have ? __ldcg(k + i) : make_uint4(0, 0, 0, 0);
                kw[4 * i] = w.x, kw[4 * i + 1] = w.y, kw[4 * i + 2] = w.z, kw[4 * i + 3] = w.w;
            }
            // scales row: (page * nkv + h) * ps + slot
            const int64_t sr = ((r >> (kv.pshift + 1)) << kv.pshift) | (r & (kv.ps - 1));
            sc = have ? __ldcg((const uint2 *)(kv.scales + sr * 4)) : make_uint2(0, 0);
            constexpr int PC = HD / 32;  // 16-byte pieces of a row
            const uint32_t raw = smem_addr(smem + M::RAW + buf * M::RAWB);
#pragma unroll
            for (int i = 0; i < PC; ++i) {
                const int id = i * kTile + d, tk = id / PC, pp = id % PC;
                const int64_t vr = s_row[buf * kTile + tk];
                if (vr >= 0)
                    ring_copy16(raw + tk * (HD / 2) + (tk >> 3) * 16 + pp * 16, kv.codes + (vr + kv.ps) * (HD / 2) + pp * 16);
            }
            ring_commit();
        };
        uint32_t cur = 0;  // which of the two pieces
        bool more = next_piece(a, walk, s_piece[role][0]);
        if (more) {
            entry = entry_of(s_piece[role][0], s_piece[role][0].j0);
            fetch(s_piece[role][0], s_piece[role][0].j0, 0);
        }
        while (more) {
            const Piece &pc = s_piece[role][cur];
            const int j1 = pc.j1;
            for (int j = pc.j0; j < j1; ++j, ++blk) {
                const uint32_t st = blk & 1, ph = (blk >> 1) & 1;
                const uint2 s = sc;
                const bool had = have;
                // a value row that is not finite is a zero operand (and its key's scale NaN)
                const bool poison = !isfinite(bf_lo(s.y)) || !isfinite(bf_hi(s.y));
                // scales
                if (blk >= 2) wait(&sc_empty[st], ph ^ 1);
                {
                    const float ks = poison ? NAN : bf_lo(s.x), km = bf_hi(s.x);
                    const float vs = bf_lo(s.y), vm = bf_hi(s.y);
                    float *f = (float *)(smem + M::SC + st * kTile * 16) + (d >> 1) * 8 + (d & 1);
                    f[0] = had ? ks * sl : 0.f;
                    f[2] = had ? fmaf(-128.f, ks, km) * sl : 0.f;
                    f[4] = had && !poison ? vs : 0.f;
                    f[6] = had && !poison ? fmaf(8.f, vs, vm) : 0.f;
                    const uint32_t lv = __ballot_sync(0xffffffffu, had);
                    if (lane == 0) {
                        live[st * 4 + dw] = lv;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[st]);
                }
                // keys: a row of 128 + c in the order of the pairs
                if (blk >= 2) wait(&k_empty[st], ph ^ 1);
                {
                    uint8_t *ks = smem + M::K + st * (HD / 64) * M::PANEL + d * 128;
#pragma unroll
                    for (int c = 0; c < RW; ++c)
                        *(uint4 *)(ks + (c >> 3) * M::PANEL + (((c & 7) ^ (d & 7)) << 4)) =
                            make_uint4(codes128(kw[c]), codes128(kw[c] >> 4), codes128(kw[c] >> 8), codes128(kw[c] >> 12));
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&k_full[st]);
                }
                // the codes of the values have landed before the next copies begin
                ring_wait<0>();
                if (j + 1 < j1) {
                    fetch(pc, j + 1, (blk + 1) & 1);
                } else {
                    Piece &nx = s_piece[role][cur ^ 1];
                    more = next_piece(a, walk, nx);
                    if (more) {
                        entry = entry_of(nx, nx.j0);
                        fetch(nx, nx.j0, (blk + 1) & 1);
                    } else {
                        group_sync<kDeq * 32>(2);
                    }
                }
                // values, eight positions of an element a piece. (The named barrier in fetch
                // has made every thread's copies and scales of this block visible.)
                if (blk >= 2) wait(&v_empty[st], ph ^ 1);
                {
                    const int kg = d & 7, panel = (d >> 3) & 1, dg = d >> 4;  // positions 64 panel + 8 kg ..., elements (HD / 8) dg ...
                    const uint8_t *raw = smem + M::RAW + (blk & 1) * M::RAWB + (panel * 64 + kg * 8) * (HD / 2) +
                                         (panel * 8 + kg) * 16 + dg * (HD / 16);
                    uint8_t *vs = smem + M::V + st * 2 * M::VPANEL + panel * M::VPANEL;
                    constexpr int VW = HD / 64;
                    uint32_t v[8][VW];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if constexpr (VW == 2) {
                            const uint2 x = *(const uint2 *)(raw + i * (HD / 2));
                            v[i][0] = x.x, v[i][1] = x.y;
                        } else {
                            v[i][0] = *(const uint32_t *)(raw + i * (HD / 2));
                        }
                    }
#pragma unroll
                    for (int k = 0; k < VW; ++k)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            uint32_t pr[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                pr[i] = __byte_perm(v[2 * i][k], v[2 * i + 1][k], half ? 0x7632 : 0x5410);
#pragma unroll
                            for (int n = 0; n < 4; ++n) {
                                const int e = dg * (HD / 8) + 8 * k + 4 * half + n;
                                uint32_t x[4];
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    x[i] = less136(codes128(pr[i] >> (4 * n)));
                                *(uint4 *)(vs + e * 128 + ((kg ^ (e & 7)) << 4)) = make_uint4(x[0], x[1], x[2], x[3]);
                            }
                        }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&v_full[st]);
                }
            }
            cur ^= 1;
        }
        ring_wait<0>();
    } else {
        // ---------------------------------------------------------- MMA --
        regs_down<88>();
        if (warp == kMmaWarp) {
            constexpr uint32_t ID_S = idesc_f16(kTile, kTile), ID_O = idesc_f16(kTile, HD);
            const uint32_t lead = elect();
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), base = smem_addr(smem);
            uint32_t blk = 0, pieces[2] = {0, 0}, use[2] = {0, 0};  // use: S products issued for the tile
            auto wait = [&](uint64_t *b, uint32_t parity) {
                if (ok) ok = mbar_wait(b, parity, err, kKvErrWait);
                __syncwarp();
            };
            const Piece &pc = s_piece[role][0];
            while (next_piece(a, walk, s_piece[role][0])) {
                const int nt = __shfl_sync(0xffffffffu, pc.rows > kTile ? 2 : 1, 0);
                auto score = [&](int t, uint32_t st) {  // S of a tile; its last P has been read
                    if (use[t] > 0) wait(&pv_done[t], (use[t] - 1) & 1);
                    tmem_after();
                    if (ok) {
                        const uint64_t q = sw128_desc(base + M::Q + t * (HD / 64) * M::PANEL),
                                       k = sw128_desc(base + M::K + st * (HD / 64) * M::PANEL);
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk) {
                            constexpr uint32_t P16 = M::PANEL / 16;
                            mma_ss(tm + t * kTile, q + (kk >> 2) * P16 + (kk & 3) * 2, k + (kk >> 2) * P16 + (kk & 3) * 2, ID_S,
                                   kk > 0, lead);
                        }
                    }
                    mma_commit(&s_full[t], lead);
                    ++use[t];
                };
                wait(&k_full[blk & 1], (blk >> 1) & 1);
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (t < nt) {
                        wait(&q_ready[t], pieces[t] & 1);
                        ++pieces[t];
                        score(t, blk & 1);
                    }
                mma_commit(&k_empty[blk & 1], lead);
                const int n = __shfl_sync(0xffffffffu, pc.j1 - pc.j0, 0);
                for (int j = 0; j < n; ++j, ++blk) {
                    const uint32_t st = blk & 1, nst = (blk + 1) & 1;
                    wait(&v_full[st], (blk >> 1) & 1);
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        if (t < nt) {
                            wait(&p_ready[t], (use[t] - 1) & 1);
                            tmem_after();
                            if (ok) {
                                const uint64_t v = sw128_desc(base + M::V + st * 2 * M::VPANEL);
#pragma unroll
                                for (int kk = 0; kk < kTile / 16; ++kk)
                                    mma_ts(tm + 2 * kTile + t * HD, tm + t * kTile + kk * 8,
                                           v + (kk >> 2) * (M::VPANEL / 16) + (kk & 3) * 2, ID_O, j > 0 || kk > 0, lead);
                            }
                            mma_commit(&pv_done[t], lead);
                            if (t == nt - 1) mma_commit(&v_empty[st], lead);
                            if (j + 1 < n) {
                                if (t == 0) wait(&k_full[nst], ((blk + 1) >> 1) & 1);
                                score(t, nst);
                                if (t == nt - 1) mma_commit(&k_empty[nst], lead);
                            }
                        }
                }
            }
            // every product issued has completed before the tensor memory is freed, also
            // after a wait that gave up
            mma_commit(drain, lead);
            mbar_wait(drain, 0, err, kKvErrWait);
            __syncwarp();
        }
        __syncwarp();
    }
    tmem_before();
    __syncthreads();
    tmem_after();
    if (warp == kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <int HD>
cudaError_t launch(const AttnArgs &g, void *stream) {
    static bool ready[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(kv4_prompt_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD>::BYTES);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready[dev] = true;
    }
    return launch_pdl(kv4_prompt_kernel<HD>, dim3(kGrid), dim3(kThreads), Smem<HD>::BYTES, stream, g);
}

}  // namespace

int64_t prompt_pairs(int64_t rows) { return (rows + 2 * kTile - 1) / (2 * kTile); }
int64_t prompt_part_bytes(int hd) { return (int64_t)kGrid * 2 * 2 * kTile * (hd + 4) * 4; }

cudaError_t launch_prompt(const AttnArgs &g, int hd, void *stream) {
    return hd == 64 ? launch<64>(g, stream) : launch<128>(g, stream);
}

}  // namespace dm
