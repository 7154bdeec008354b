// What the two attention kernels over the 4-bit cache share.
#pragma once

#include "kv4.cuh"

namespace dm {

constexpr float kLog2e = 1.4426950408889634f;
// A weight may exceed 1 by this power of two before a row's running maximum is
// raised: the sums are rescaled only then.
constexpr float kSlack = 8.f;

struct AttnArgs {
    KvView kv;
    const uint16_t *q;
    int64_t qs;
    void *out;
    int32_t nh, grp, out_f32, max_q;
    int32_t few;      // sequences of at most this many query rows a kv head are the few-rows kernel's, the others the prompt kernel's
    int32_t nrb;      // the prompt kernel's pairs of row tiles of the longest sequence
    int32_t rest;     // this kernel writes the rows of no sequence
    float scale;
    int64_t window;
    uint32_t *count;  // arrivals by sequence and kv head (and pair of tiles), zero between launches
    float *part;      // CTAs' parts of what they share with others
};

// A sequence's new tokens [t0, t0 + n): n is 0 where they are not rows of the
// batch or more than max_q (recorded; such a sequence is left out).
struct Tokens {
    int32_t t0, n;
    bool rest;  // rows of the batch before the first sequence, after the last or of this one are no sequence's
};
__device__ __forceinline__ Tokens tokens_of(const AttnArgs &a, int b) {
    Tokens s;
    s.t0 = a.kv.q_start[b];
    const int end = a.kv.q_start[b + 1];
    s.n = end - s.t0;
    s.rest = (b == 0 && s.t0 > 0) || (b == a.kv.seqs - 1 && end < a.kv.tokens);
    if (s.t0 < 0 || s.n < 0 || s.n > a.max_q || end > a.kv.tokens) {
        s.rest = true;
        if (s.n != 0) atomicExch(a.kv.err, kKvErrRange);
        s.n = 0;
    }
    return s;
}

// The first position that a token at position p sees.
__device__ __forceinline__ int64_t first_seen(const AttnArgs &a, int64_t p) {
    return a.window > 0 ? max((int64_t)0, p - a.window + 1) : 0;
}

// Zeros for the rows of `out` that no sequence's tokens are: before the first, past the
// last, of one left out. A warp a token; called by whole CTAs, where there are such rows.
// Not in line: its registers are not the loop's.
template <int HD>
__device__ __noinline__ void zero_rest(const AttnArgs &a) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    for (int t = blockIdx.x * warps + (threadIdx.x >> 5); t < a.kv.tokens; t += gridDim.x * warps) {
        const int b = kv_sequence(a.kv, t, lane);
        if (b < a.kv.seqs) {
            const Tokens s = tokens_of(a, b);
            if (t >= s.t0 && t - s.t0 < s.n) continue;
        }
        const int64_t row = (int64_t)a.nh * HD, n = row * (a.out_f32 ? 4 : 2) / 16;
        uint4 *out = (uint4 *)a.out + t * n;
        for (int64_t i = lane; i < n; i += 32) out[i] = make_uint4(0u, 0u, 0u, 0u);
    }
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
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));  // weights below 2^-126 of the largest are 0
    return y;
}
__device__ __forceinline__ float bf_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf_hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// 16 bytes global -> shared, asynchronously; a group is what was copied since the last commit
__device__ __forceinline__ void ring_copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ring_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The prompt kernel (kv4_prompt.cu)
int64_t prompt_pairs(int64_t rows);
int64_t prompt_part_bytes(int hd);
cudaError_t launch_prompt(const AttnArgs &g, int hd, void *stream);

}  // namespace dm
