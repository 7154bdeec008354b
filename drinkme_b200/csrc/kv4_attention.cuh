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
    float scale;
    int64_t window;
    uint32_t *count;  // arrivals by sequence and kv head (and pair of tiles), zero between launches
    float *part;      // CTAs' parts of what they share with others
};

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
