// Logits before a token is chosen: penalties for repeated tokens, biases and
// the grammar's mask, one launch for a batch.
//
// Bound: each logit is read once and written once, and few of them change: the
// tokens of the history and of the biases, and what the mask hides. A block
// takes a slice of a row's vocabulary. It streams the slice through with the mask
// alone (in place and without a mask there is nothing to stream; where a mask byte
// is zero nothing is read). Beside that it reads the row's whole history (from
// L2 after the first block), counts the ids of its slice with shared-memory
// atomics — integers, so their order changes nothing — and lists each that it meets for
// the first time; after a barrier it computes the listed tokens from their
// logits and writes them over. No count table in device memory, no second launch,
// no look-up for the tokens in between.
//
// Slices: a block reads the whole history whatever its slice, so large ones are
// cheaper, but one row alone has to be spread over the GPU and a block's phases
// (loads, counts, the listed tokens) are waits that other blocks on the SM fill: up to 8192
// tokens, halved down to 1024 while there are fewer blocks than two an SM. Vocabulary 151936,
// histories of 2000 to 4000, (us): 64 fp32 rows 28.2 (4096: 26.8, 16384: 30), 256 bf16 rows 52.8
// (4096: 65, 16384: 63), that is 2.8 and 3.1 TB/s of the 6.57 that a copy reaches; one row 3.5, a
// launch's time. What is left above the bytes' 12 and 24.7 us is each block's chain: history, counts,
// listed tokens, one after the other, against 12 to 16 warps' loads.
#include <type_traits>

#include "kv4.cuh"

namespace dm {
namespace {

// A vocabulary entry of the slice: seen in the history, place + 1 of its bias, times generated.
constexpr uint32_t kSeen = 1u << 31, kTimes = 0xffffu;
constexpr int kPlace = 16, kPlaces = 0x7fff;
constexpr int kLogitThreads = 256;
constexpr int kSliceMin = 1024, kSliceMax = 8192;

// N elements of a 16-byte piece, or one element
template <bool F32, bool VEC>
struct Piece {
    static constexpr int N = VEC ? (F32 ? 4 : 8) : 1;
};

// Shared memory: uint32 entries [slice], uint16 list of those that changed [slice]; WIDE (histories
// or biases longer than the fields): uint32 times [slice], int32 places [slice] beside them.
template <bool F32, bool VEC, bool WIDE>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const __grid_constant__ dm_logits_args a, int slice,
                                                               bool in_place) {
    extern __shared__ uint32_t entry[];
    uint16_t *list = (uint16_t *)(entry + slice);
    uint32_t *times_of = (uint32_t *)(list + slice);
    int32_t *place_of = (int32_t *)(times_of + slice);
    __shared__ uint32_t listed;
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.y, v0 = blockIdx.x * slice, n = min(slice, a.vocab - v0), tid = threadIdx.x;
    const bool touch = a.history || a.bias_ids;

    // what does not depend on anything else is on its way first: the first ids
    // of the history (the row is there to its stride), its lengths, the penalties
    constexpr int IDS = 8;
    const int32_t *ids = a.history ? a.history + (int64_t)row * a.history_stride : nullptr;
    const int64_t most = ids ? a.history_stride : 0;
    int32_t id[IDS];
    auto load_ids = [&](int64_t i0) {
#pragma unroll
        for (int k = 0; k < IDS; ++k) id[k] = i0 + k * kLogitThreads + tid < most ? __ldcg(ids + i0 + k * kLogitThreads + tid) : -1;
    };
    load_ids(0);
    const int64_t total = a.total_len && ids ? min((int64_t)max(a.total_len[row], 0), most) : most;
    const int64_t prompt = a.prompt_len ? a.prompt_len[row] : 0;
    const float rep = a.repetition ? a.repetition[row] : 1.f, pres = a.presence ? a.presence[row] : 0.f,
                freq = a.frequency ? a.frequency[row] : 0.f;
    if (touch) {
        for (int i = tid; i < slice / 4; i += kLogitThreads) {
            ((uint4 *)entry)[i] = make_uint4(0u, 0u, 0u, 0u);
            if (WIDE) ((uint4 *)times_of)[i] = make_uint4(0u, 0u, 0u, 0u), ((int4 *)place_of)[i] = make_int4(0, 0, 0, 0);
        }
        if (tid == 0) listed = 0;
    }

    // the slice with the mask alone
    const int64_t in0 = (int64_t)row * a.stride + v0, out0 = (int64_t)row * a.out_stride + v0;
    const uint32_t *mask = a.allowed ? (const uint32_t *)a.allowed + (int64_t)row * a.allowed_stride : nullptr;
    using E = typename std::conditional<F32, uint32_t, uint16_t>::type;
    const E *src = (const E *)a.logits + in0;
    E *dst = (E *)a.out + out0;
    constexpr E HIDDEN = F32 ? (E)0xff800000u : (E)0xff80u;  // -inf
    if (!in_place || mask) {
        constexpr int N = Piece<F32, VEC>::N;
        constexpr int AHEAD = VEC ? 4 : 1;
        constexpr uint32_t ALL = F32 ? 0xfu : 0xffu;
        const int whole = VEC ? n / N * N : 0;  // elements in pieces
        for (int i0 = N * tid; i0 < whole; i0 += N * kLogitThreads * AHEAD) {  // four pieces a thread in flight
            uint32_t m[AHEAD];
            uint4 x[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int i = i0 + N * kLogitThreads * k;
                // bits v .. v + 7 of the mask are byte v / 8
                m[k] = i >= whole ? (in_place ? ALL : 0u) : mask ? (uint32_t)((const uint8_t *)mask)[(v0 + i) >> 3] >> (F32 ? (i & 4) : 0) : ALL;
                m[k] &= ALL;
            }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
                x[k] = m[k] && !(in_place && m[k] == ALL) ? *(const uint4 *)(src + i0 + N * kLogitThreads * k) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int i = i0 + N * kLogitThreads * k;
                if (i >= whole || (in_place && m[k] == ALL)) continue;
                if (mask) {
                    uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (F32) {
                            if (!((m[k] >> e) & 1)) w[e] = HIDDEN;
                        } else {
                            if (!((m[k] >> (2 * e)) & 1)) w[e] = (w[e] & 0xffff0000u) | HIDDEN;
                            if (!((m[k] >> (2 * e + 1)) & 1)) w[e] = (w[e] & 0xffffu) | ((uint32_t)HIDDEN << 16);
                        }
                    }
                    x[k] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                *(uint4 *)(dst + i) = x[k];
            }
        }
        for (int i = whole + tid; i < n; i += kLogitThreads) {
            const bool may = !mask || ((mask[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1);
            if (!may) dst[i] = HIDDEN;
            else if (!in_place) dst[i] = src[i];
        }
    }
    if (!touch) return;

    __syncthreads();  // the entries are zero
    for (int64_t i0 = 0; i0 < total; i0 += IDS * kLogitThreads) {
        uint32_t at[IDS];
#pragma unroll
        for (int k = 0; k < IDS; ++k)
            at[k] = id[k] < 0 || i0 + k * kLogitThreads + tid >= total ? ~0u : (uint32_t)id[k] - (uint32_t)v0;
        if (i0 + IDS * kLogitThreads < total) load_ids(i0 + IDS * kLogitThreads);
#pragma unroll
        for (int k = 0; k < IDS; ++k) {
            if (at[k] >= (uint32_t)n) continue;
            const bool made = i0 + k * kLogitThreads + tid >= prompt;
            if (!atomicOr(&entry[at[k]], kSeen)) list[atomicAdd(&listed, 1u)] = (uint16_t)at[k];
            if (made) atomicAdd(WIDE ? &times_of[at[k]] : &entry[at[k]], 1u);
        }
    }
    if (a.bias_ids) {
        __syncthreads();  // the counts are done: a place is put beside them
        const int32_t *biased = a.bias_ids + (int64_t)row * a.bias_stride;
        for (int64_t i = tid; i < a.bias_stride; i += kLogitThreads) {
            const int32_t b = __ldcg(biased + i);
            const uint32_t at = (uint32_t)b - (uint32_t)v0;
            if (b < 0 || at >= (uint32_t)n) continue;
            uint32_t was;
            if (WIDE) {
                atomicMax(&place_of[at], (int)i + 1);
                was = atomicOr(&entry[at], 1u);  // any bit: it is listed
            } else {  // the last place that names the token
                was = entry[at];
                while ((was >> kPlace & kPlaces) < (uint32_t)i + 1) {
                    const uint32_t now = atomicCAS(&entry[at], was, (was & ~((uint32_t)kPlaces << kPlace)) | ((uint32_t)(i + 1) << kPlace));
                    if (now == was) break;
                    was = now;
                }
            }
            if (!was) list[atomicAdd(&listed, 1u)] = (uint16_t)at;
        }
    }
    __syncthreads();  // the entries, and the slice as it was streamed

    for (uint32_t k = tid; k < listed; k += kLogitThreads) {
        const int i = list[k], v = v0 + i;
        if (mask && !((mask[v >> 5] >> (v & 31)) & 1)) continue;
        // in place the logit is still there: the stream wrote over hidden ones only
        float x = F32 ? ((const float *)src)[i] : bf16_bits_to_f32(((const uint16_t *)src)[i]);
        const uint32_t c = entry[i], place = WIDE ? (uint32_t)place_of[i] : c >> kPlace & kPlaces;
        const float bias = place ? a.bias_values[(int64_t)row * a.bias_stride + place - 1] : 0.f;
        if (c & kSeen) {
            x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
            const uint32_t times = WIDE ? times_of[i] : c & kTimes;
            x = __fsub_rn(x, __fmul_rn(freq, (float)times));
            if (times) x = __fsub_rn(x, pres);
        }
        if (place) x = __fadd_rn(x, bias);
        if (F32) ((float *)dst)[i] = x;
        else ((uint16_t *)dst)[i] = f32_to_bf16_bits(x);
    }
}

template <bool F32, bool VEC, bool WIDE>
cudaError_t launch_wide(const dm_logits_args &a, bool in_place, void *stream) {
    int slice = WIDE ? kSliceMax / 2 : kSliceMax;
    while (slice > kSliceMin && (int64_t)((a.vocab + slice - 1) / slice) * a.rows < 2 * 148) slice /= 2;
    const int smem = slice * (WIDE ? 14 : 6);
    if (smem > 40 * 1024) {  // above the default with what is static
        static bool ready[64];  // the attribute is per device
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev >= 64 || !ready[dev]) {
            e = cudaFuncSetAttribute(logits_kernel<F32, VEC, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (e != cudaSuccess) return e;
            if (dev < 64) ready[dev] = true;
        }
    }
    const dim3 grid((unsigned)((a.vocab + slice - 1) / slice), (unsigned)a.rows);
    return launch_pdl(logits_kernel<F32, VEC, WIDE>, grid, dim3(kLogitThreads), (size_t)smem, stream, a, slice, in_place);
}

template <bool F32, bool VEC>
cudaError_t launch_logits(const dm_logits_args &a, bool in_place, void *stream) {
    // entries of one word hold counts to 65535 and 32766 places
    const bool wide = (a.history && a.history_stride > kTimes) || (a.bias_ids && a.bias_stride >= kPlaces);
    return wide ? launch_wide<F32, VEC, true>(a, in_place, stream) : launch_wide<F32, VEC, false>(a, in_place, stream);
}

}  // namespace
}  // namespace dm

extern "C" int dm_logits_process(const dm_logits_args *a, void *stream, char *err, size_t err_len) {
    using namespace dm;
    const char *who = "dm_logits_process";
    if (!a || !a->logits || !a->out) return kv_refuse(err, err_len, "%s: null logits or output", who);
    if (a->dtype != DM_BF16 && a->dtype != DM_F32)
        return kv_refuse(err, err_len, "%s: the logits must be bf16 or fp32", who);
    if (a->rows < 0 || a->rows > 65535 || a->vocab < 1)
        return kv_refuse(err, err_len, "%s: rows outside 0..65535 or an empty vocabulary", who);
    if (a->rows > 1 && (a->stride < a->vocab || a->out_stride < a->vocab))
        return kv_refuse(err, err_len, "%s: rows overlap", who);
    const uintptr_t size = a->dtype == DM_F32 ? 4 : 2;
    if (!kv_aligned(a->logits, size) || !kv_aligned(a->out, size))
        return kv_refuse(err, err_len, "%s: logits not aligned to their type", who);
    if ((a->bias_ids == nullptr) != (a->bias_values == nullptr))
        return kv_refuse(err, err_len, "%s: bias ids without values or values without ids", who);
    if (a->rows > 1 && a->logits == a->out && a->stride != a->out_stride)
        return kv_refuse(err, err_len, "%s: in place the strides must be the same", who);
    if (a->history_stride < 0 || a->bias_stride < 0 || a->bias_stride > INT32_MAX)
        return kv_refuse(err, err_len, "%s: bad stride", who);
    if (a->allowed && a->rows > 1 && a->allowed_stride < (a->vocab + 31) / 32)
        return kv_refuse(err, err_len, "%s: the mask's rows are shorter than the vocabulary", who);
    if (a->rows == 0) return DM_OK;
    const bool in_place = a->logits == a->out && (a->rows == 1 || a->stride == a->out_stride);
    const int64_t step = 16 / (int64_t)size;  // 16-byte pieces of whole rows
    const bool vec = kv_aligned(a->logits, 16) && kv_aligned(a->out, 16) &&
                     (a->rows == 1 || (a->stride % step == 0 && a->out_stride % step == 0));
    const cudaError_t e = a->dtype == DM_F32 ? (vec ? launch_logits<true, true>(*a, in_place, stream)
                                                    : launch_logits<true, false>(*a, in_place, stream))
                                             : (vec ? launch_logits<false, true>(*a, in_place, stream)
                                                    : launch_logits<false, false>(*a, in_place, stream));
    return kv_launched("logits_kernel", e, err, err_len);
}
