// Logits before a token is chosen: penalties for repeated tokens, biases and
// the grammar's mask in one pass over the row.
//
// Bound: each logit is read once and written once. A block takes a slice of a
// row's vocabulary and keeps the slice's counts in shared memory: it reads the
// row's whole history (from L2 after the first block) and counts the ids that
// fall into its slice with shared-memory atomics — integers, so their order
// changes nothing — which needs neither a count table in device memory nor a
// second launch.
#include "kv4.cuh"

namespace dm {
namespace {

constexpr uint32_t kSeen = 1u << 31;
constexpr int kSlice = 4096;
constexpr int kLogitThreads = 256;

template <bool F32>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(dm_logits_args a) {
    __shared__ uint32_t count[kSlice];
    __shared__ int32_t bias_at[kSlice];
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.y, v0 = blockIdx.x * kSlice, n = min(kSlice, a.vocab - v0), tid = threadIdx.x;
    for (int i = tid; i < n; i += kLogitThreads) count[i] = 0u, bias_at[i] = -1;
    __syncthreads();
    if (a.history) {
        const int32_t *ids = a.history + (int64_t)row * a.history_stride;
        const int64_t total = a.total_len ? min((int64_t)max(a.total_len[row], 0), a.history_stride) : a.history_stride;
        const int64_t prompt = a.prompt_len ? a.prompt_len[row] : 0;
        for (int64_t i = tid; i < total; i += kLogitThreads) {
            const int64_t k = (int64_t)ids[i] - v0;
            if (k < 0 || k >= n) continue;
            atomicOr(&count[k], kSeen);
            if (i >= prompt) atomicAdd(&count[k], 1u);
        }
    }
    if (a.bias_ids) {
        const int32_t *ids = a.bias_ids + (int64_t)row * a.bias_stride;
        for (int64_t i = tid; i < a.bias_stride; i += kLogitThreads) {
            const int64_t k = (int64_t)ids[i] - v0;
            if (k >= 0 && k < n) atomicMax(&bias_at[k], (int)i);
        }
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[row] : 1.f, pres = a.presence ? a.presence[row] : 0.f,
                freq = a.frequency ? a.frequency[row] : 0.f;
    for (int i = tid; i < n; i += kLogitThreads) {
        const int v = v0 + i;
        const int64_t at = (int64_t)row * a.stride + v;
        float x = F32 ? ((const float *)a.logits)[at] : bf16_bits_to_f32(((const uint16_t *)a.logits)[at]);
        const uint32_t c = count[i];
        if (c & kSeen) {
            x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
            const uint32_t times = c & ~kSeen;
            x = __fsub_rn(x, __fmul_rn(freq, (float)times));
            if (times) x = __fsub_rn(x, pres);
        }
        if (bias_at[i] >= 0) x = __fadd_rn(x, a.bias_values[(int64_t)row * a.bias_stride + bias_at[i]]);
        if (a.allowed && !((a.allowed[(int64_t)row * a.allowed_stride + (v >> 5)] >> (v & 31)) & 1)) x = -INFINITY;
        const int64_t o = (int64_t)row * a.out_stride + v;
        if (F32)
            ((float *)a.out)[o] = x;
        else
            ((uint16_t *)a.out)[o] = f32_to_bf16_bits(x);
    }
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
    if (a->history_stride < 0 || a->bias_stride < 0 || a->bias_stride > INT32_MAX)
        return kv_refuse(err, err_len, "%s: bad stride", who);
    if (a->allowed && a->rows > 1 && a->allowed_stride < (a->vocab + 31) / 32)
        return kv_refuse(err, err_len, "%s: the mask's rows are shorter than the vocabulary", who);
    if (a->rows == 0) return DM_OK;
    const dim3 grid((unsigned)((a->vocab + kSlice - 1) / kSlice), (unsigned)a->rows);
    const cudaError_t e =
        a->dtype == DM_F32 ? launch_pdl(logits_kernel<true>, grid, dim3(kLogitThreads), 0, stream, *a)
                           : launch_pdl(logits_kernel<false>, grid, dim3(kLogitThreads), 0, stream, *a);
    return kv_launched("logits_kernel", e, err, err_len);
}
