// Grouped-query attention over the paged 4-bit cache.
#include "kv4.cuh"

namespace dm {
namespace {

struct AttnArgs {
    KvView kv;
    const uint16_t *q;
    int64_t qs;
    void *out;
    int32_t nh, grp, out_f32;
    float scale;
    int64_t window;
};

// A warp per (token, head): the keys in order, one at a time, with a running
// maximum and sum; lane l holds elements [l * HD / 32, (l + 1) * HD / 32).
template <int HD>
__global__ void __launch_bounds__(128) kv4_attn_rows_kernel(AttnArgs a) {
    constexpr int E = HD / 32;
    pdl_launch_dependents();
    pdl_wait();
    const KvView &kv = a.kv;
    const int t = blockIdx.x, lane = threadIdx.x & 31, head = blockIdx.y * 4 + (threadIdx.x >> 5);
    const int b = kv_sequence(kv, t, lane);
    if (head >= a.nh) return;
    const int g = head / a.grp;
    const bool none = b >= kv.seqs || t < kv.q_start[b];
    const int64_t p = none ? -1 : (int64_t)kv.kv_len[b] - (kv.q_start[b + 1] - t);
    int64_t first = a.window > 0 ? p - a.window + 1 : 0;
    if (first < 0) first = 0;
    float q[E], acc[E], m = -INFINITY, sum = 0.f;
    for (int e = 0; e < E; ++e) {
        q[e] = bf16_bits_to_f32(a.q[(int64_t)t * a.qs + (int64_t)head * HD + lane * E + e]) * a.scale;
        acc[e] = 0.f;
    }
    for (int64_t j = first; j <= p; ++j) {
        const int64_t page = kv_page(kv, b, j);
        if (page < 0) continue;
        const int slot = (int)(j & (kv.ps - 1));
        const int64_t at = page * kv.nkv + g;
        const uint8_t *kc = kv.codes + (at * 2 * kv.ps + slot) * (HD / 2), *vc = kc + (int64_t)kv.ps * (HD / 2);
        const uint16_t *sc = kv.scales + (at * kv.ps + slot) * 4;
        const float ks = bf16_bits_to_f32(sc[0]), km = bf16_bits_to_f32(sc[1]);
        const float vs = bf16_bits_to_f32(sc[2]), vm = bf16_bits_to_f32(sc[3]);
        float s = 0.f, v[E];
        for (int e = 0; e < E; ++e) {
            const int i = lane * E + e, sh = 4 * (i & 1);
            s += q[e] * (ks * (float)((kc[i >> 1] >> sh) & 15) + km);
            v[e] = vs * (float)((vc[i >> 1] >> sh) & 15) + vm;
        }
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const float mn = fmaxf(m, s), r = m == mn ? 1.f : __expf(m - mn), w = __expf(s - mn);
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * r + w * v[e];
        sum = sum * r + w;
        m = mn;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int e = 0; e < E; ++e) {
        const int64_t o = ((int64_t)t * a.nh + head) * HD + lane * E + e;
        if (a.out_f32)
            ((float *)a.out)[o] = acc[e] * inv;
        else
            ((uint16_t *)a.out)[o] = f32_to_bf16_bits(acc[e] * inv);
    }
}

}  // namespace
}  // namespace dm

extern "C" int64_t dm_kv4_workspace_bytes(const dm_kv4_cache *c, int32_t seqs, int32_t max_q, int32_t heads) {
    if (!c || seqs < 1 || max_q < 1 || heads < 1 || c->kv_heads < 1 || heads % c->kv_heads) return -1;
    return dm::kKvHead;
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
    g.scale = scale;
    g.window = window;
    const dim3 grid((unsigned)b->tokens, (unsigned)((heads + 3) / 4));
    const cudaError_t e = c->head_dim == 64 ? launch_pdl(kv4_attn_rows_kernel<64>, grid, dim3(128), 0, stream, g)
                                            : launch_pdl(kv4_attn_rows_kernel<128>, grid, dim3(128), 0, stream, g);
    return kv_launched("kv4_attn_rows_kernel", e, err, err_len);
}
