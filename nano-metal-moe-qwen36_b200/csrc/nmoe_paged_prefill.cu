// nmoe_paged_prefill.cu -- causal attention of packed prompts over a paged bf16 cache.
#include <cuda_runtime.h>

#include "nmoe_paged.cuh"

namespace nmoe {
namespace {

struct PrefillArgs {
    PagedDev c;
    RotaryDev rot;
    HeadDev h;
    const int *cu_rows, *kv_lens;
    const void *q;
    long long q_stride;
    uint16_t *out;
    float scale;   // softmax scale
    int num_seqs, total_rows, kv_heads, group, gated, x_bf16;
};

constexpr int kThreads = 128;

// A warp per (row, query head): the positions one after another, lane l holding dims E l ..
template <int D>
__global__ void __launch_bounds__(kThreads) k_prefill_rows(const __grid_constant__ PrefillArgs a) {
    constexpr int E = D / 32;
    __shared__ float2 cs[kThreads / 32][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int heads = a.kv_heads * a.group;
    const long long unit = (long long)blockIdx.x * (kThreads / 32) + warp;
    if (unit >= (long long)a.total_rows * heads) return;
    const int r = (int)(unit / heads), head = (int)(unit - (long long)r * heads), kvh = head / a.group;
    const int b = find_sequence(a.cu_rows, a.num_seqs, r, lane);
    if (b < 0) return;
    const long long at = (long long)a.kv_lens[b] - a.cu_rows[b + 1] + r;
    const int position = at < 0 ? -1 : (int)min(at, (long long)a.c.capacity - 1);
    float q[E], o[E];
    const long long src = (long long)r * a.q_stride + (long long)head * (a.gated ? 2 * D : D) + E * lane;
    load_elems<E>(a.q, src, a.x_bf16, q);
    for (int t = lane; t < a.rot.half; t += 32) cs[warp][t] = rotary_cs(a.rot.freq[t], (int)at);
    __syncwarp();
    prepare_head<E>(q, a.h.q_norm, a.h.eps, cs[warp], a.rot.half, lane);
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = 0.f;
    for (int p = 0; p <= position; ++p) {
        const long long row = paged_row(a.c, b, p);
        if (row < 0) continue;
        const long long x = row + kvh * a.c.head_stride + E * lane;
        float k[E], v[E];
        load_elems<E>(a.c.k, x, true, k);
        load_elems<E>(a.c.v, x, true, v);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s = fmaf(q[i], k[i], s);
        s = warp_sum(s) * a.scale;
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.f : __expf(m - mn), w = __expf(s - mn);
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = fmaf(o[i], c, w * v[i]);
        l = fmaf(l, c, w);
        m = mn;
    }
    float g[E];
    if (a.gated) load_elems<E>(a.q, src + D, a.x_bf16, g);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = l == 0.f ? 0.f : o[i] / l * (a.gated ? sigmoidf_(g[i]) : 1.f);
    store_bf16<E>(a.out + (long long)r * heads * D + (long long)head * D + E * lane, o);
}

}  // namespace
}  // namespace nmoe

using namespace nmoe;

extern "C" size_t nmoe_full_attn_prefill_paged_workspace_bytes(const nmoe_full_attn_shape *s, int num_seqs,
                                                               int total_rows) {
    (void)s;
    (void)num_seqs;
    (void)total_rows;
    return 0;
}

extern "C" int nmoe_full_attn_prefill_paged(const nmoe_full_attn_weights *w, const nmoe_full_attn_shape *shape,
                                            const nmoe_paged_kv *kv, int num_seqs, int total_rows,
                                            const int32_t *cu_rows, const int32_t *kv_lens, const void *q, int x_dtype,
                                            int64_t q_stride, float scale, uint16_t *out, void *workspace,
                                            void *stream) {
    PrefillArgs a;
    int rc = check_full_attn_shape(w, shape);
    if (rc == NMOE_OK) rc = check_paged_kv(kv, &a.c);
    if (rc != NMOE_OK) return rc;
    if (num_seqs < 0 || total_rows < 0) return full_attn_fail(NMOE_EINVAL, "num_seqs or total_rows is negative");
    if (num_seqs == 0 || total_rows == 0) return NMOE_OK;
    if (cu_rows == nullptr || kv_lens == nullptr || !aligned_to(cu_rows, 4) || !aligned_to(kv_lens, 4))
        return full_attn_fail(NMOE_EINVAL, "cu_rows or kv_lens is NULL or not aligned");
    const long long qw = (long long)shape->q_heads * shape->head_dim * (shape->gated ? 2 : 1);
    a.q_stride = q_stride == 0 ? qw : q_stride;
    rc = check_x("q", q, x_dtype, a.q_stride, qw);
    if (rc != NMOE_OK) return rc;
    if (out == nullptr || !aligned_to(out, 16)) return full_attn_fail(NMOE_EINVAL, "out is NULL or not 16-byte aligned");
    if (!(scale >= 0.f && scale <= 3.0e38f)) return full_attn_fail(NMOE_EINVAL, "scale must be finite and not negative");
    fill_rotary(shape, &a.rot);
    a.h = {w->q_norm, nullptr, shape->norm_eps};
    a.cu_rows = cu_rows;
    a.kv_lens = kv_lens;
    a.q = q;
    a.out = out;
    a.scale = scale == 0.f ? 1.0f / sqrtf((float)shape->head_dim) : scale;
    a.num_seqs = num_seqs;
    a.total_rows = total_rows;
    a.kv_heads = shape->kv_heads;
    a.group = shape->q_heads / shape->kv_heads;
    a.gated = shape->gated;
    a.x_bf16 = x_dtype == NMOE_DTYPE_BF16;
    (void)workspace;
    const long long units = (long long)total_rows * shape->q_heads;
    const long long grid = (units + kThreads / 32 - 1) / (kThreads / 32);
    if (grid > 2147483647ll) return full_attn_fail(NMOE_EINVAL, "too many rows");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (shape->head_dim == 256)
        k_prefill_rows<256><<<(unsigned)grid, kThreads, 0, st>>>(a);
    else
        k_prefill_rows<128><<<(unsigned)grid, kThreads, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? NMOE_OK : full_attn_fail(NMOE_ECUDA, "prefill: %s", cudaGetErrorString(e));
}
