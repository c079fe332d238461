// nmoe_gdn_prefill.cu -- the GatedDeltaNet core of packed prompts.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>

#include "nmoe/moe_cuda.h"
#include "nmoe_common.cuh"

namespace nmoe {
namespace {

thread_local char g_err[256];

int fail(int status, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
    return status;
}

constexpr int kD = 128;

struct GdnArgs {
    const int *cu_rows;
    const void *qkv, *z, *alpha, *beta;
    long long qkv_stride, z_stride, ab_stride;
    const uint16_t *conv_w, *dt_bias, *norm_w;
    const float *A_log;
    const float *conv_in, *delta_in;
    float *conv_out, *delta_out;
    void *out;
    int num_seqs, total_rows, key_heads, value_heads, channels, x_bf16, out_bf16;
};

__device__ __forceinline__ float load_x(const void *p, long long at, int bf16) {
    return bf16 ? bf16_to_f32(static_cast<const uint16_t *>(p)[at]) : static_cast<const float *>(p)[at];
}
// log(1 + exp(x)) without overflow
__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

__device__ __forceinline__ float block_sum(float v, float *red, int warp, int lane) {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// A CTA per (value head, sequence), token by token; thread t holds row t of the state and
// convolves channel t of the head's q, k and v.
__global__ void __launch_bounds__(kD) k_gdn_rows(const __grid_constant__ GdnArgs a) {
    __shared__ __align__(16) float qs[kD], ks[kD];
    __shared__ float red[4];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int vh = blockIdx.x, b = blockIdx.y, kh = vh / (a.value_heads / a.key_heads);
    const int r0 = max(0, min(a.cu_rows[b], a.total_rows)), r1 = min(a.cu_rows[b + 1], a.total_rows);
    float S[kD];
    const long long so = (((long long)b * a.value_heads + vh) * kD + t) * kD;
#pragma unroll
    for (int i = 0; i < kD; ++i) S[i] = a.delta_in ? a.delta_in[so + i] : 0.f;
    const int ch[3] = {kh * kD + t, (a.key_heads + kh) * kD + t, (2 * a.key_heads + vh) * kD + t};
    float w[3][4], x[3][3];
#pragma unroll
    for (int c = 0; c < 3; ++c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[c][j] = bf16_to_f32(a.conv_w[4 * ch[c] + j]);
#pragma unroll
        for (int j = 0; j < 3; ++j) x[c][j] = a.conv_in ? a.conv_in[((long long)b * 3 + j) * a.channels + ch[c]] : 0.f;
    }
    const float rate = -expf(a.A_log[vh]), dt = bf16_to_f32(a.dt_bias[vh]), nw = bf16_to_f32(a.norm_w[t]);
    for (long long r = r0; r < r1; ++r) {
        float y[3];
#pragma unroll
        for (int c = 0; c < 3; ++c) {
            const float n = load_x(a.qkv, r * a.qkv_stride + ch[c], a.x_bf16);
            const float s = x[c][0] * w[c][0] + x[c][1] * w[c][1] + x[c][2] * w[c][2] + n * w[c][3];
            y[c] = siluf_(s);
            x[c][0] = x[c][1], x[c][1] = x[c][2], x[c][2] = n;
        }
        const float qq = block_sum(y[0] * y[0], red, warp, lane), kk = block_sum(y[1] * y[1], red, warp, lane);
        qs[t] = y[0] * rsqrtf(qq / kD + 1e-12f) * (1.0f / kD);
        ks[t] = y[1] * rsqrtf(kk / kD + 1e-12f) * rsqrtf((float)kD);
        __syncthreads();
        const float g = expf(rate * softplus(load_x(a.alpha, r * a.ab_stride + vh, a.x_bf16) + dt));
        const float beta = sigmoidf_(load_x(a.beta, r * a.ab_stride + vh, a.x_bf16));
        float kv = 0.f;
#pragma unroll
        for (int i = 0; i < kD; ++i) {
            S[i] *= g;
            kv = fmaf(S[i], ks[i], kv);
        }
        const float d = (y[2] - kv) * beta;
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < kD; ++i) {
            S[i] = fmaf(ks[i], d, S[i]);
            o = fmaf(S[i], qs[i], o);
        }
        const float oo = block_sum(o * o, red, warp, lane);
        const float zz = load_x(a.z, r * a.z_stride + vh * kD + t, a.x_bf16);
        const float v = o * rsqrtf(oo / kD + 1e-6f) * nw * siluf_(zz);
        const long long at = (r * a.value_heads + vh) * kD + t;
        if (a.out_bf16)
            static_cast<uint16_t *>(a.out)[at] = __bfloat16_as_ushort(__float2bfloat16(v));
        else
            static_cast<float *>(a.out)[at] = v;
    }
#pragma unroll
    for (int i = 0; i < kD; ++i) a.delta_out[so + i] = S[i];
}

// The last three inputs of every channel. After the rows: the states may be updated in place.
__global__ void k_gdn_conv_state(const __grid_constant__ GdnArgs a) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x, b = blockIdx.y;
    if (c >= a.channels) return;
    const int r0 = max(0, min(a.cu_rows[b], a.total_rows)), r1 = min(a.cu_rows[b + 1], a.total_rows);
    const int n = max(0, r1 - r0);
    float v[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
        const int i = n + j - 3;   // row of the sequence, negative: of the state before it
        v[j] = i >= 0 ? load_x(a.qkv, (long long)(r0 + i) * a.qkv_stride + c, a.x_bf16)
                      : (a.conv_in ? a.conv_in[((long long)b * 3 + 3 + i) * a.channels + c] : 0.f);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) a.conv_out[((long long)b * 3 + j) * a.channels + c] = v[j];
}

int check_shape(const nmoe_linear_attn_shape *s) {
    if (s == nullptr) return fail(NMOE_EINVAL, "shape is NULL");
    if (s->key_heads < 1 || s->key_heads > 1024 || s->value_heads < 1 || s->value_heads > 8192 ||
        s->value_heads % s->key_heads != 0)
        return fail(NMOE_EINVAL, "value_heads %d must be a multiple of key_heads %d (at most 1024; 8192 value heads)",
                    s->value_heads, s->key_heads);
    return NMOE_OK;
}

bool aligned_to(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace nmoe

using namespace nmoe;

extern "C" const char *nmoe_linear_attn_error(void) { return g_err; }

extern "C" size_t nmoe_linear_attn_prefill_workspace_bytes(const nmoe_linear_attn_shape *s, int num_seqs,
                                                           int total_rows) {
    (void)s;
    (void)num_seqs;
    (void)total_rows;
    return 0;
}

extern "C" int nmoe_linear_attn_prefill(const nmoe_linear_attn_weights *w, const nmoe_linear_attn_shape *shape,
                                        int num_seqs, int total_rows, const int32_t *cu_rows, const void *qkv,
                                        int64_t qkv_stride, const void *z, int64_t z_stride, const void *alpha,
                                        const void *beta, int64_t ab_stride, int x_dtype, const float *conv_in,
                                        const float *delta_in, float *conv_out, float *delta_out, void *out,
                                        int out_dtype, void *workspace, void *stream) {
    int rc = check_shape(shape);
    if (rc != NMOE_OK) return rc;
    if (w == nullptr || w->conv_w == nullptr || w->A_log == nullptr || w->dt_bias == nullptr || w->norm_w == nullptr)
        return fail(NMOE_EINVAL, "a weight is NULL");
    if (num_seqs < 0 || total_rows < 0) return fail(NMOE_EINVAL, "num_seqs or total_rows is negative");
    if (num_seqs > 65535) return fail(NMOE_EINVAL, "num_seqs %d: at most 65535", num_seqs);
    if (num_seqs == 0) return NMOE_OK;
    if (cu_rows == nullptr || !aligned_to(cu_rows, 4)) return fail(NMOE_EINVAL, "cu_rows is NULL or not aligned");
    if (conv_out == nullptr || delta_out == nullptr) return fail(NMOE_EINVAL, "conv_out or delta_out is NULL");
    if (total_rows > 0 && (qkv == nullptr || z == nullptr || alpha == nullptr || beta == nullptr || out == nullptr))
        return fail(NMOE_EINVAL, "an operand is NULL");
    if ((x_dtype != NMOE_DTYPE_F32 && x_dtype != NMOE_DTYPE_BF16) ||
        (out_dtype != NMOE_DTYPE_F32 && out_dtype != NMOE_DTYPE_BF16))
        return fail(NMOE_EINVAL, "x_dtype and out_dtype: NMOE_DTYPE_F32 or NMOE_DTYPE_BF16");
    const long long ch = (2ll * shape->key_heads + shape->value_heads) * kD, vw = (long long)shape->value_heads * kD;
    GdnArgs a;
    a.qkv_stride = qkv_stride == 0 ? ch : qkv_stride;
    a.z_stride = z_stride == 0 ? vw : z_stride;
    a.ab_stride = ab_stride == 0 ? shape->value_heads : ab_stride;
    const int unit = x_dtype == NMOE_DTYPE_BF16 ? 8 : 4;
    if (a.qkv_stride < ch || a.z_stride < vw || a.ab_stride < shape->value_heads || a.qkv_stride % unit != 0 ||
        a.z_stride % unit != 0 || !aligned_to(qkv, 16) || !aligned_to(z, 16) || !aligned_to(alpha, 4) ||
        !aligned_to(beta, 4))
        return fail(NMOE_EINVAL, "a row stride is too small, or qkv or z rows are not 16-byte aligned");
    if (!aligned_to(w->conv_w, 8) || !aligned_to(w->A_log, 4) || !aligned_to(conv_in, 16) || !aligned_to(conv_out, 16) ||
        !aligned_to(delta_in, 16) || !aligned_to(delta_out, 16) || !aligned_to(out, 16))
        return fail(NMOE_EINVAL, "a state, weight or output is not aligned");
    a.cu_rows = cu_rows;
    a.qkv = qkv;
    a.z = z;
    a.alpha = alpha;
    a.beta = beta;
    a.conv_w = w->conv_w;
    a.dt_bias = w->dt_bias;
    a.norm_w = w->norm_w;
    a.A_log = w->A_log;
    a.conv_in = conv_in;
    a.delta_in = delta_in;
    a.conv_out = conv_out;
    a.delta_out = delta_out;
    a.out = out;
    a.num_seqs = num_seqs;
    a.total_rows = total_rows;
    a.key_heads = shape->key_heads;
    a.value_heads = shape->value_heads;
    a.channels = (int)ch;
    a.x_bf16 = x_dtype == NMOE_DTYPE_BF16;
    a.out_bf16 = out_dtype == NMOE_DTYPE_BF16;
    (void)workspace;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    k_gdn_rows<<<dim3(shape->value_heads, num_seqs), kD, 0, st>>>(a);
    k_gdn_conv_state<<<dim3((unsigned)((ch + 255) / 256), num_seqs), 256, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? NMOE_OK : fail(NMOE_ECUDA, "prefill: %s", cudaGetErrorString(e));
}
