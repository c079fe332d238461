// nmoe_paged.cuh -- what the paged full-attention kernels share: the device view of a paged
// cache, the row -> sequence search, and the preparation of one head (RMS norm, rotation).
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "nmoe/moe_cuda.h"
#include "nmoe_common.cuh"
#include "nmoe_sm100.cuh"

namespace nmoe {

struct PagedDev {
    uint16_t *k, *v;
    long long page_stride, row_stride, head_stride;   // elements
    const int *table;
    long long table_stride;
    int num_pages, page_size, max_pages;
    int capacity;   // max_pages * page_size positions (checked to fit an int)
};

// Rotation: pair t < half turns by position * theta^(-t / half), in 64 bits, since the angle has to
// be reduced before it is rounded (an fp32 angle at position 32768 is off by 2e-3). A thread that
// needs a frequency makes it once, of the powers for t's bits: a table of all of them in the kernel's
// parameters, read by 32 lanes at 32 addresses, costs tens of microseconds of constant-cache misses,
// and exp2 in 64 bits as much as the rest of a head's work.
struct RotaryDev {
    double bit[7];   // theta^(-2^k / half)
    int half;        // rotary_dims / 2
};

struct HeadDev {
    const uint16_t *q_norm, *k_norm;   // bf16 [head_dim] or null
    float eps;
};

// theta^(-t / half) / pi: half turns per position
__device__ __forceinline__ double rotary_freq(const RotaryDev &r, int t) {
    double f = 0.31830988618379067;
#pragma unroll
    for (int k = 0; k < 7; ++k) f *= (t >> k & 1) ? r.bit[k] : 1.0;
    return f;
}

__device__ __forceinline__ float2 rotary_cs(double freq, int position) {
    double a = (double)position * freq;
    a -= 2.0 * rint(0.5 * a);   // half turns in [-1, 1]
    float s, c;
    sincospif((float)a, &s, &c);
    return make_float2(c, s);
}

// Element offset of (sequence, position) without the head, or -1: no page holds it.
__device__ __forceinline__ long long paged_row(const PagedDev &c, int seq, int position) {
    if (position < 0 || position >= c.capacity) return -1;
    const int slot = (unsigned)position / (unsigned)c.page_size;
    const int page = c.table[(long long)seq * c.table_stride + slot];
    if (page < 0 || page >= c.num_pages) return -1;
    return (long long)page * c.page_stride + (long long)(position - slot * c.page_size) * c.row_stride;
}

// The sequence that holds packed row r (cu[b] <= r < cu[b + 1]), or -1 for a row behind the last
// sequence or before the first: the number of i in 1..n with cu[i] <= r.
__device__ __forceinline__ int find_sequence(const int *cu, int n, int r) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (cu[mid + 1] <= r)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo < n && cu[0] <= r ? lo : -1;
}

// E elements of x_dtype as floats. The type is a template argument wherever several loads are on their
// way together: a branch per load makes each wait for the one before it.
template <int E, bool kBf16>
__device__ __forceinline__ void load_typed(const void *base, long long at, float *v) {
    if constexpr (kBf16) {
        const uint16_t *p = static_cast<const uint16_t *>(base) + at;
        uint32_t w[E / 2];
        if constexpr (E == 8) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p);
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        } else {
            const uint2 u = *reinterpret_cast<const uint2 *>(p);
            w[0] = u.x, w[1] = u.y;
        }
#pragma unroll
        for (int i = 0; i < E / 2; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
    } else {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
            const float4 f = p[i];
            v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
        }
    }
}
template <int E>
__device__ __forceinline__ void load_elems(const void *base, long long at, bool bf16, float *v) {
    if (bf16)
        load_typed<E, true>(base, at, v);
    else
        load_typed<E, false>(base, at, v);
}

__device__ __forceinline__ uint32_t pack2_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int E>
__device__ __forceinline__ void store_bf16(uint16_t *p, const float *v) {
    if constexpr (E == 8)
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]),
                                                   pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7]));
    else
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
}

// This lane's norm weights + 1 (dims E lane ..): ones without a norm.
template <int E>
__device__ __forceinline__ void load_weight(const uint16_t *weight, int lane, float *w) {
    if (weight != nullptr) {
        load_typed<E, true>(weight, E * lane, w);
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] += 1.0f;
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = 1.0f;
    }
}

// One warp prepares one head of 32 E dims, lane l holding dims E l .. E l + E - 1: RMS norm by the weights
// w (where `norm`), then the rotation of dims 0 .. 2 half - 1 with the row's (cos, sin) table cs[half].
// half is a power of two of at least 8 >= E, so a pair's other dim is in lane ^ (half / E).
template <int E>
__device__ __forceinline__ void prepare_head(float *v, const float *w, bool norm, float eps, const float2 *cs, int half,
                                             int lane) {
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) ss = fmaf(v[i], v[i], ss);
        const float inv = rsqrtf(warp_sum(ss) / (float)(32 * E) + eps);
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = v[i] * inv * w[i];
    }
    if (half > 0) {
        const int d = E * lane;
        const uint32_t flip = d >= half ? 0u : 0x80000000u;   // the sine's sign in a pair's first dim
        const float4 *t = reinterpret_cast<const float4 *>(cs + (d & (half - 1)));
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            const float o0 = __shfl_xor_sync(0xffffffffu, v[i], half / E), o1 = __shfl_xor_sync(0xffffffffu, v[i + 1], half / E);
            if (d < 2 * half) {
                const float4 k = t[i / 2];
                v[i] = fmaf(o0, __uint_as_float(__float_as_uint(k.y) ^ flip), v[i] * k.x);
                v[i + 1] = fmaf(o1, __uint_as_float(__float_as_uint(k.w) ^ flip), v[i + 1] * k.z);
            }
        }
    }
}

// ---- host side -------------------------------------------------------------------------------
// Fills the message of nmoe_full_attn_error() and returns `status`.
int full_attn_fail(int status, const char *fmt, ...);
int check_full_attn_shape(const nmoe_full_attn_weights *w, const nmoe_full_attn_shape *s);
int check_paged_kv(const nmoe_paged_kv *kv, PagedDev *dev);
void fill_rotary(const nmoe_full_attn_shape *s, RotaryDev *r);
int check_x(const char *what, const void *p, int x_dtype, long long stride, long long width);
// Rows of a CTA of eight warps that prepares rows: the largest power of two up to `want` (and 8, and from 1
// on), and the logarithm of the warps that share a row.
void rows_a_cta(int want, int *rows, int *share_log);
int device_sm_count(int *sms);
// Tries of a wait on the device before it gives up and its outputs become NaN: kMaxSpins, or what NMOE_WAIT_TRIES
// says (for tests: 0 gives up at once).
uint32_t wait_tries();
using TensorMapEncode = PFN_cuTensorMapEncodeTiled_v12000;
TensorMapEncode tensor_map_encode();
// Pages as a 5D tensor (64 columns, page rows, panels of 64 columns, heads, pages); boxes of `rows`
// rows and `panels` panels of one page and head, 128-byte swizzle: in shared memory [panel][row][64].
bool page_map(CUtensorMap *m, const PagedDev &c, const uint16_t *base, int d, int heads, int rows, int panels);

// The dynamic shared memory of a kernel: a property of the function on each device, set at its first call there.
struct SmemOnce {
    std::atomic<uint64_t> done{0};   // a bit per device
    template <class K>
    cudaError_t set(K kernel, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (bit != 0 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
        return e;
    }
};

inline bool aligned_to(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace nmoe
