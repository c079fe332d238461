// nmoe_gdn_prefill.cu -- the GatedDeltaNet core of packed prompts, 64 tokens of a sequence at a time.
//
// Per value head, with k, q of unit length times a constant, g_t the decay and b_t the step:
//     S_t = g_t S_{t-1} + b_t (v_t - g_t S_{t-1} k_t) k_t^T,   o_t = S_t q_t
// Inside a chunk (G_t: the sum of log g up to t, S the state before it) the rank-one updates are
//     u_t = b_t (v_t - e^{G_t} S k_t - sum_{s<t} e^{G_t-G_s} (k_t . k_s) u_s)
// a unit lower triangular system: U = T b (V - e^G K S^T), T = (I + M)^{-1},
// M_ts = b_t e^{G_t-G_s} k_t . k_s (s < t): the WY form of a product of rank-one updates (Bischof and Van Loan 1987),
// for the delta rule in chunks as in Yang et al. 2024. Then, with P_ts = e^{G_t-G_s} q_t . k_s (s <= t),
//     O = e^G Q S^T + P U,   S' = e^{G_63} S + sum_t (e^{G_63-G_t} u_t) k_t^T
//
// With R = V - e^G K S^T, U = T b R, so P U = (P T b) R and, with Z = K^T (e^{G_63 - G} T b),
//     S'^T = e^{G_63} S^T + Z R:
// all that meets the state is one product with [K; Q] and, after R is made of it, one with [Z; P T b].
//
// Three kinds of launch. k_gdn_chunks, a CTA per (chunk, key head): convolution and norms of q and k, K K^T and
// Q K^T, P T b and Z of its value heads; nothing here depends on the state. k_gdn_scan, a CTA per
// (sequence, value head, 64 of the 128 value columns): the recurrence over the chunks; the columns of
// the state never mix, so the CTAs of a head share nothing. k_gdn_finish: gated norm and conv states.
// Long sequences that leave SMs idle go in parts: the preparation of a part and the norm of an earlier one run on
// those SMs beside the scan of the part between (see parts_of).
//
// Arithmetic: every product's operands are split into two fp16 parts, x = hi + lo (22 bits), and the
// products hi hi, hi lo, lo hi summed in fp32, so that states are as exact as with fp32 operands (4e-7 of
// their norm). fp16 has the range of 2^40 only: k, q, P and Z are scaled by constants (Z's columns, like
// k, are no longer than one: what a token leaves in the state after contractions), the state and R by a power of two
// that follows a bound on them (|u| <= max |v| + |S|, |S'|^2 <= e^{2 G_63} |S|^2 + sum v^2, row by row, since |k| <= 1
// and b <= 1), from the largest element that the state had a chunk or two ago.
//
// The scan is a chain of two products a chunk, 128 rows high, on tcgen05: [K; Q] S^T (128 x 64 x 128) and Z R
// (128 x 64 x 64); P T b R follows beside the work on the state. Between them eight warps read the sums from tensor
// memory, a thread per row and 32 columns, and write the next operand as rows of 128 bytes, which the MMA takes as
// they are (MN-major). What bounds it: the chain's latency, 4600 cycles a chunk, of which the products, bound by
// shared memory's bandwidth, take 1800; and the preparation, which needs more of the machine than the scan (57 ms of an
// SM against 38 at 16384 rows). Measured, 16 key and 32 value heads, bf16: 16384 rows 857 us (preparation, scan and
// norm one after the other: 1061), of which 78 us are the first part's preparation.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>

#include <type_traits>

#include "nmoe/moe_cuda.h"
#include "nmoe_gemm.cuh"
#include "nmoe_paged.cuh"

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

constexpr int kD = 128, kC = 64;      // head dim, tokens of a chunk
constexpr int kSplit = 2, kN = kD / kSplit;   // value columns of a scan CTA: 64
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kScanThreads = 416;     // warps 0-7: the rows, 8: copies and MMAs, 9-12: V
constexpr float kScaleK = 16.f, kScaleQ = 128.f;   // k and q elements are about 1 / 11 and 1 / 128

// Tile images, the same in the workspace and in shared memory: rows of 128 bytes (64 fp16) in 16-byte
// pieces, piece p of row r at p ^ (r & 7): the MMA's 128-byte swizzle, and 8 bank groups for an ldmatrix.
constexpr int kPanel = 128 * 128;     // 128 rows
constexpr int kTileX = 2 * kPanel;    // K over Q, one part (hi or lo): two panels of 64 dims
constexpr int kTileZ = kPanel;        // Z, one part: 128 dims, 64 tokens
constexpr int kTileP = kC * 128;      // P T b, one part: 64 tokens by 64
constexpr int kTileZP = 2 * kTileZ + 2 * kTileP;   // Z hi, lo, then P T b hi, lo
constexpr int kGates = kC * 4;        // e^{G_t}

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
    int part, parts;   // of every sequence's chunks: those that a launch takes
    uint32_t tries;    // of a wait of the scan, before it gives up
    int room;          // chunks that the workspace holds: as many as there are when cu_rows does not decrease
    // workspace, per chunk and head: K over Q, hi and lo; Z, hi and lo, and P T b, hi and lo; gates; and O
    uint8_t *kq, *tp, *gates;
    float *o;
};

__device__ __forceinline__ float load_x(const void *p, long long at, int bf16) {
    return bf16 ? bf16_to_f32(static_cast<const uint16_t *>(p)[at]) : static_cast<const float *>(p)[at];
}
// log(1 + exp(x)) without overflow
__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

__device__ __forceinline__ int seq_first(const GdnArgs &a, int b) { return max(0, min(a.cu_rows[b], a.total_rows)); }
__device__ __forceinline__ int seq_rows(const GdnArgs &a, int b) {
    return max(0, min(a.cu_rows[b + 1], a.total_rows) - seq_first(a, b));
}
__device__ __forceinline__ int seq_chunks(const GdnArgs &a, int b) { return (seq_rows(a, b) + kC - 1) / kC; }
// first of the `chunks` chunks of a sequence that belongs to part p
__device__ __forceinline__ int part_first(const GdnArgs &a, int chunks, int p) {
    return a.parts == 1 ? p * chunks : (int)((unsigned)chunks * p / (unsigned)a.parts);   // at most 2^25 chunks, 16 parts
}

// Two floats in a register pair, one instruction for both.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// x = hi + lo in fp16, two values at a time: hi is x rounded to 11 bits (Veltkamp's splitting: t = (2^13 + 1) x,
// hi = t - (t - x)), which fp16 holds as it is, so that lo comes out of one subtraction (unpacking a
// converted hi goes through the slow conversion unit)
__device__ __forceinline__ void split2(uint64_t x, uint32_t &hi, uint32_t &lo) {
    const uint64_t minus = pair(-1.f, -1.f), t = mul2(x, pair(8193.f, 8193.f));
    const uint64_t h = fma2(fma2(x, minus, t), minus, t), l = fma2(h, minus, x);
    float h0, h1, l0, l1;
    unpair(h, h0, h1);
    unpair(l, l0, l1);
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(h1), "f"(h0));
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(l1), "f"(l0));
}
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) { split2(pair(x, y), hi, lo); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t *r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t *r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void stsm4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}
__device__ __forceinline__ void mma_f16(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A copy out of shared memory, one group; what it reads was fenced for it.
__device__ __forceinline__ void bulk_s2g(void *to, const void *from, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(smem_u32(from)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
// After a wait that ran out: what a barrier still counts, copies or products, lands before its memory goes. Of
// either parity, as one of them is in flight; bounded too.
__device__ __forceinline__ void settle(uint64_t *bar) {
    for (int p = 0; p < 2; ++p)
        for (int k = 0; k < 1000 && !mbar_try_wait_sleep(bar, p, 1000); ++k) {}
}
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// x / (1 + e^-x) with the hardware's exponential and reciprocal: a few 2^-23 of it
__device__ __forceinline__ float silu_fast(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return x * r;
}
__device__ __forceinline__ uint64_t silu2(uint64_t x) {
    float e0, e1, r0, r1;
    unpair(mul2(x, pair(-1.4426950408889634f, -1.4426950408889634f)), e0, e1);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(e0));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(e1));
    unpair(add2(pair(e0, e1), pair(1.f, 1.f)), e0, e1);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(e0));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(e1));
    return mul2(x, pair(r0, r1));
}
// byte offset of 16-byte piece p of row r: in a 128-byte row; in two panels of 128 rows
__device__ __forceinline__ uint32_t at128(int r, int p) { return r * 128 + ((p ^ (r & 7)) << 4); }
__device__ __forceinline__ uint32_t at_kq(int r, int p) { return (p >> 3) * kPanel + at128(r, p & 7); }

// O in the workspace: 8 rows of the batch, a head, 4 columns, then the row of the 8. The scan has a row in a thread,
// so its stores are 128 bytes in a row (row by row they were 16 bytes each, and kept shared memory from the
// other warps for 900 of a chunk's 6400 cycles); the norm reads whole sectors.
__device__ __forceinline__ long long o_at(const GdnArgs &a, long long row, int vh, int col) {
    return (((row >> 3) * a.value_heads + vh) * (kD / 4) + (col >> 2)) * 32 + (row & 7) * 4;
}

// Gated RMS norm of every value head of rows first .. end - 1, 8 rows of a head a warp, a quarter of a row a lane;
// by warp `warp` of `warps`. O comes from an earlier launch that this one may have run beside: past the L1.
template <bool kBf16>
__device__ __forceinline__ void gate_rows(const GdnArgs &a, long long first, long long end, int warp, int warps) {
    const int lane = threadIdx.x & 31, g = lane >> 3;
    const long long eight0 = first >> 3, units = first < end ? (((end + 7) >> 3) - eight0) * a.value_heads : 0;
    using Raw = typename std::conditional<kBf16, uint16_t, float>::type;
    constexpr int kZ = kBf16 ? 1 : 2;   // 16-byte loads of 8 columns
    uint2 w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const uint2 *>(a.norm_w + 8 * (4 * (i >> 1) + g) + 4 * (i & 1));
    for (long long u = warp; u < units; u += warps) {
        const int vh = (int)(u % a.value_heads);
        const long long row = ((eight0 + u / a.value_heads) << 3) + (lane & 7);
        const bool in = row >= first && row < end;
        const long long src = in ? row : row < first ? first : end - 1;
        const Raw *zp = static_cast<const Raw *>(a.z) + src * a.z_stride + vh * kD;
        float4 o[8];
        uint4 zr[4 * kZ];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = 8 * (4 * i + g);
#pragma unroll
            for (int x = 0; x < 2; ++x) o[2 * i + x] = __ldcg(reinterpret_cast<const float4 *>(a.o + o_at(a, src, vh, c + 4 * x)));
#pragma unroll
            for (int x = 0; x < kZ; ++x) zr[kZ * i + x] = *reinterpret_cast<const uint4 *>(zp + c + 4 * x);
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += o[i].x * o[i].x + o[i].y * o[i].y + o[i].z * o[i].z + o[i].w * o[i].w;
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const float inv = rsqrtf(sum / kD + 1e-6f);
        const long long at = (row * a.value_heads + vh) * kD;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float z[8], v[8];
            if constexpr (kBf16) {
                const uint32_t r[4] = {zr[i].x, zr[i].y, zr[i].z, zr[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) z[2 * j] = bf16_lo(r[j]), z[2 * j + 1] = bf16_hi(r[j]);
            } else {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const uint4 r = zr[2 * i + x];
                    z[4 * x] = __uint_as_float(r.x), z[4 * x + 1] = __uint_as_float(r.y);
                    z[4 * x + 2] = __uint_as_float(r.z), z[4 * x + 3] = __uint_as_float(r.w);
                }
            }
            const uint32_t wr[4] = {w[2 * i].x, w[2 * i].y, w[2 * i + 1].x, w[2 * i + 1].y};
            const float ov[8] = {o[2 * i].x,     o[2 * i].y,     o[2 * i].z,     o[2 * i].w,
                                 o[2 * i + 1].x, o[2 * i + 1].y, o[2 * i + 1].z, o[2 * i + 1].w};
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = ov[j] * inv * (j & 1 ? bf16_hi(wr[j / 2]) : bf16_lo(wr[j / 2])) * silu_fast(z[j]);
            if (!in) continue;
            const long long to = at + 8 * (4 * i + g);
            if (a.out_bf16) {
                *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + to) =
                    make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
            } else {
                float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(a.out) + to);
                p[0] = make_float4(v[0], v[1], v[2], v[3]);
                p[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
    }
}

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// One thread of a converged warp issues (`one` != 0): M = 128, fp16, fp32 sums.
__device__ __forceinline__ void mma_one(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one)
        : "memory");
}
__device__ __forceinline__ void commit_one(uint64_t *bar, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(one)
        : "memory");
}
__device__ __forceinline__ uint32_t idesc_f16(int a_mn, int b_mn, int n) {
    return (1u << 4) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// rows are the sum's index, 64 columns a row; further columns `panel` bytes away
__device__ __forceinline__ uint64_t desc_rows(uint32_t addr, uint32_t panel) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)(panel >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
// Polls (a suspended wait wakes some hundred cycles later, five times a chunk). Bounded: a barrier that
// never completes sets `stop`, and every later wait goes at once.
__device__ __forceinline__ bool wait_bar(uint64_t *bar, uint32_t parity, volatile int *stop, uint32_t tries = kMaxSpins) {
    for (uint32_t n = 0;; ++n) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((n & 1023) == 1023 && *stop) return false;
        if (n >= tries) {
            *stop = 1;
            return false;
        }
    }
}

// ---- chunks ---------------------------------------------------------------------------------------

constexpr int kGateRows = 8;   // rows of the grid that norm the heads of an earlier part
constexpr int kLdT = 68;   // T rows
struct ChunkSmem {
    // K over Q, hi and lo, two panels each: K stays; the heads' P hi and lo (later P T b's, then half of Z's lo) go
    // where Q was, head h into panel h. Beside them T (fp32, later images in its place)
    static constexpr int kT = 2 * kTileX, kTBytes = kC * kLdT * 4, kP = kTileP, kPStride = kPanel;
    static constexpr int kBytes = kT + 2 * kTBytes + 1024;   // and to align it
    static_assert(kT % 1024 == 0 && kTBytes % 1024 == 0 && kTBytes >= kTileZ, "images in T's place");
};

// A chunk of a key head: the products that meet tokens with tokens only. What bounds it: instructions, issued 40 % of
// the time by the 16 warps that shared memory leaves room for (three CTAs an SM at 80 registers a thread spilled and
// gained nothing); 832 CTAs 77 us. K stays in shared memory from the convolution to Z.
template <bool kBf16>
__global__ void __launch_bounds__(kThreads, 2) k_gdn_chunks(const __grid_constant__ GdnArgs a) {
    extern __shared__ uint8_t raw_smem[];
    uint8_t *smem = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);   // the swizzle goes by the address
    __shared__ __align__(16) float2 G[2][kC];
    __shared__ __align__(16) float beta[2][kC], mid[2][kC / 2];   // mid: e^{G_31 - G_s}
    __shared__ int scan[kWarps], scan_all[kWarps], found[5], stop;
    __shared__ uint64_t products, z_done[2];
    __shared__ uint32_t tmem_at;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Rows of the grid: the key heads, and spread among them (waiting for memory, where the others wait for the
    // arithmetic) the value heads' norm of part - 2, whose scan is complete, an eighth of a chunk each. The last CTA
    // returns when the scan of part - 1 has ended, and so does the launch: what waits for it has all of the
    // parts before.
    const int gating = a.part >= 2 ? kGateRows : 0, y = blockIdx.y;
    const int gate = y * gating / (int)gridDim.y;   // norm rows before this one
    const bool is_gate = (y + 1) * gating / (int)gridDim.y > gate;
    const int kh = y - gate, part = is_gate ? a.part - 2 : a.part;
    const bool last_cta = a.part > 0 && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1;
    pdl_trigger();

    // ---- the chunk's sequence, and its place in it
    if (tid == 0) found[0] = -1;
    {
        const int chunk = blockIdx.x;
        const int per = (a.num_seqs + kThreads - 1) / kThreads;
        const int first = min(a.num_seqs, tid * per), last = min(a.num_seqs, first + per);
        int own = 0, all = 0, row = 0, rows = 0, from = 0;   // chunks of this part, of all parts; the last sequence's
        auto one = [&](int b) {
            row = max(0, min(a.cu_rows[b], a.total_rows));
            rows = max(0, min(a.cu_rows[b + 1], a.total_rows) - row);
            const int n = (rows + kC - 1) / kC;
            from = part_first(a, n, part);
            all += n;
            return part_first(a, n, part + 1) - from;
        };
        for (int b = first; b < last; ++b) own += one(b);
        int inc = own, inc_all = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o), w = __shfl_up_sync(0xffffffffu, inc_all, o);
            if (lane >= o) inc += v, inc_all += w;
        }
        if (lane == 31) scan[warp] = inc, scan_all[warp] = inc_all;
        __syncthreads();
        int before = inc - own, before_all = inc_all - all;
        for (int w = 0; w < warp; ++w) before += scan[w], before_all += scan_all[w];
        if (chunk >= before && chunk < before + own) {
            all = before_all;
            int b = first, n = own;
            if (per > 1)
                for (; b < last; ++b) {
                    const int at = all;
                    n = one(b);
                    if (chunk < before + n) {
                        all = at;
                        break;
                    }
                    before += n;
                }
            found[0] = b, found[1] = chunk - before + from, found[2] = row, found[3] = rows, found[4] = all;
        }
        __syncthreads();
    }
    const int b = found[0];
    if (b < 0) {   // fewer chunks than the grid has room for
        if (last_cta) pdl_wait();
        return;
    }
    const int row0 = found[2], in_seq = found[1] * kC, n = min(kC, found[3] - in_seq);
    if (is_gate) {
        gate_rows<kBf16>(a, row0 + in_seq, row0 + in_seq + n, gate * kWarps + warp, kGateRows * kWarps);
        if (last_cta) pdl_wait();
        return;
    }
    const int chunk = found[4] + found[1];   // in the workspace: over all chunks of all sequences
    if ((unsigned)chunk >= (unsigned)a.room) {
        if (last_cta) pdl_wait();
        return;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(&tmem_at)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 0) {
        mbar_init(&products, 1);
        mbar_init(&z_done[0], 1);
        mbar_init(&z_done[1], 1);
        mbar_fence_init();
        stop = 0;
    }
    const uint32_t sm = smem_u32(smem);

    const int ratio = a.value_heads / a.key_heads;
    const int half = warp >> 2, q4 = warp & 3, t128 = tid & 127;
    // G: the running sum of log g, in two floats (sums run to -1000 and beyond, and it is differences
    // that count); a warp per head, on different schedulers, two tokens a lane
    const bool gate_warp = warp == 3 || warp == 6;
    using Raw1 = typename std::conditional<kBf16, uint16_t, float>::type;
    Raw1 al_raw[2] = {}, be_raw[2] = {};
    float a_log = 0.f;
    uint16_t dt_raw = 0;
    auto load_gates = [&](int v0) {
        if (!gate_warp || v0 + half >= ratio) return;
        const int vh = kh * ratio + v0 + half;
        a_log = a.A_log[vh];
        dt_raw = a.dt_bias[vh];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const long long at = (long long)(row0 + in_seq + min(2 * lane + j, n - 1)) * a.ab_stride + vh;
            al_raw[j] = static_cast<const Raw1 *>(a.alpha)[at];
            be_raw[j] = static_cast<const Raw1 *>(a.beta)[at];
        }
    };
    auto make_gates = [&](int v0) {
        if (!gate_warp || v0 + half >= ratio) return;
        const float rate = -expf(a_log), dt = bf16_to_f32(dt_raw);
        double g[2];
        float bt[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int t = 2 * lane + j;
            float al, be;
            if constexpr (kBf16)
                al = bf16_to_f32(al_raw[j]), be = bf16_to_f32(be_raw[j]);
            else
                al = al_raw[j], be = be_raw[j];
            const float lg = t < n ? rate * softplus(al + dt) : 0.f;
            // e^-1000 is zero too, and sums of it keep the decays beside it: with 1e12 or an infinity, the differences
            // between the tokens behind would be lost, or NaN
            g[j] = lg < -1000.f ? -1000.f : lg;
            bt[j] = t < n ? sigmoidf_(be) : 0.f;
        }
        double inc = g[0] + g[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        const double first = inc - g[1];
        const float h0 = (float)first, h1 = (float)inc;
        *reinterpret_cast<float4 *>(&G[half][2 * lane]) = make_float4(h0, (float)(first - h0), h1, (float)(inc - h1));
        *reinterpret_cast<float2 *>(&beta[half][2 * lane]) = make_float2(bt[0], bt[1]);
        const double g31 = __shfl_sync(0xffffffffu, inc, 15);
        if (lane < 16) *reinterpret_cast<float2 *>(&mid[half][2 * lane]) = make_float2(__expf((float)(g31 - first)), __expf((float)(g31 - inc)));
    };

    // ---- convolution, SiLU and norm of q and k: a warp takes 8 tokens, a lane 4 channels of each; four tokens of
    // q or k at a time, the rows of the next four asked for before. Rows beyond the sequence's ends are asked
    // for at its ends, and replaced.
    {
        using Raw4 = typename std::conditional<kBf16, uint2, float4>::type;
        using Raw = typename std::conditional<kBf16, uint16_t, float>::type;
        const int t0 = 8 * warp;
        Raw4 next[7];
        uint2 w_next[4];
        auto channel = [&](int side) { return (side * a.key_heads + kh) * kD + 4 * lane; };
        auto load_rows = [&](int batch) {
            const Raw *p = static_cast<const Raw *>(a.qkv) + channel(batch >> 1);
#pragma unroll
            for (int i = 0; i < 7; ++i) {
                const int r = min(max(in_seq + t0 + 4 * (batch & 1) + i - 3, 0), in_seq + n - 1);
                next[i] = *reinterpret_cast<const Raw4 *>(p + (long long)(row0 + r) * a.qkv_stride);
            }
            if ((batch & 1) == 0)
#pragma unroll
                for (int j = 0; j < 4; ++j) w_next[j] = *reinterpret_cast<const uint2 *>(a.conv_w + 4ll * (channel(batch >> 1) + j));
        };
        load_gates(0);
        load_rows(0);
        uint64_t w[2][4];   // of two channels, by tap
#pragma unroll
        for (int batch = 0; batch < 4; ++batch) {
            const int side = batch >> 1, i0 = 4 * (batch & 1);
            uint64_t x[7][2];
#pragma unroll
            for (int i = 0; i < 7; ++i) {
                if constexpr (kBf16) {
                    x[i][0] = pair(bf16_lo(next[i].x), bf16_hi(next[i].x));
                    x[i][1] = pair(bf16_lo(next[i].y), bf16_hi(next[i].y));
                } else {
                    x[i][0] = pair(next[i].x, next[i].y);
                    x[i][1] = pair(next[i].z, next[i].w);
                }
            }
            if (i0 == 0)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint2 u = w_next[2 * j], v = w_next[2 * j + 1];
                    w[j][0] = pair(bf16_lo(u.x), bf16_lo(v.x)), w[j][1] = pair(bf16_hi(u.x), bf16_hi(v.x));
                    w[j][2] = pair(bf16_lo(u.y), bf16_lo(v.y)), w[j][3] = pair(bf16_hi(u.y), bf16_hi(v.y));
                }
            if (batch < 3) load_rows(batch + 1);
            if (in_seq == 0 && warp == 0 && i0 == 0) {   // the inputs before the sequence
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    float4 c = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (a.conv_in != nullptr)
                        c = *reinterpret_cast<const float4 *>(a.conv_in + ((long long)b * 3 + i) * a.channels + channel(side));
                    x[i][0] = pair(c.x, c.y), x[i][1] = pair(c.z, c.w);
                }
            }
            const float scale = side ? kScaleK * 0.08838834764831845f : kScaleQ / kD;
            uint64_t y[4][2];
            float ss[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint64_t sum2 = 0;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint64_t v = fma2(x[i + 3][j], w[j][3], fma2(x[i + 2][j], w[j][2], fma2(x[i + 1][j], w[j][1], mul2(x[i][j], w[j][0]))));
                    y[i][j] = t0 + i0 + i < n ? silu2(v) : 0;
                    sum2 = fma2(y[i][j], y[i][j], sum2);
                }
                float s0, s1;
                unpair(sum2, s0, s1);
                ss[i] = s0 + s1;
            }
            // the four sums over the warp together: a lane keeps half of them in each of two exchanges, so
            // that lane l ends with that of token l & 3 and takes its root
            const bool odd = lane & 1, upper = lane & 2;
            const float a0 = (odd ? ss[1] : ss[0]) + __shfl_xor_sync(0xffffffffu, odd ? ss[0] : ss[1], 1);
            const float a1 = (odd ? ss[3] : ss[2]) + __shfl_xor_sync(0xffffffffu, odd ? ss[2] : ss[3], 1);
            float sum = (upper ? a1 : a0) + __shfl_xor_sync(0xffffffffu, upper ? a0 : a1, 2);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float root = rsqrtf(sum / kD + 1e-12f) * scale;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t0 + i0 + i;
                const float inv = __shfl_sync(0xffffffffu, root, i);
                uint32_t h0, l0, h1, l1;
                const uint32_t at = at_kq(side ? t : kC + t, lane >> 1) + (lane & 1) * 8;
                split2(mul2(y[i][0], pair(inv, inv)), h0, l0);
                split2(mul2(y[i][1], pair(inv, inv)), h1, l1);
                *reinterpret_cast<uint2 *>(smem + at) = make_uint2(h0, h1);
                *reinterpret_cast<uint2 *>(smem + kTileX + at) = make_uint2(l0, l1);
            }
        }
    }
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    if (warp == 0) {
        // K K^T over Q K^T: the products of [K; Q] with K, as the scan takes its operands; and the tile images
        // into the workspace meanwhile
        const uint32_t one = elect_lane(), tm = __shfl_sync(0xffffffffu, tmem, 0);
        if (one) bulk_s2g(a.kq + ((long long)chunk * a.key_heads + kh) * 2 * kTileX, smem, 2 * kTileX);
#pragma unroll
        for (int x = 0; x < 3; ++x)   // hi hi, lo hi, hi lo
#pragma unroll
            for (int k = 0; k < kD / 16; ++k) {
                const uint32_t at = sm + (k >> 2) * kPanel + (k & 3) * 32;
                mma_one(tm, sw128_desc(at + (x == 1) * kTileX), sw128_desc(at + (x == 2) * kTileX), idesc_f16(0, 0, kC),
                        x + k > 0 ? 1u : 0u, one);
            }
        commit_one(&products, one);
    }
    make_gates(0);
    wait_bar(&products, 0, &stop);
    tc_fence_after();

    // ---- the value heads of the key head, two at a time: four warps each
    auto diff = [&](int t, int s) { return (G[half][t].x - G[half][s].x) + (G[half][t].y - G[half][s].y); };
    for (int v0 = 0; v0 < ratio; v0 += 2) {
        const bool on = v0 + half < ratio;
        const int vh = kh * ratio + v0 + half;
        float *T = reinterpret_cast<float *>(smem + ChunkSmem::kT + half * ChunkSmem::kTBytes);
        uint8_t *P = smem + ChunkSmem::kP + half * ChunkSmem::kPStride;   // hi; lo kTileX behind it
        float *scratch = T + 32 + 8 * q4;   // 8 columns of T's quarter above the diagonal, which is not used otherwise
        auto head_sync = [&] { bar_sync(1 + half, 128); };
        // what was copied out of this shared memory has been read
        if (v0 == 0 ? warp == 0 : t128 == 0) bulk_wait_read();
        if (v0 > 0) {
            load_gates(v0);
            make_gates(v0);
        }
        __syncthreads();   // and the products that read K and Q are complete
        // M below the diagonal, P with its diagonal: a thread a row (of K K^T: M; of Q K^T: P), as the products lie in
        // tensor memory, four warps a head. What is above the 32 x 32 blocks on the diagonal is not read. The block
        // below them: e^{G_t - G_s} = e^{G_t - G_31} e^{G_31 - G_s}, neither above 1.
        if (on) {
            const int block = warp & 1, t = 32 * block + lane;
            const bool is_q = warp & 2;
            const float2 g = G[half][t], g31 = G[half][31];
            // Q K^T keeps the scale of q: P does
            const float scale = is_q ? 1.f / kScaleK : beta[half][t] * (1.f / (kScaleK * kScaleK));
            const float far = scale * __expf((g.x - g31.x) + (g.y - g31.y));
#pragma unroll 2
            for (int s0 = 0; s0 < 32 * block + 32; s0 += 16) {
                float x[16];
                uint64_t y[8];
                tc_ld16(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + s0, reinterpret_cast<uint32_t *>(x));
                tc_wait_ld();
                if (s0 < 32 * block) {
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const ulonglong2 e = *reinterpret_cast<const ulonglong2 *>(&mid[half][s0 + 2 * j]);
                        y[j] = mul2(mul2(pair(x[2 * j], x[2 * j + 1]), e.x), pair(far, far));
                        y[j + 1] = mul2(mul2(pair(x[2 * j + 2], x[2 * j + 3]), e.y), pair(far, far));
                    }
                } else {
                    const int seen = t - s0 + (is_q ? 1 : 0);   // columns
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float4 gs = *reinterpret_cast<const float4 *>(&G[half][s0 + j]);   // of two columns
                        const float e0 = __expf((g.x - gs.x) + (g.y - gs.y)), e1 = __expf((g.x - gs.z) + (g.y - gs.w));
                        // e at most 1: 2^-22 or so of it, and of 1
                        y[j / 2] = pair(j < seen ? scale * e0 * x[j] : 0.f, j + 1 < seen ? scale * e1 * x[j + 1] : 0.f);
                    }
                }
                if (!is_q) {
                    ulonglong2 *to = reinterpret_cast<ulonglong2 *>(T + t * kLdT + s0);
#pragma unroll
                    for (int j = 0; j < 4; ++j) to[j] = make_ulonglong2(y[2 * j], y[2 * j + 1]);
                } else {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) split2(y[4 * q + j], hi[j], lo[j]);
                        const int at = at128(t, s0 / 8 + q);
                        *reinterpret_cast<uint4 *>(P + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4 *>(P + kTileX + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            }
        }
        __syncthreads();
        if (on) {
            float *gates = reinterpret_cast<float *>(a.gates + ((long long)chunk * a.value_heads + vh) * kGates);
            if (t128 < kC) gates[t128] = expf(G[half][t128].x + G[half][t128].y);
            // (I + M)^-1. The 16 x 16 blocks on the diagonal by substitution, a lane per column, ..
            if (lane < 16) {
                const float *m = T + 16 * q4 * kLdT + 16 * q4;
                float x[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = i == lane ? 1.f : 0.f;
#pragma unroll
                for (int i = 1; i < 16; ++i)
#pragma unroll
                    for (int k = 0; k < i; k += 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(m + i * kLdT + k);
                        x[i] = fmaf(-v.x, x[k], x[i]);
                        if (k + 1 < i) x[i] = fmaf(-v.y, x[k + 1], x[i]);
                        if (k + 2 < i) x[i] = fmaf(-v.z, x[k + 2], x[i]);
                        if (k + 3 < i) x[i] = fmaf(-v.w, x[k + 3], x[i]);
                    }
                __syncwarp(0xffffu);
                float *to = T + 16 * q4 * kLdT + 16 * q4 + lane;
#pragma unroll
                for (int i = 0; i < 16; ++i) to[i * kLdT] = x[i];
            }
            head_sync();
            // .. then the block below of each 32 x 32 block, and of the whole: -T_22 (M_21 T_11), 8 columns a warp,
            // four of a row a lane (of two rows, in the second)
            const int lr = lane & 15, lc = (lane >> 4) * 4;
            auto add = [&](float *acc, const float *m, const float *u, int ldu) {   // acc += m[0..3] u[0..3][0..3]
                const float4 f = *reinterpret_cast<const float4 *>(m);
                const float mm[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float4 v = *reinterpret_cast<const float4 *>(u + k * ldu);
                    acc[0] = fmaf(mm[k], v.x, acc[0]), acc[1] = fmaf(mm[k], v.y, acc[1]);
                    acc[2] = fmaf(mm[k], v.z, acc[2]), acc[3] = fmaf(mm[k], v.w, acc[3]);
                }
            };
            auto put = [&](float *to, const float *v, float sign) {
                *reinterpret_cast<float4 *>(to) = make_float4(sign * v[0], sign * v[1], sign * v[2], sign * v[3]);
            };
            {
                const int d = 32 * (q4 >> 1), col = d + 8 * (q4 & 1) + lc;
                float acc[4] = {};
#pragma unroll
                for (int k = 0; k < 16; k += 4) add(acc, T + (d + 16 + lr) * kLdT + d + k, T + (d + k) * kLdT + col, kLdT);
                put(scratch + lr * kLdT + lc, acc, 1.f);
                head_sync();   // M_21 is read
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[x] = 0.f;
#pragma unroll
                for (int k = 0; k < 16; k += 4) add(acc, T + (d + 16 + lr) * kLdT + d + 16 + k, scratch + k * kLdT + lc, kLdT);
                put(T + (d + 16 + lr) * kLdT + col, acc, -1.f);
                head_sync();
            }
            {
                const int col = 8 * q4 + lc;
                float x0[4] = {}, x1[4] = {};   // rows lr, lr + 16
#pragma unroll 2
                for (int k = 8 * q4; k < 32; k += 4) {   // T_11 is zero above its diagonal
                    add(x0, T + (32 + lr) * kLdT + k, T + k * kLdT + col, kLdT);
                    add(x1, T + (48 + lr) * kLdT + k, T + k * kLdT + col, kLdT);
                }
                put(scratch + lr * kLdT + lc, x0, 1.f);
                put(scratch + (lr + 16) * kLdT + lc, x1, 1.f);
                head_sync();
#pragma unroll
                for (int x = 0; x < 4; ++x) x0[x] = x1[x] = 0.f;
#pragma unroll 2
                for (int k = 0; k < 16; k += 4) {
                    add(x0, T + (32 + lr) * kLdT + 32 + k, scratch + k * kLdT + lc, kLdT);
                    add(x1, T + (48 + lr) * kLdT + 32 + k, scratch + k * kLdT + lc, kLdT);
                }
#pragma unroll 2
                for (int k = 16; k < 32; k += 4) add(x1, T + (48 + lr) * kLdT + 32 + k, scratch + k * kLdT + lc, kLdT);
                put(T + (32 + lr) * kLdT + col, x0, -1.f);
                put(T + (48 + lr) * kLdT + col, x1, -1.f);
                head_sync();
            }
            // T b in T's place, for P T b (a thread holds four 16-byte pieces of it)
            uint8_t *to = a.tp + ((long long)chunk * a.value_heads + vh) * kTileZP, *TB = reinterpret_cast<uint8_t *>(T);
            uint64_t tb[4][4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int i = t128 + 128 * x, t = i >> 3, s0 = (i & 7) * 8;
#pragma unroll
                for (int j = 0; j < 4; ++j) tb[x][j] = 0;
                if (s0 <= t) {   // T holds nothing above its blocks on the diagonal, and zeros within them
                    const ulonglong2 t0 = *reinterpret_cast<const ulonglong2 *>(T + t * kLdT + s0);
                    const ulonglong2 t1 = *reinterpret_cast<const ulonglong2 *>(T + t * kLdT + s0 + 4);
                    const ulonglong2 b0 = *reinterpret_cast<const ulonglong2 *>(&beta[half][s0]);
                    const ulonglong2 b1 = *reinterpret_cast<const ulonglong2 *>(&beta[half][s0 + 4]);
                    tb[x][0] = mul2(t0.x, b0.x), tb[x][1] = mul2(t0.y, b0.y);
                    tb[x][2] = mul2(t1.x, b1.x), tb[x][3] = mul2(t1.y, b1.y);
                }
            }
            auto put_tb = [&](bool decayed) {   // its hi and lo; with row t times e^{G_63 - G_t}
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int i = t128 + 128 * x, t = i >> 3, at = at128(t, i & 7);
                    const float left = decayed ? __expf(diff(kC - 1, t)) : 1.f;
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) split2(decayed ? mul2(tb[x][j], pair(left, left)) : tb[x][j], h[j], l[j]);
                    *reinterpret_cast<uint4 *>(TB + at) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(TB + kTileP + at) = make_uint4(l[0], l[1], l[2], l[3]);
                }
            };
            head_sync();
            put_tb(false);
            head_sync();
            // P T b: 16 rows a warp, the columns in pairs of 8; lower triangular as both are, so the two heads'
            // blocks of rows run in opposite orders over the warp schedulers
            const int rb = half ? 3 - q4 : q4;
            float c[4][2][4] = {};
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int k = j; k < 4; ++k)
                    if (k <= rb) {
                        uint32_t ah[4], al[4], bh[4], bl[4];
                        const uint32_t pa = smem_u32(P) + at128(16 * rb + (lane & 15), 2 * k + (lane >> 4));
                        const uint32_t pb = smem_u32(TB) + at128(16 * k + (lane & 15), 2 * j + (lane >> 4));
                        ldsm4(pa, ah);
                        ldsm4(pa + kTileX, al);
                        ldsm4t(pb, bh);
                        ldsm4t(pb + kTileP, bl);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            mma_f16(c[j][x], al, bh[2 * x], bh[2 * x + 1]);
                            mma_f16(c[j][x], ah, bl[2 * x], bl[2 * x + 1]);
                            mma_f16(c[j][x], ah, bh[2 * x], bh[2 * x + 1]);
                        }
                    }
            __syncwarp();   // a warp reads and writes its own rows of P
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t h[4], l[4];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    split2(c[j][x][0], c[j][x][1], h[2 * x], l[2 * x]);
                    split2(c[j][x][2], c[j][x][3], h[2 * x + 1], l[2 * x + 1]);
                }
                const uint32_t at = smem_u32(P) + at128(16 * rb + (lane & 15), 2 * j + (lane >> 4));
                stsm4(at, h[0], h[1], h[2], h[3]);
                stsm4(at + kTileX, l[0], l[1], l[2], l[3]);
            }
            fence_async_smem();
            head_sync();
            if (t128 == 0)
                for (int x = 0; x < 2; ++x) bulk_s2g(to + 2 * kTileZ + x * kTileP, P + x * kTileX, kTileP);
            // Z = K^T (e^{G_63 - G} T b), with which the state takes in R in one product
            put_tb(true);
            fence_async_smem();
            tc_fence_before();
            head_sync();
            const uint32_t acc = tmem + kC + half * kC;
            if (q4 == 0) {
                tc_fence_after();
                const uint32_t one = elect_lane(), tm = __shfl_sync(0xffffffffu, acc, 0);
                const uint32_t tb_at = __shfl_sync(0xffffffffu, smem_u32(TB), 0);
#pragma unroll
                for (int x = 0; x < 3; ++x)   // hi hi, lo hi, hi lo
#pragma unroll
                    for (int k = 0; k < kC / 16; ++k)
                        mma_one(tm, desc_rows(sm + (x == 1) * kTileX + k * 2048, kPanel), desc_rows(tb_at + (x == 2) * kTileP + k * 2048, 0),
                                idesc_f16(1, 1, kC), x + k > 0 ? 1u : 0u, one);
                commit_one(&z_done[half], one);
            }
            if (t128 == 0) bulk_wait_read();   // P T b, which Z's lo goes over
            wait_bar(&z_done[half], (v0 >> 1) & 1, &stop);
            tc_fence_after();
            head_sync();
            if (stop && t128 < kC) gates[t128] = NAN;   // products that never came must not pass for an answer
            const int dim = 32 * q4 + lane;
            uint8_t *z_lo = P + (dim >> 6) * kTileX;   // rows 0-63 where P's hi was, 64-127 where its lo was
#pragma unroll
            for (int c16 = 0; c16 < 4; ++c16) {
                float x[16];
                tc_ld16(acc + ((uint32_t)(32 * q4) << 16) + 16 * c16, reinterpret_cast<uint32_t *>(x));
                tc_wait_ld();
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) split2(x[8 * q + 2 * j], x[8 * q + 2 * j + 1], h[j], l[j]);
                    *reinterpret_cast<uint4 *>(TB + at128(dim, 2 * c16 + q)) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(z_lo + at128(dim & 63, 2 * c16 + q)) = make_uint4(l[0], l[1], l[2], l[3]);
                }
            }
            fence_async_smem();
            tc_fence_before();
            head_sync();
            if (t128 == 0) {
                bulk_s2g(to, TB, kTileZ);
                bulk_s2g(to + kTileZ, P, kTileP);
                bulk_s2g(to + kTileZ + kTileP, P + kTileX, kTileP);
            }
        }
    }
    if (t128 == 0) bulk_wait_read();   // the shared memory stays until it is copied
    tc_fence_before();
    __syncthreads();
    if (stop && warp == 0) {
        settle(&products);
        settle(&z_done[0]);
        settle(&z_done[1]);
    }
    tc_fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem));
    if (last_cta) pdl_wait();
}

// ---- scan -------------------------------------------------------------------------------------------

struct ScanSmem {
    static constexpr int kStage = 2 * kTileX;                       // K over Q of a chunk, hi and lo; two of them
    static constexpr int kZ = 2 * kStage;                           // Z, hi and lo
    static constexpr int kS = kZ + 2 * kTileZ, kTileS = kD * 128;   // the state: [dim][64 columns], hi and lo
    // R: [token][64 columns], hi and lo; before it V (fp32), every value in the bytes of the thread that makes R of it
    static constexpr int kR = kS + 2 * kTileS, kTileR = kC * 128;
    static constexpr int kP = kR + 2 * kTileR;                      // P T b, hi and lo
    static constexpr int kGate = kP + 2 * kTileP;                   // gates of two chunks
    static constexpr int kBytes = kGate + 2 * kGates;
};

// byte of V's column c (a multiple of 2; 4 in a piece) of token t in R's place: 16 columns in two pieces each of
// the hi and the lo image
__device__ __forceinline__ uint32_t v_at(int t, int c) {
    return ((c >> 3) & 1) * (kC * 128) + at128(t, 2 * (c >> 4) + ((c >> 2) & 1)) + (c & 3) * 4;
}

struct ScanShared {
    uint64_t kq_full[2], zp_full, d, zr, pr, r_ready, s_ready, v_ready;   // d: [K; Q] S^T, zr: Z R, pr: P T b R
    int vmax[3], first_chunk, stop;
    uint32_t tmem;
    __align__(16) float s_max[2][8];   // largest |S| of a row warp, of the state before a chunk, by the chunk's parity
};

__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }
// The scale 2^-e for values whose square is at most `square`: they come below 2^13, so that fp16 holds
// them and its parts reach 2^-37 of that.
__device__ __forceinline__ int exponent_of(float square) {
    const int e = (((__float_as_int(square) >> 23) - 127 + 2) >> 1) - 13;   // 2^(e + 13) > sqrt(square)
    return min(100, max(-100, e));
}

// Threads 0-255: row r = 32 (warp % 4) + lane of the 128, columns 32 (warp / 4) .. + 31 of the CTA's 64.
// Rows 0-63 are tokens (K's rows: R), rows 64-127 are tokens too (Q's rows: the output), and all of
// them are dims of the state. Warp 8 issues the MMAs, warps 9-12 convolve V a chunk ahead.
template <bool kBf16>
__global__ void __launch_bounds__(kScanThreads, 1) k_gdn_scan(const __grid_constant__ GdnArgs a) {
    using L = ScanSmem;
    extern __shared__ uint8_t raw_smem[];
    __shared__ ScanShared S;
    uint8_t *smem = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, vh = blockIdx.y, kh = vh / (a.value_heads / a.key_heads);
    const uint32_t sm = smem_u32(smem);
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) mbar_init(&S.kq_full[i], 1);
        for (int i = 0; i < 3; ++i) S.vmax[i] = 0;
        mbar_init(&S.d, 1);
        mbar_init(&S.zr, 1);
        mbar_init(&S.pr, 1);
        mbar_init(&S.zp_full, 1);
        mbar_init(&S.r_ready, 8);
        mbar_init(&S.s_ready, 8);
        mbar_init(&S.v_ready, 4);
        mbar_fence_init();
        S.first_chunk = S.stop = 0;
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&S.tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // The sequence, and the chunks of those before it. The longest first, as far as a lane a sequence goes: CTAs
    // begin as SMs become free
    int b = blockIdx.z, first_chunk = 0;
    if (a.num_seqs <= 32) {
        const int n = lane < a.num_seqs ? seq_chunks(a, lane) : -1;
        int rank = 0;
        for (int i = 0; i < a.num_seqs; ++i) {
            const int v = __shfl_sync(0xffffffffu, n, i);
            rank += v > n || (v == n && i < lane);
        }
        b = __ffs(__ballot_sync(0xffffffffu, lane < a.num_seqs && rank == b)) - 1;
        first_chunk = __reduce_add_sync(0xffffffffu, lane < b ? n : 0);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = S.tmem;
    // This part's chunks, and with them the parts before, are complete: for the warp that copies them, and from the
    // second part on for the state too. The inputs were there when the first part's chunks were begun.
    if (a.part > 0 || warp == 8) pdl_wait();
    if (warp == 8) pdl_trigger();
    if (a.num_seqs > 32) {
        int before = 0;
        for (int i = tid; i < b; i += kScanThreads) before += seq_chunks(a, i);
        if (before) atomicAdd(&S.first_chunk, before);   // integers: the order does not matter
        __syncthreads();
        first_chunk = S.first_chunk;
    }
    const int all = seq_chunks(a, b), from = part_first(a, all, a.part);
    const int row0 = seq_first(a, b) + from * kC, rows = seq_rows(a, b) - from * kC;   // from this part's first on
    const int wg = warp >> 2, r = 32 * (warp & 3) + lane, c0 = 32 * wg;
    const bool is_q = warp < 8 && (warp & 3) >= 2;

    const long long chunk0 = (long long)first_chunk + from;
    const int here = part_first(a, all, a.part + 1) - from;
    const int chunks = chunk0 < 0 || chunk0 + here > a.room ? 0 : here;   // not beyond the workspace, whatever cu_rows holds

    auto wait_for = [&](uint64_t *bar, uint32_t parity) { return wait_bar(bar, parity, &S.stop, a.tries); };
    if (warp == 8) {
        // ---- copies and MMAs; every value is the same in all lanes
        const uint32_t one = elect_lane(), tm = __shfl_sync(0xffffffffu, tmem, 0);
        const int n = __shfl_sync(0xffffffffu, chunks, 0);
        const uint64_t keep = policy_evict_normal();
        auto copy_kq = [&](int c) {
            if (!one) return;
            uint64_t *bar = &S.kq_full[c & 1];
            mbar_arrive_expect_tx(bar, L::kStage + kGates);
            bulk_g2s(smem + (c & 1) * L::kStage, a.kq + ((chunk0 + c) * a.key_heads + kh) * 2 * kTileX, L::kStage, bar, keep);
            bulk_g2s(smem + L::kGate + (c & 1) * kGates, a.gates + ((chunk0 + c) * a.value_heads + vh) * kGates, kGates, bar, keep);
        };
        auto zp = [&](int c) { return a.tp + ((chunk0 + c) * a.value_heads + vh) * kTileZP; };
        auto copy_z = [&](int c) {
            if (!one) return;
            mbar_arrive_expect_tx(&S.zp_full, kTileZP);
            bulk_g2s(smem + L::kZ, zp(c), 2 * kTileZ, &S.zp_full, keep);
        };
        auto copy_p = [&](int c) {
            if (one) bulk_g2s(smem + L::kP, zp(c) + 2 * kTileZ, 2 * kTileP, &S.zp_full, keep);
        };
        auto wait = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_for(bar, parity)); };
        // The products of kSteps k-steps: A's hi with B's hi and lo, which lie side by side as 128 columns (one
        // reading of A for both: these are bound by shared memory), then A's lo with B's hi onto the first 64.
        // A's address of k-step k, part (0 hi, 1 lo); B's of k-step k.
        auto issue = [&](uint32_t d, auto steps, auto at_a, auto at_b) {
            constexpr int kSteps = decltype(steps)::value;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) mma_one(d, at_a(k, 0), at_b(k), idesc_f16(0, 1, 2 * kN), k > 0 ? 1u : 0u, one);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) mma_one(d, at_a(k, 1), at_b(k), idesc_f16(0, 1, kN), 1u, one);
        };
        if (n > 0) {
            copy_kq(0);
            copy_z(0);
            copy_p(0);
        }
        for (int c = 0; c < n; ++c) {
            const uint32_t st = sm + (c & 1) * L::kStage;
            auto state_rows = [&](int k) { return desc_rows(sm + L::kS + k * 2048, L::kTileS); };
            auto token_rows = [&](int k) { return desc_rows(sm + L::kR + k * 2048, L::kTileR); };
            if (!wait(&S.kq_full[c & 1], (c >> 1) & 1) || !wait(&S.s_ready, c & 1)) break;
            tc_fence_after();
            issue(tm + (c & 1) * 2 * kN, std::integral_constant<int, kD / 16>{},
                  [&](int k, int part) { return sw128_desc(st + part * kTileX + (k >> 2) * kPanel + (k & 3) * 32); }, state_rows);
            commit_one(&S.d, one);
            // the other stage was last read by the product of the chunk before. The copies are timed to land while
            // rows are at work: beside a product they take shared memory from it
            if (c + 1 < n) copy_kq(c + 1);
            if (!wait(&S.zp_full, c & 1) || !wait(&S.r_ready, c & 1)) break;
            tc_fence_after();
            issue(tm + 4 * kN, std::integral_constant<int, kC / 16>{},
                  [&](int k, int part) { return sw128_desc(sm + L::kZ + part * kTileZ + k * 32); }, token_rows);
            commit_one(&S.zr, one);
            // P T b as the lower 64 of 128 rows, where Q S^T is; the upper ones (R, which is before it) are not read
            issue(tm + 6 * kN, std::integral_constant<int, kC / 16>{},
                  [&](int k, int part) { return sw128_desc(sm + L::kP + (part - 1) * kTileP + k * 32); }, token_rows);
            commit_one(&S.pr, one);
            if (c + 1 < n) {
                if (!wait(&S.zr, c & 1)) break;
                copy_z(c + 1);
                if (!wait(&S.pr, c & 1)) break;
                copy_p(c + 1);
            }
        }
    } else if (warp >= 9) {
        // ---- V of a chunk: a lane two of 32 channels (warps 9, 10: the first 32) and 16 tokens (lanes 0-15 the
        // first 16 of the warp's 32, lanes 16-31 the others). The inputs are loaded a chunk ahead and stay as they
        // are until they are used (a conversion would wait for them).
        using Raw2 = typename std::conditional<kBf16, uint32_t, float2>::type;
        using Raw = typename std::conditional<kBf16, uint16_t, float>::type;
        const int vt = 32 * ((warp - 9) & 1) + 16 * (lane >> 4), vc = 32 * ((warp - 9) >> 1) + 2 * (lane & 15);
        const int ch = (2 * a.key_heads + vh) * kD + split * kN + vc;
        Raw2 raw[19];
        uint64_t w[4];   // of both channels, by tap
        {
            const uint2 u = *reinterpret_cast<const uint2 *>(a.conv_w + 4ll * ch);
            const uint2 v = *reinterpret_cast<const uint2 *>(a.conv_w + 4ll * (ch + 1));
            w[0] = pair(bf16_lo(u.x), bf16_lo(v.x)), w[1] = pair(bf16_hi(u.x), bf16_hi(v.x));
            w[2] = pair(bf16_lo(u.y), bf16_lo(v.y)), w[3] = pair(bf16_hi(u.y), bf16_hi(v.y));
        }
        auto load_raw = [&](int c) {   // rows beyond the sequence's ends are asked for at its ends
            const Raw *p = static_cast<const Raw *>(a.qkv) + ch;
#pragma unroll
            for (int i = 0; i < 19; ++i) {
                const int x = min(max(c * kC + vt + i - 3, from > 0 ? -3 : 0), rows - 1);
                raw[i] = *reinterpret_cast<const Raw2 *>(p + (long long)(row0 + x) * a.qkv_stride);
            }
        };
        if (chunks > 0) load_raw(0);
        for (int c = 0; c < chunks; ++c) {
            uint64_t x[19], v[16];
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 19; ++i) {
                if constexpr (kBf16)
                    x[i] = pair(bf16_lo(raw[i]), bf16_hi(raw[i]));
                else
                    x[i] = pair(raw[i].x, raw[i].y);
            }
            if (c + 1 < chunks) load_raw(c + 1);
            if (from + c == 0 && vt == 0)   // the inputs before the sequence
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    float2 f = make_float2(0.f, 0.f);
                    if (a.conv_in != nullptr)
                        f = *reinterpret_cast<const float2 *>(a.conv_in + ((long long)b * 3 + i) * a.channels + ch);
                    x[i] = pair(f.x, f.y);
                }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint64_t y = fma2(x[i + 3], w[3], fma2(x[i + 2], w[2], fma2(x[i + 1], w[1], mul2(x[i], w[0]))));
                v[i] = c * kC + vt + i < rows ? silu2(y) : 0;
                float v0, v1;
                unpair(v[i], v0, v1);
                m = fmaxf(m, fmaxf(fabsf(v0), fabsf(v1)));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            // over R of the chunk before, once the products have read it
            if (c > 0) wait_for(&S.pr, (c - 1) & 1);
            if (lane == 0) atomicMax(&S.vmax[c % 3], __float_as_int(m));
#pragma unroll
            for (int i = 0; i < 16; ++i) *reinterpret_cast<uint64_t *>(smem + L::kR + v_at(vt + i, vc)) = v[i];
            // a barrier whose waits are bounded: arrivals at a named one, once they no longer wait for the rows, would
            // leave the rows waiting
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.v_ready);
        }
    } else {
        // ---- the state: dim r, columns c0 .. c0 + 31; and a bound of |S|^2, per value row
        uint64_t St[16];
        const float *before = a.part > 0 ? a.delta_out : a.delta_in;
        const long long s_at = (((long long)b * a.value_heads + vh) * kD + split * kN + c0) * kD + r;
#pragma unroll
        for (int j = 0; j < 16; ++j) {   // a launch beside this one may have written them
            const float x = before ? __ldcg(before + s_at + (long long)(2 * j) * kD) : 0.f;
            const float y = before ? __ldcg(before + s_at + (long long)(2 * j + 1) * kD) : 0.f;
            St[j] = pair(x, y);
        }
        // The largest |S| of the CTA before chunk c: every warp leaves its own, and reads all of them once it has met
        // a product that all have signalled for since
        auto leave_max = [&](int c) {
            float m = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                float x, y;
                unpair(St[j], x, y);
                m = fmaxf(m, fmaxf(fabsf(x), fabsf(y)));
            }
            m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));   // not negative: ordered as integers
            if (lane == 0) S.s_max[c & 1][warp] = m;
        };
        auto square_of = [&](int c) {   // of a value row's norm, at most
            const float4 x = *reinterpret_cast<const float4 *>(S.s_max[c & 1]), y = *reinterpret_cast<const float4 *>(S.s_max[c & 1] + 4);
            const float m = fmaxf(fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)), fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)));
            return m * m * kD;
        };
        leave_max(0);
        bar_sync(3, 256);
        float bound2 = square_of(0);

        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        // 16 columns (half hf of the thread's 32) of row `row` of an operand image, hi and lo `part` bytes apart
        auto store_half = [&](uint32_t image, int part, int row, int hf, const uint64_t *v) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t h[4], l[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) split2(v[4 * x + y], h[y], l[y]);
                uint8_t *to = smem + image + at128(row, 4 * wg + 2 * hf + x);
                *reinterpret_cast<uint4 *>(to) = make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4 *>(to + part) = make_uint4(l[0], l[1], l[2], l[3]);
            }
        };
        auto signal = [&](uint64_t *bar) {   // this warp's operand rows are written, and its sums are read
            fence_async_smem();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        auto read_half = [&](int which, int hf, uint64_t *v) {   // 16 sums, of both halves of the product
            float x[16], u[16];
            tc_ld16(tmem + lanes + 2 * which * kN + c0 + 16 * hf, reinterpret_cast<uint32_t *>(x));   // hi hi and lo hi
            tc_ld16(tmem + lanes + (2 * which + 1) * kN + c0 + 16 * hf, reinterpret_cast<uint32_t *>(u));   // hi lo
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = add2(pair(x[2 * j], x[2 * j + 1]), pair(u[2 * j], u[2 * j + 1]));
        };
        auto store_state = [&](int e) {
            const uint64_t s = pair(pow2(-e), pow2(-e));
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                uint64_t v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = mul2(St[8 * hf + j], s);
                store_half(L::kS, L::kTileS, r, hf, v);
            }
            signal(&S.s_ready);
        };

        int es = exponent_of(bound2);
        if (chunks > 0) store_state(es);
        const int t = r & 63;   // this row's token
        for (int c = 0; c < chunks; ++c) {
            wait_for(&S.v_ready, c & 1);   // V of the chunk is stored; Q's rows only need its size
            if (tid == 0) S.vmax[(c + 2) % 3] = 0;   // of chunk c - 1: read by all; next added to for chunk c + 2
            const float vm = __int_as_float(S.vmax[c % 3]);
            const float before2 = bound2, in2 = kC * vm * vm;
            const int eu = exponent_of(before2 + in2) + 1;   // max |v| + |S| <= 9/8 of its root
            const float *eg = reinterpret_cast<const float *>(smem + L::kGate + (c & 1) * kGates);
            wait_for(&S.kq_full[c & 1], (c >> 1) & 1);
            const float g = eg[t], keep = eg[kC - 1];
            if (!is_q) {
                // R = V - e^G K S^T, scaled
                const float k0 = -g * pow2(es) * pow2(-eu) * (1.f / kScaleK), s = pow2(-eu);
                const uint64_t kk = pair(k0, k0), ss = pair(s, s);
                wait_for(&S.d, c & 1);
                tc_fence_after();
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint64_t x[8];
                    read_half(c & 1, hf, x);
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const ulonglong2 v = *reinterpret_cast<const ulonglong2 *>(smem + L::kR + v_at(t, c0 + 16 * hf + 2 * j));
                        x[j] = fma2(kk, x[j], mul2(v.x, ss)), x[j + 1] = fma2(kk, x[j + 1], mul2(v.y, ss));
                    }
                    store_half(L::kR, L::kTileR, t, hf, x);
                }
            }
            signal(&S.r_ready);   // the rows of Q: P T b R of the chunk before is read
            const float k0 = g * pow2(es) * pow2(-eu);
            es = exponent_of(keep * before2 * keep + in2);   // in this order: keep^2 alone may be zero when the state is not
            wait_for(&S.zr, c & 1);
            tc_fence_after();
            const float add = pow2(eu) * (1.f / kScaleK);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                uint64_t x[8];
                read_half(2, hf, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) St[8 * hf + j] = fma2(St[8 * hf + j], pair(keep, keep), mul2(x[j], pair(add, add)));
            }
            if (c + 1 < chunks) {
                store_state(es);
                leave_max(c + 1);
                // The next chunk's bound goes by the state before this one, known by now (on the way to the state's
                // scale it would have cost 1.4 % of 16384 rows): by its decay alone it would keep what the rule
                // itself has erased, and the small parts of what is left would be lost
                bound2 = keep * fminf(before2, square_of(c)) * keep + in2;
            }
            if (is_q) {
                // the output before its norm, e^G Q S^T + P U, while the next chunk's first product runs
                wait_for(&S.pr, c & 1);
                tc_fence_after();
                const float s = pow2(eu) * (1.f / kScaleQ);
                const uint64_t kk = pair(k0, k0), ss = pair(s, s);
                const int row = c * kC + t;
                float4 *o = reinterpret_cast<float4 *>(a.o + o_at(a, row0 + row, vh, split * kN + c0));
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint64_t x[8], y[8];
                    read_half(c & 1, hf, x);
                    read_half(3, hf, y);
                    if (row < rows)
#pragma unroll
                        for (int j = 0; j < 8; j += 2) {
                            float4 f;
                            unpair(mul2(fma2(kk, x[j], y[j]), ss), f.x, f.y);
                            unpair(mul2(fma2(kk, x[j + 1], y[j + 1]), ss), f.z, f.w);
                            o[8 * (4 * hf + j / 2)] = f;
                        }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            float x, y;
            unpair(St[j], x, y);
            a.delta_out[s_at + (long long)(2 * j) * kD] = x;
            a.delta_out[s_at + (long long)(2 * j + 1) * kD] = y;
        }
        tc_fence_before();
    }
    __syncthreads();
    if (S.stop) {
        // A copy or product that never came must not pass for an answer: this part's outputs, and the state that it
        // leaves, and with it all behind
        const int n = min(rows, chunks * kC);
        for (int i = tid; i < n * (kN / 4); i += kScanThreads)
            *reinterpret_cast<float4 *>(a.o + o_at(a, row0 + i / (kN / 4), vh, split * kN + 4 * (i % (kN / 4)))) =
                make_float4(NAN, NAN, NAN, NAN);
        for (int i = tid; i < kN * kD; i += kScanThreads)
            a.delta_out[(((long long)b * a.value_heads + vh) * kD + split * kN) * kD + i] = NAN;
        if (warp == 8) {
            settle(&S.kq_full[0]);
            settle(&S.kq_full[1]);
            settle(&S.zp_full);
            settle(&S.d);
            settle(&S.zr);
            settle(&S.pr);
        }
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// ---- finish -------------------------------------------------------------------------------------------

// Gated RMS norm of every value head, 8 rows a warp; then (the last blocks) the last three inputs of every
// channel: after the other launches, so that the states may be updated in place. HBM bound: 4065 rows of 32 heads in
// fp32, 200 MB, 43 us; more warps an SM had to spill and took 55.
template <bool kBf16>
__global__ void __launch_bounds__(kThreads) k_gdn_finish(const __grid_constant__ GdnArgs a, int norm_blocks) {
    const int tid = threadIdx.x, warp = tid >> 5;
    if ((int)blockIdx.x >= norm_blocks) {
        pdl_wait();
        const long long i = (long long)(blockIdx.x - norm_blocks) * kThreads + tid;
        if (i >= (long long)a.num_seqs * a.channels) return;
        const int b = (int)(i / a.channels), c = (int)(i - (long long)b * a.channels);
        const int r0 = seq_first(a, b), n = seq_rows(a, b);
        float v[3];
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            const int r = n + j - 3;   // row of the sequence, negative: of the state before it
            v[j] = r >= 0 ? load_x(a.qkv, (long long)(r0 + r) * a.qkv_stride + c, kBf16)
                          : (a.conv_in ? a.conv_in[((long long)b * 3 + 3 + r) * a.channels + c] : 0.f);
        }
#pragma unroll
        for (int j = 0; j < 3; ++j) a.conv_out[((long long)b * 3 + j) * a.channels + c] = v[j];
        return;
    }
    const int w = blockIdx.x * kWarps + warp, warps = norm_blocks * kWarps;
    if (a.parts == 1) {
        pdl_wait();
        const int first = max(0, min(a.cu_rows[0], a.total_rows)), end = min(a.cu_rows[a.num_seqs], a.total_rows);
        gate_rows<kBf16>(a, first, end, w, warps);
        return;
    }
    for (int p = a.parts - 2; p < a.parts; ++p) {   // the last but one while the scan of the last runs
        if (p == a.parts - 1) pdl_wait();
        for (int b = 0; b < a.num_seqs; ++b) {
            const int chunks = seq_chunks(a, b), c0 = part_first(a, chunks, p), c1 = part_first(a, chunks, p + 1);
            const int row0 = seq_first(a, b);
            gate_rows<kBf16>(a, row0 + c0 * kC, row0 + min(seq_rows(a, b), c1 * kC), w, warps);
        }
    }
}

long long max_chunks(int num_seqs, int total_rows) { return (long long)total_rows / kC + num_seqs; }

// Into how many parts the chunks go. With one, every launch has the machine to itself in turn. A scan that leaves
// more than half of the SMs idle runs beside the launch that prepares the next part, on those SMs; a part more
// costs about 10 us, and what hides is 1 us a chunk of every part but one: best near sqrt(chunks / 10).
// 16384 rows, 16 key and 32 value heads (64 scan CTAs): 1 part 1061 us, 3 892, 4 866, 5 849, 6 862, 8 883, 16 979;
// 4 and 8 heads: 1 part 781 us, 3 720, 5 721, 8 717, 16 749; 1 and 2 heads, with little to hide: 1 part 667 us, 3 670,
// 5 674, 8 690, so the rule costs 1 % there.
// The scan's CTAs come in clusters of two for their place only: those take the two SMs of a TPC. Beside an SM
// that runs the other kernel a CTA of the scan took 20 % longer (1118 us in all, for 992 us in pairs).
int parts_of(const GdnArgs &a, int sms) {
    if (2ll * kSplit * a.value_heads * a.num_seqs > sms) return 1;
    const int chunks = a.total_rows / kC / a.num_seqs;
    int parts = 1;
    while (parts < 16 && 10 * (parts + 1) * (parts + 1) <= chunks) ++parts;
    return parts;
}

template <class K, class... Args>
cudaError_t launch_one(K kernel, dim3 grid, int threads, int smem, cudaStream_t st, bool early, int cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = early ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <bool kBf16>
cudaError_t launch(GdnArgs a, cudaStream_t st) {
    static SmemOnce chunks_smem, scan_smem;
    cudaError_t e = chunks_smem.set(k_gdn_chunks<kBf16>, ChunkSmem::kBytes);
    if (e == cudaSuccess) e = scan_smem.set(k_gdn_scan<kBf16>, ScanSmem::kBytes + 1024);
    int dev = 0, sms = 0;
    if (e == cudaSuccess) e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    a.parts = parts_of(a, sms);
    a.room = (int)max_chunks(a.num_seqs, a.total_rows);
    for (a.part = 0; a.part < a.parts; ++a.part) {
        if (a.total_rows > 0) {
            // a sequence's part has at most its chunks / parts, rounded up
            const long long most = max_chunks(a.num_seqs, a.total_rows) / a.parts + (a.parts > 1 ? a.num_seqs : 0);
            const dim3 grid((unsigned)most, a.key_heads + (a.part >= 2 ? kGateRows : 0));
            e = launch_one(k_gdn_chunks<kBf16>, grid, kThreads, ChunkSmem::kBytes, st, a.part > 0, 1, a);
            if (e != cudaSuccess) return e;
        }
        e = launch_one(k_gdn_scan<kBf16>, dim3(kSplit, a.value_heads, a.num_seqs), kScanThreads, ScanSmem::kBytes + 1024, st,
                       a.total_rows > 0, kSplit, a);
        if (e != cudaSuccess) return e;
    }
    const long long want = ((a.total_rows + 14ll) / 8 * a.value_heads + kWarps - 1) / kWarps;   // a warp 8 rows of a head
    const int norm_blocks = a.total_rows == 0 ? 0 : (int)(want < 2ll * sms ? want : 2ll * sms);
    const long long conv_blocks = ((long long)a.num_seqs * a.channels + kThreads - 1) / kThreads;
    return launch_one(k_gdn_finish<kBf16>, dim3((unsigned)(norm_blocks + conv_blocks)), kThreads, 0, st, true, 1, a, norm_blocks);
}

int check_shape(const nmoe_linear_attn_shape *s) {
    if (s == nullptr) return fail(NMOE_EINVAL, "shape is NULL");
    if (s->key_heads < 1 || s->key_heads > 1024 || s->value_heads < 1 || s->value_heads > 8192 ||
        s->value_heads % s->key_heads != 0)
        return fail(NMOE_EINVAL, "value_heads %d must be a multiple of key_heads %d (at most 1024; 8192 value heads)",
                    s->value_heads, s->key_heads);
    return NMOE_OK;
}

// The parts of the workspace, 256-byte aligned, from `base`; returns their size.
size_t carve(const nmoe_linear_attn_shape &s, int num_seqs, int total_rows, uint8_t *base, GdnArgs *a) {
    const size_t chunks = (size_t)max_chunks(num_seqs, total_rows);
    size_t at = 0;
    auto take = [&](size_t n) {
        uint8_t *p = base + at;
        at += (n + 255) & ~(size_t)255;
        return p;
    };
    uint8_t *kq = take(chunks * s.key_heads * 2 * kTileX), *tp = take(chunks * s.value_heads * kTileZP);
    uint8_t *gates = take(chunks * s.value_heads * kGates), *o = take(((size_t)total_rows + 7) / 8 * 8 * s.value_heads * kD * 4);
    if (a != nullptr) {
        a->kq = kq;
        a->tp = tp;
        a->gates = gates;
        a->o = reinterpret_cast<float *>(o);
    }
    return at;
}

}  // namespace
}  // namespace nmoe

using namespace nmoe;

extern "C" const char *nmoe_linear_attn_error(void) { return g_err; }

extern "C" size_t nmoe_linear_attn_prefill_workspace_bytes(const nmoe_linear_attn_shape *s, int num_seqs,
                                                           int total_rows) {
    if (check_shape(s) != NMOE_OK || num_seqs < 1 || total_rows < 0) return 0;
    return carve(*s, num_seqs, total_rows, nullptr, nullptr);
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
        a.z_stride % unit != 0 || !aligned_to(qkv, 16) || !aligned_to(z, 16) || !aligned_to(alpha, 16 / unit) ||
        !aligned_to(beta, 16 / unit))
        return fail(NMOE_EINVAL, "a row stride is too small, or qkv or z rows are not 16-byte aligned");
    if (!aligned_to(w->conv_w, 8) || !aligned_to(w->A_log, 4) || !aligned_to(w->norm_w, 8) || !aligned_to(w->dt_bias, 2) || !aligned_to(conv_in, 16) || !aligned_to(conv_out, 16) ||
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
    a.tries = wait_tries();
    if (workspace == nullptr || !aligned_to(workspace, 16)) return fail(NMOE_EINVAL, "workspace is NULL or not aligned");
    if (max_chunks(num_seqs, total_rows) > 2147483647ll || total_rows > 2147483647 - kC)
        return fail(NMOE_EINVAL, "too many rows or sequences");
    carve(*shape, num_seqs, total_rows, static_cast<uint8_t *>(workspace), &a);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = a.x_bf16 ? launch<true>(a, st) : launch<false>(a, st);
    return e == cudaSuccess ? NMOE_OK : fail(NMOE_ECUDA, "prefill: %s", cudaGetErrorString(e));
}
