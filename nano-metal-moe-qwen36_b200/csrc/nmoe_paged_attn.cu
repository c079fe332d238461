// nmoe_paged_attn.cu -- full attention over a paged bf16 cache: append of packed rows, and the
// decode step of one new token per sequence.
//
// Step: out = sigmoid(gate) * sum_p softmax_p(scale q . k_p) v_p over the positions of a
// sequence. The bound is HBM: every K and V row is read once (4 head_dim bytes a position and KV
// head) and used for all the query heads of its KV head, so the arithmetic, 8 head_dim flops per
// position and query head, goes to the warp tensor instructions (m16n8k16): the 16 rows of A are
// the 8 query heads' upper and lower bf16 parts, so q and p lose nothing against fp32 sums but the
// parts' own residue (2^-17), and K and V are the B operands straight from shared memory.
//
// Split: the positions of all (sequence, KV head) pairs, in tiles of 64 or 128, form one line that is cut
// into equal pieces, one per CTA (one CTA per SM), whatever the lengths are; a piece may end one
// pair and begin the next. Lengths are read on the device. Each of a CTA's four or eight warps takes 16
// positions of every tile with its own ring of copies (16 rows of K, 16 of V, by TMA) and its own
// running maximum and sum; warps join through shared memory at the end of a pair, and pieces of
// one pair join in a second launch. Beginning and ending a pair costs a piece about four tiles' time, and
// counts as that much on the line. Measured: 64 sequences of 32768 (2 KV heads of 256, bf16) 655 us, 6.5 TB/s; 64 of
// 8192 187 us, with an fp32 output, three parts, 232 us; 37 of up to 16384 (32 heads over 4 of 128, fp32) 64 us with
// the join, 55 of it here, 4.2 TB/s; one of 4096 14 us with the join. Pages that are no multiple of 16 rows are copied row
// by row, each waited for: 64 of 8192 2.2 ms.
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>

#include "nmoe_paged.cuh"
#include "nmoe_sm100.cuh"

namespace nmoe {

namespace {
thread_local char g_err[256];
}

int full_attn_fail(int status, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
    return status;
}

int check_full_attn_shape(const nmoe_full_attn_weights *w, const nmoe_full_attn_shape *s) {
    if (w == nullptr || s == nullptr) return full_attn_fail(NMOE_EINVAL, "weights or shape is NULL");
    if (s->head_dim != 128 && s->head_dim != 256)
        return full_attn_fail(NMOE_EINVAL, "head_dim %d: 128 or 256", s->head_dim);
    if (s->kv_heads < 1 || s->kv_heads > 1024 || s->q_heads < 1 || s->q_heads % s->kv_heads != 0 ||
        s->q_heads / s->kv_heads > 8)
        return full_attn_fail(NMOE_EINVAL, "q_heads %d must be 1..8 times kv_heads %d (at most 1024)", s->q_heads,
                              s->kv_heads);
    const int r = s->rotary_dims;
    if (r != 0 && (r < 16 || r > s->head_dim || (r & (r - 1)) != 0))
        return full_attn_fail(NMOE_EINVAL, "rotary_dims %d: 0 or a power of two from 16 to head_dim", r);
    if (r != 0 && !(s->rope_theta > 0.f && s->rope_theta <= 3.0e38f))
        return full_attn_fail(NMOE_EINVAL, "rope_theta must be positive and finite");
    if (!aligned_to(w->q_norm, 16) || !aligned_to(w->k_norm, 16))
        return full_attn_fail(NMOE_EINVAL, "q_norm and k_norm must be 16-byte aligned");
    if ((w->q_norm != nullptr || w->k_norm != nullptr) && !(s->norm_eps > 0.f))
        return full_attn_fail(NMOE_EINVAL, "norm_eps must be positive");
    if (s->gated != 0 && s->gated != 1) return full_attn_fail(NMOE_EINVAL, "gated %d: 0 or 1", s->gated);
    return NMOE_OK;
}

int check_paged_kv(const nmoe_paged_kv *kv, PagedDev *d) {
    if (kv == nullptr || kv->k == nullptr || kv->v == nullptr || kv->block_table == nullptr)
        return full_attn_fail(NMOE_EINVAL, "the cache or one of its pointers is NULL");
    if (kv->num_pages < 1 || kv->page_size < 1 || kv->max_pages < 1 || kv->table_stride < 0)
        return full_attn_fail(NMOE_EINVAL, "num_pages, page_size and max_pages must be positive");
    if ((long long)kv->max_pages * kv->page_size > 2147483647ll - 256)   // the end of the last tile is an int too
        return full_attn_fail(NMOE_EINVAL, "max_pages * page_size exceeds 2^31 - 257 positions");
    if (!aligned_to(kv->k, 16) || !aligned_to(kv->v, 16) || !aligned_to(kv->block_table, 4))
        return full_attn_fail(NMOE_EINVAL, "pages must be 16-byte aligned, the block table 4-byte");
    if (((kv->page_stride | kv->row_stride | kv->head_stride) & 7) != 0 || kv->page_stride < 0 ||
        kv->row_stride < 0 || kv->head_stride < 0)
        return full_attn_fail(NMOE_EINVAL, "page strides must be multiples of 8 elements, not negative");
    d->k = kv->k;
    d->v = kv->v;
    d->page_stride = kv->page_stride;
    d->row_stride = kv->row_stride;
    d->head_stride = kv->head_stride;
    d->table = kv->block_table;
    d->table_stride = kv->table_stride;
    d->num_pages = kv->num_pages;
    d->page_size = kv->page_size;
    d->max_pages = kv->max_pages;
    d->capacity = kv->max_pages * kv->page_size;
    return NMOE_OK;
}

void fill_rotary(const nmoe_full_attn_shape *s, RotaryDev *r) {
    r->half = s->rotary_dims / 2;
    for (int k = 0; k < 7; ++k) r->bit[k] = r->half > 0 ? pow((double)s->rope_theta, -(double)(1 << k) / r->half) : 1.0;
}

int check_x(const char *what, const void *p, int x_dtype, long long stride, long long width) {
    if (p == nullptr) return full_attn_fail(NMOE_EINVAL, "%s is NULL", what);
    if (x_dtype != NMOE_DTYPE_F32 && x_dtype != NMOE_DTYPE_BF16)
        return full_attn_fail(NMOE_EINVAL, "x_dtype %d: NMOE_DTYPE_F32 or NMOE_DTYPE_BF16", x_dtype);
    const int unit = x_dtype == NMOE_DTYPE_BF16 ? 8 : 4;
    if (!aligned_to(p, 16) || stride % unit != 0 || stride < width)
        return full_attn_fail(NMOE_EINVAL, "%s rows must be 16-byte aligned and at least %lld elements apart", what, width);
    return NMOE_OK;
}

void rows_a_cta(int want, int *rows, int *share_log) {
    *rows = 8, *share_log = 0;
    while (*rows > 1 && *rows > want) *rows >>= 1, ++*share_log;
}

int device_sm_count(int *sms) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return full_attn_fail(NMOE_ECUDA, "no CUDA device");
    return NMOE_OK;
}

uint32_t wait_tries() {
    const char *t = getenv("NMOE_WAIT_TRIES");
    return t != nullptr ? (uint32_t)strtoul(t, nullptr, 10) : kMaxSpins;
}

TensorMapEncode tensor_map_encode() {
    static TensorMapEncode fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return (TensorMapEncode) nullptr;
        return reinterpret_cast<TensorMapEncode>(p);
    }();
    return fn;
}

bool page_map(CUtensorMap *m, const PagedDev &c, const uint16_t *base, int d, int heads, int rows, int panels) {
    const cuuint64_t dims[5] = {64, (cuuint64_t)c.page_size, (cuuint64_t)(d / 64), (cuuint64_t)heads,
                                (cuuint64_t)c.num_pages};
    const cuuint64_t strides[4] = {(cuuint64_t)c.row_stride * 2, 128, (cuuint64_t)c.head_stride * 2,
                                   (cuuint64_t)c.page_stride * 2};
    const cuuint32_t box[5] = {64, (cuuint32_t)rows, (cuuint32_t)panels, 1, 1};
    const cuuint32_t es[5] = {1, 1, 1, 1, 1};
    const TensorMapEncode fn = tensor_map_encode();
    return fn != nullptr &&
           fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<uint16_t *>(base), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

// ---- append ------------------------------------------------------------------------------------

struct AppendArgs {
    PagedDev c;
    RotaryDev rot;
    HeadDev h;
    const int *cu_rows, *kv_lens;
    const void *k_new, *v_new;
    long long kv_stride;
    int num_seqs, total_rows, kv_heads, rows_per_cta, share_log, x_bf16;
};

constexpr int kAppendThreads = 256, kAppendRows = 8;

// A CTA takes rows_per_cta rows (1 when there are few, so that they spread over the SMs): one (cos, sin)
// table per row for all its heads, then a warp per (row, head, k or v). The operands of a warp's first units are
// asked for before the rows' sequences, positions and angles are found, which takes three dependent reads and two
// barriers: these, in CTAs that live for 8 rows, are what bounds it (the barrier is the first stall, DRAM moves at 0.39
// of the copy rate). 32768 rows of 2 KV heads of 256: 35 us, 20.6 at the copy rate; 4095 rows 14 us.
template <int D, bool kBf16>
__global__ void __launch_bounds__(kAppendThreads) k_append_paged(const __grid_constant__ AppendArgs a) {
    constexpr int E = D / 32, kAtOnce = 4;
    __shared__ __align__(16) float2 cs[kAppendRows][128];
    __shared__ long long where[kAppendRows];
    __shared__ int at[kAppendRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row0 = blockIdx.x * a.rows_per_cta;
    const int rows = min(a.rows_per_cta, a.total_rows - row0), units = 2 * a.kv_heads;   // k and v of a head
    // 8 / rows_per_cta (a power of two) warps share a row
    const int share_log = a.share_log, share = 1 << share_log, mine = warp >> share_log, first = warp & (share - 1);
    float v[kAtOnce][E], w[E];
    const long long src = (long long)(row0 + min(mine, rows - 1)) * a.kv_stride + E * lane;
    auto load = [&](int u0) {
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
            const int u = min(u0 + (x << share_log), units - 1);
            load_typed<E, kBf16>(u & 1 ? a.v_new : a.k_new, src + (u >> 1) * D, v[x]);
        }
    };
    load(first);
    load_weight<E>(a.h.k_norm, lane, w);
    const double freq = a.rot.half > 0 ? rotary_freq(a.rot, tid & (a.rot.half - 1)) : 0.0;
    if (tid < rows) {
        const int r = row0 + tid, b = find_sequence(a.cu_rows, a.num_seqs, r);
        long long to = -1, p = -1;
        if (b >= 0) {
            p = (long long)a.kv_lens[b] - a.cu_rows[b + 1] + r;
            if (p >= 0 && p < a.c.capacity) to = paged_row(a.c, b, (int)p);
        }
        where[tid] = to;
        at[tid] = to >= 0 ? (int)p : 0;
    }
    __syncthreads();
    if (a.rot.half > 0) {   // half is a power of two that divides the threads: a thread keeps its t
        const int t = tid & (a.rot.half - 1);
        for (int r = tid / a.rot.half; r < rows; r += kAppendThreads / a.rot.half) cs[r][t] = rotary_cs(freq, at[r]);
    }
    __syncthreads();
    if (mine >= rows || where[mine] < 0) return;
    const long long dst = where[mine] + E * lane;
    for (int u0 = first; u0 < units; u0 += kAtOnce << share_log) {
        if (u0 != first) load(u0);
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
            const int u = u0 + (x << share_log);
            if (u >= units) break;
            if (!(u & 1)) prepare_head<E>(v[x], w, a.h.k_norm != nullptr, a.h.eps, cs[mine], a.rot.half, lane);
            store_bf16<E>((u & 1 ? a.c.v : a.c.k) + dst + (u >> 1) * a.c.head_stride, v[x]);
        }
    }
}

// ---- step ----------------------------------------------------------------------------------------

constexpr int kJoinThreads = 512;   // sets of D / 4 threads, each taking every n-th piece
constexpr int kMaxCtas = 512;    // pieces of the line of tiles (workspace bound)
constexpr int kGroupMax = 8;
constexpr int kPairCost = 4;     // tiles

struct StepArgs {
    CUtensorMap k_map, v_map;   // pages in boxes of 16 rows and all columns, where boxed
    PagedDev c;
    RotaryDev rot;
    HeadDev h;
    const int *kv_lens;
    const void *q, *k_new, *v_new;
    long long q_stride, kv_stride;
    float *part;   // [pairs + CTAs][group][D + 4]: weighted values, maximum, sum
    void *out;
    float scale;   // softmax scale times log2(e)
    int batch, kv_heads, group, gated, x_bf16, out_bf16, ctas, boxed;
    uint32_t tries;   // of a wait, before it gives up
};

// Warps a CTA: what a scheduler needs to hide a step's chain of products behind another warp's, as far as
// the registers allow. head_dim 128: 8 (a ragged fp32 batch 95 us with 4); 256: 4, whose
// sums take 128 registers a thread (64 sequences of 32768: 99% of the copy rate).
template <int D>
struct StepCfg {
    static constexpr int kWarps = D == 256 ? 4 : 8, kThreads = 32 * kWarps;
    static constexpr int kTile = 16 * kWarps;         // positions of a tile: 16 per warp
    static constexpr int kHalfB = 16 * D * 2;         // 16 rows of K (or V): panels of [16 rows][64 columns], swizzled
    static constexpr int kStageB = 2 * kHalfB;
    static constexpr int kStages = 3;
    static constexpr int kRingB = kWarps * kStages * kStageB;
    static constexpr int kQ = kRingB;                 // query parts: rows of kRowB
    static constexpr int kRowB = D * 2 + 16;          // 16 bytes of padding: 8 rows of an ldmatrix in 8 bank groups
    static constexpr int q_bytes(int parts) { return (parts == 3 ? 32 : 16) * kRowB; }
    static constexpr int bytes(int parts) { return kRingB + q_bytes(parts) + 1024; }   // + alignment
};

// byte offset of 16-byte piece x of row r (of 16) of a half stage
__device__ __forceinline__ uint32_t at_panel(int r, int x) {
    return (uint32_t)(x >> 3) * 2048u + (uint32_t)r * 128u + (uint32_t)(((x & 7) ^ (r & 7)) << 4);
}

template <int D>
__device__ __forceinline__ int seq_tiles(int len, int capacity) {
    constexpr int kTile = StepCfg<D>::kTile;
    return len < 1 || len > capacity ? 0 : (len + kTile - 1) / kTile;
}
// What a (sequence, KV head) pair counts on the line: its tiles and what beginning and ending it costs
// (queries, first copies, the join of the warps), in tiles.
__device__ __forceinline__ long long pair_weight(int tiles) { return tiles > 0 ? tiles + kPairCost : 0; }

// All threads of a CTA: weight of the sequences before this thread's stripe of them, and of all.
struct Plan {
    long long before, total;   // per KV head
    int first, last;           // this thread's stripe of sequences
};
template <int D, int kThreads>
__device__ __forceinline__ Plan plan_tiles(const int *lens, int batch, int capacity, long long *sm) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (batch + kThreads - 1) / kThreads;
    Plan p;
    p.first = min(batch, tid * per);
    p.last = min(batch, p.first + per);
    long long own = 0;
    for (int b = p.first; b < p.last; ++b) own += pair_weight(seq_tiles<D>(lens[b], capacity));
    long long inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) sm[warp] = inc;
    __syncthreads();
    long long pre = 0, tot = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) pre += sm[w];
        tot += sm[w];
    }
    p.before = pre + inc - own;
    p.total = tot;
    return p;
}

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
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16 page rows of one head, all columns
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap *map, int row, int head, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
        "%6}], [%7];" ::"r"(dst),
        "l"(map), "r"(0), "r"(row), "r"(0), "r"(head), "r"(page), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// out[b][head][d .. d + 3] = weighted values / sum, times the gate; nothing seen: zeros.
template <int D>
__device__ __forceinline__ void write_out(const StepArgs &a, int b, int head, int d, float4 A, float L) {
    float v[4] = {A.x, A.y, A.z, A.w};
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    float g[4] = {1.f, 1.f, 1.f, 1.f};
    if (a.gated) {
        load_elems<4>(a.q, (long long)b * a.q_stride + (long long)head * 2 * D + D + d, a.x_bf16, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = sigmoidf_(g[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = L == 0.f ? 0.f : v[i] * inv * g[i];
    const long long at = ((long long)b * a.kv_heads * a.group + head) * D + d;
    if (a.out_bf16)
        store_bf16<4>(static_cast<uint16_t *>(a.out) + at, v);
    else
        *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
}

// PARTS: bf16 parts of q and p: 2 (residue 2^-17) for a bf16 output, 3 (fp32) for an fp32 one.
template <int D, int PARTS>
__global__ void __launch_bounds__(StepCfg<D>::kThreads, 1) k_step_paged(const __grid_constant__ StepArgs a) {
    using Cfg = StepCfg<D>;
    constexpr int E = D / 32, kRowB = Cfg::kRowB, kStages = Cfg::kStages;
    constexpr int kWarps = Cfg::kWarps, kThreads = Cfg::kThreads, kTile = Cfg::kTile;
    extern __shared__ uint8_t raw_smem[];
    __shared__ uint64_t bars[kWarps][kStages];
    __shared__ uint32_t live[kWarps][kStages];   // bit i: position i of the stage takes part
    __shared__ __align__(16) float2 cs[128];
    __shared__ float sm_m[kWarps][kGroupMax], sm_l[kWarps][kGroupMax];
    __shared__ long long sm_scan[kWarps];
    __shared__ int sm_seq;
    __shared__ long long sm_off;

    uint8_t *smem = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);   // the swizzle goes by the address
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(&bars[warp][s], 1);
        mbar_fence_init();
    }
    const double freq = tid < a.rot.half ? rotary_freq(a.rot, tid) : 0.0;
    const Plan plan = plan_tiles<D, kThreads>(a.kv_lens, a.batch, a.c.capacity, sm_scan);
    const long long total = plan.total * a.kv_heads;
    const long long pieces = min((long long)a.ctas, total);   // no piece is empty
    if (blockIdx.x >= pieces) return;
    long long cur = total * blockIdx.x / pieces;
    const long long end = total * (blockIdx.x + 1) / pieces;
    {
        long long before = plan.before;
        for (int b = plan.first; b < plan.last; ++b) {
            const long long n = pair_weight(seq_tiles<D>(a.kv_lens[b], a.c.capacity));
            if (cur >= before * a.kv_heads && cur < (before + n) * a.kv_heads) {
                sm_seq = b;
                sm_off = cur - before * a.kv_heads;
            }
            before += n;
        }
    }
    __syncthreads();
    int b = sm_seq, len = a.kv_lens[b], nt = seq_tiles<D>(len, a.c.capacity);
    int kvh = (int)(sm_off / (nt + kPairCost));
    int at = (int)(sm_off - (long long)kvh * (nt + kPairCost));   // where the piece begins in its pair

    const uint32_t ring = smem_u32(smem) + warp * kStages * Cfg::kStageB;
    uint8_t *ring_p = smem + warp * kStages * Cfg::kStageB;
    const uint32_t sq = smem_u32(smem) + Cfg::kQ;
    uint32_t it = 0;   // stages this warp has filled
    uint32_t used = 0;
    bool lost = false;   // a wait has run out: this warp copies and waits no more, and its sums are NaN

    while (true) {
        // tiles t0 .. t1 - 1 of this pair; none when the piece holds no more than the pair's cost
        const int to = (int)min((long long)nt + kPairCost, at + (end - cur));
        const int t0 = max(0, at - kPairCost), t1 = max(0, to - kPairCost);
        const int steps = t1 - t0;
        const bool whole = steps == nt;
        const int fresh = a.k_new != nullptr ? len - 1 : -1;   // position that comes from k_new / v_new

        // ---- copies of this warp's 16 positions of tile t0 + i
        int page_next = -1;
        auto page_of = [&](int i) {   // boxed: of all 16 positions; else of position lane % 16
            const int p = (t0 + i) * kTile + 16 * warp + (a.boxed ? 0 : lane & 15);
            return i < steps && p < len ? a.c.table[(long long)b * a.c.table_stride + (unsigned)p / (unsigned)a.c.page_size]
                                        : -1;
        };
        auto issue = [&](int i) {
            const int s = it % kStages;
            const int page = page_next;
            page_next = page_of(i + 1);
            const int base = (t0 + i) * kTile + 16 * warp;
            const bool ok = page >= 0 && page < a.c.num_pages;   // page is -1 past the end
            uint8_t *stage = ring_p + s * Cfg::kStageB;
            uint32_t okm;
            if (a.boxed) {
                okm = ok ? (len - base >= 16 ? 0xffffu : (1u << (len - base)) - 1u) : 0u;
            } else {
                okm = __ballot_sync(0xffffffffu, ok) & 0xffffu;
            }
            if (lane == 0) {
                live[warp][s] = okm;
                mbar_arrive_expect_tx(&bars[warp][s], a.boxed && ok ? Cfg::kStageB : 0);
            }
            fence_async_shared();   // this warp's reads and writes of the stage, before the copies
            __syncwarp();
            if (a.boxed && ok) {
                if (lane < 2)
                    copy_box(ring + s * Cfg::kStageB + lane * Cfg::kHalfB, lane ? &a.v_map : &a.k_map,
                             (int)((unsigned)base % (unsigned)a.c.page_size), kvh, page, smem_u32(&bars[warp][s]));
            } else if (!a.boxed) {   // pages that no box fits: row by row, D / 8 pieces each
                for (int r = 0; r < 16; ++r) {
                    const int pg = __shfl_sync(0xffffffffu, page, r);
                    if (!(okm >> r & 1u)) continue;
                    const long long off = (long long)pg * a.c.page_stride +
                                          (long long)((unsigned)(base + r) % (unsigned)a.c.page_size) * a.c.row_stride +
                                          (long long)kvh * a.c.head_stride;
                    for (int x = lane; x < D / 4; x += 32) {
                        const int v = x >= D / 8, piece = x - v * (D / 8);
                        *reinterpret_cast<uint4 *>(stage + v * Cfg::kHalfB + at_panel(r, piece)) =
                            *reinterpret_cast<const uint4 *>((v ? a.c.v : a.c.k) + off + 8 * piece);
                    }
                }
            }
            ++it;
        };
        if (steps > 0) {
        page_next = page_of(0);
        int issued = 0;
        for (; issued < kStages && issued < steps && !lost; ++issued) issue(issued);

        // ---- the queries of the group, prepared, scaled and split into bf16 parts
        if (tid < a.rot.half) cs[tid] = rotary_cs(freq, len - 1);
        for (int i = tid; i < Cfg::q_bytes(PARTS) / 16; i += kThreads)
            *reinterpret_cast<uint4 *>(smem + Cfg::kQ + 16 * i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (int g = warp; g < a.group; g += kWarps) {
            float v[E];
            load_elems<E>(a.q, (long long)b * a.q_stride + (long long)(kvh * a.group + g) * (a.gated ? 2 * D : D) + E * lane,
                          a.x_bf16, v);
            float w[E];
            load_weight<E>(a.h.q_norm, lane, w);
            prepare_head<E>(v, w, a.h.q_norm != nullptr, a.h.eps, cs, a.rot.half, lane);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] *= a.scale;
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                uint16_t *dst = reinterpret_cast<uint16_t *>(smem + Cfg::kQ + (8 * part + g) * kRowB) + E * lane;
                store_bf16<E>(dst, v);
#pragma unroll
                for (int i = 0; i < E; ++i) v[i] -= bf16_round(v[i]);
            }
        }
        __syncthreads();
        uint32_t qf[D / 16][4];
        const uint32_t qa = sq + (lane & 15) * kRowB + (lane >> 4) * 16;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) ldsm4(qa + 32 * kk, qf[kk]);

        float m = -INFINITY, l = 0.f;   // of head lane / 4, l over this thread's positions
        float acc[D / 8][4];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;

        for (int i = 0; i < steps && !lost; ++i) {
            const int s = used % kStages;
            lost = !__all_sync(0xffffffffu, mbar_wait_spin(&bars[warp][s], (used / kStages) & 1, a.tries));
            if (lost) break;
            const int base = (t0 + i) * kTile + 16 * warp;
            uint32_t lv = live[warp][s];
            const uint32_t ks = ring + s * Cfg::kStageB, vs = ks + Cfg::kHalfB;
            uint8_t *stage = ring_p + s * Cfg::kStageB;
            // a V row that takes no part is zero: its probability is zero, and 0 * NaN is NaN
            if (lv != 0xffffu) {
                for (uint32_t z = ~lv & 0xffffu; z != 0; z &= z - 1)
                    if (lane < D / 8)
                        *reinterpret_cast<uint4 *>(stage + Cfg::kHalfB + at_panel(__ffs(z) - 1, lane)) = make_uint4(0, 0, 0, 0);
                __syncwarp();
            }
            if (fresh >= base && fresh < base + 16 && (lv >> (fresh - base) & 1u)) {
                // the new token: its key and value into the cache and into this stage
                float v[E];
                const long long src = (long long)b * a.kv_stride + (long long)kvh * D + E * lane;
                const long long dst = paged_row(a.c, b, fresh) + (long long)kvh * a.c.head_stride + E * lane;
                uint8_t *row = stage + at_panel(fresh - base, E * lane / 8) + (E * lane % 8) * 2;
                load_elems<E>(a.k_new, src, a.x_bf16, v);
                float w[E];
                load_weight<E>(a.h.k_norm, lane, w);
                prepare_head<E>(v, w, a.h.k_norm != nullptr, a.h.eps, cs, a.rot.half, lane);
                store_bf16<E>(a.c.k + dst, v);
                store_bf16<E>(reinterpret_cast<uint16_t *>(row), v);
                load_elems<E>(a.v_new, src, a.x_bf16, v);
                store_bf16<E>(a.c.v + dst, v);
                store_bf16<E>(reinterpret_cast<uint16_t *>(row + Cfg::kHalfB), v);
                __syncwarp();
            }
            float sc[2][2][4];   // [kk parity][8 positions][fragment]
#pragma unroll
            for (int x = 0; x < 16; ++x) (&sc[0][0][0])[x] = 0.f;
            const int kr = (lane >> 4) * 8 + (lane & 7), kx = (lane >> 3) & 1;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                uint32_t kf[4];
                ldsm4(ks + at_panel(kr, 2 * kk + kx), kf);
                mma_bf16(sc[kk & 1][0], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], kf[0], kf[1]);
                mma_bf16(sc[kk & 1][1], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], kf[2], kf[3]);
                if constexpr (PARTS == 3) {
                    uint32_t q3[4];
                    ldsm4(qa + 16 * kRowB + 32 * kk, q3);
                    mma_bf16(sc[kk & 1][0], q3[0], q3[1], q3[2], q3[3], kf[0], kf[1]);
                    mma_bf16(sc[kk & 1][1], q3[0], q3[1], q3[2], q3[3], kf[2], kf[3]);
                }
            }
            float x[4];   // positions base + 8 j + 2 (lane % 4) + e, j = index / 2, e = index % 2
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float v = (sc[0][j][e] + sc[1][j][e]) + (sc[0][j][e + 2] + sc[1][j][e + 2]);
                    x[2 * j + e] = (lv >> (8 * j + 2 * (lane & 3) + e)) & 1u ? v : -INFINITY;
                    mx = fmaxf(mx, x[2 * j + e]);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mn = fmaxf(m, mx);
            const float ms = mn == -INFINITY ? 0.f : mn;
            if (__any_sync(0xffffffffu, mn != m)) {
                const float c = ex2(m - ms);
                l *= c;
#pragma unroll
                for (int n = 0; n < D / 8; ++n) acc[n][0] *= c, acc[n][1] *= c, acc[n][2] *= c, acc[n][3] *= c;
                m = mn;
            }
            float p[4], r1[4];
            uint32_t pf[4], pf3[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = ex2(x[e] - ms);
                l += p[e];
            }
            pf[0] = pack2_bf16(p[0], p[1]);
            pf[2] = pack2_bf16(p[2], p[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) r1[e] = p[e] - bf16_round(p[e]);
            pf[1] = pack2_bf16(r1[0], r1[1]);
            pf[3] = pack2_bf16(r1[2], r1[3]);
            if constexpr (PARTS == 3) {
                pf3[0] = pack2_bf16(r1[0] - bf16_round(r1[0]), r1[1] - bf16_round(r1[1]));
                pf3[2] = pack2_bf16(r1[2] - bf16_round(r1[2]), r1[3] - bf16_round(r1[3]));
                pf3[1] = pf3[3] = 0u;
            }
            const int vr = lane & 15, vx = lane >> 4;
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                uint32_t vf[4];
                ldsm4t(vs + at_panel(vr, 2 * n + vx), vf);
                mma_bf16(acc[2 * n], pf[0], pf[1], pf[2], pf[3], vf[0], vf[1]);
                mma_bf16(acc[2 * n + 1], pf[0], pf[1], pf[2], pf[3], vf[2], vf[3]);
                if constexpr (PARTS == 3) {
                    mma_bf16(acc[2 * n], pf3[0], pf3[1], pf3[2], pf3[3], vf[0], vf[1]);
                    mma_bf16(acc[2 * n + 1], pf3[0], pf3[1], pf3[2], pf3[3], vf[2], vf[3]);
                }
            }
            ++used;
            __syncwarp();
            if (issued < steps) issue(issued++);
        }
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (lost) l = NAN;   // a copy that never landed must not pass for an answer

        // ---- join the warps through the (drained) ring
        __syncthreads();
        float *so = reinterpret_cast<float *>(smem) + (warp * kGroupMax + (lane >> 2)) * D + 2 * (lane & 3);
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2 *>(so + 8 * n) = make_float2(acc[n][0] + acc[n][2], acc[n][1] + acc[n][3]);
        if ((lane & 3) == 0) {
            sm_m[warp][lane >> 2] = m;
            sm_l[warp][lane >> 2] = l;
        }
        __syncthreads();
        const long long pair = (long long)b * a.kv_heads + kvh;
        for (int u = tid; u < a.group * (D / 4); u += kThreads) {
            const int g = u / (D / 4), d = 4 * (u - g * (D / 4));
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w][g]);
            const float ms = M == -INFINITY ? 0.f : M;
            float L = 0.f;
            float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float e = ex2(sm_m[w][g] - ms);
                const float4 o = *reinterpret_cast<const float4 *>(reinterpret_cast<float *>(smem) +
                                                                   (w * kGroupMax + g) * D + d);
                L = fmaf(sm_l[w][g], e, L);
                A.x = fmaf(o.x, e, A.x), A.y = fmaf(o.y, e, A.y), A.z = fmaf(o.z, e, A.z), A.w = fmaf(o.w, e, A.w);
            }
            if (whole) {
                write_out<D>(a, b, kvh * a.group + g, d, A, L);
            } else {
                float *pb = a.part + ((pair + blockIdx.x) * a.group + g) * (D + 4);
                *reinterpret_cast<float4 *>(pb + d) = A;
                if (d == 0) *reinterpret_cast<float2 *>(pb + D) = make_float2(M, L);
            }
        }
        }
        cur += to - at;
        if (cur >= end) break;
        __syncthreads();
        at = 0;   // the next pair that has tiles
        if (++kvh == a.kv_heads) {
            kvh = 0;
            do {
                ++b;
                len = a.kv_lens[b];
                nt = seq_tiles<D>(len, a.c.capacity);
            } while (nt == 0 && b < a.batch - 1);   // tiles are left (cur < end): a later sequence has some
            if (nt == 0) break;
        }
    }
    if (lost)   // copies in flight land before the shared memory goes: of either parity, as one is in flight; bounded too
        for (int s = 0; s < 2 * kStages; ++s)
            for (int n = 0; n < 1000 && !mbar_try_wait_sleep(&bars[warp][s >> 1], s & 1, 1000); ++n) {}
}

// The pieces of one (pair, query head), or zeros for a sequence without positions. The plan is
// recomputed while the step kernel runs (it reads only the lengths). 512 threads, since one pair may have all 148
// pieces and their reads are what it waits for.
template <int D>
__global__ void __launch_bounds__(kJoinThreads) k_step_join(const __grid_constant__ StepArgs a) {
    constexpr int kLanes = D / 4, kSets = kJoinThreads / kLanes;
    __shared__ long long sm_scan[kJoinThreads / 32];
    __shared__ long long sm_before;
    __shared__ float sm_m[kMaxCtas], sm_l[kMaxCtas];
    __shared__ float4 sm_a[kJoinThreads];
    __shared__ float sm_s[kSets];
    const int tid = threadIdx.x;
    const int pair = blockIdx.x, b = pair / a.kv_heads, kvh = pair - b * a.kv_heads, g = blockIdx.y;
    const Plan plan = plan_tiles<D, kJoinThreads>(a.kv_lens, a.batch, a.c.capacity, sm_scan);
    if (b >= plan.first && b < plan.last) {
        long long before = plan.before;
        for (int x = plan.first; x < b; ++x) before += pair_weight(seq_tiles<D>(a.kv_lens[x], a.c.capacity));
        sm_before = before;
    }
    __syncthreads();
    const int nt = seq_tiles<D>(a.kv_lens[b], a.c.capacity);
    // every CTA waits for the step kernel, so that this launch never ends before it
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int d = 4 * (tid % kLanes), set = tid / kLanes;
    if (nt == 0) {
        if (set == 0) write_out<D>(a, b, kvh * a.group + g, d, make_float4(0.f, 0.f, 0.f, 0.f), 0.f);
        return;
    }
    const long long total = plan.total * a.kv_heads;
    // where the pair's first and last tile are on the line
    const long long first = sm_before * a.kv_heads + (long long)kvh * (nt + kPairCost) + kPairCost, last = first + nt - 1;
    // the CTA that takes tile t: the largest c with total * c / pieces <= t
    const long long pieces = min((long long)a.ctas, total);
    const int c0 = (int)(((first + 1) * pieces - 1) / total), c1 = (int)(((last + 1) * pieces - 1) / total);
    if (c0 == c1) return;   // one CTA had the whole pair and wrote the output
    const int n = c1 - c0 + 1;
    const float *pb = a.part + (((long long)pair + c0) * a.group + g) * (D + 4);
    const long long step = (long long)a.group * (D + 4);
    for (int i = tid; i < n; i += kJoinThreads) {
        const float2 ml = *reinterpret_cast<const float2 *>(pb + i * step + D);
        sm_m[i] = ml.x;
        sm_l[i] = ml.y;
    }
    __syncthreads();
    float M = -INFINITY;
    for (int i = tid & 31; i < n; i += 32) M = fmaxf(M, sm_m[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float ms = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int i = set; i < n; i += kSets) {
        const float e = ex2(sm_m[i] - ms);
        const float4 o = *reinterpret_cast<const float4 *>(pb + i * step + d);
        L = fmaf(sm_l[i], e, L);
        A.x = fmaf(o.x, e, A.x), A.y = fmaf(o.y, e, A.y), A.z = fmaf(o.z, e, A.z), A.w = fmaf(o.w, e, A.w);
    }
    sm_a[tid] = A;
    if (d == 0) sm_s[set] = L;
    __syncthreads();
    if (set != 0) return;
#pragma unroll
    for (int x = 1; x < kSets; ++x) {
        const float4 o = sm_a[x * kLanes + tid];
        A.x += o.x, A.y += o.y, A.z += o.z, A.w += o.w;
    }
    L = 0.f;
#pragma unroll
    for (int x = 0; x < kSets; ++x) L += sm_s[x];
    write_out<D>(a, b, kvh * a.group + g, d, A, L);
}

template <int D, int PARTS>
int launch_step(const StepArgs &a, cudaStream_t st) {
    constexpr int smem = StepCfg<D>::bytes(PARTS);
    static SmemOnce once;
    cudaError_t e = once.set(k_step_paged<D, PARTS>, smem);
    if (e == cudaSuccess) {
        k_step_paged<D, PARTS><<<a.ctas, StepCfg<D>::kThreads, smem, st>>>(a);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(a.batch * a.kv_heads, a.group);
        cfg.blockDim = dim3(kJoinThreads);
        cfg.stream = st;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, k_step_join<D>, a);
    }
    return e == cudaSuccess ? NMOE_OK : full_attn_fail(NMOE_ECUDA, "step: %s", cudaGetErrorString(e));
}

}  // namespace
}  // namespace nmoe

using namespace nmoe;

extern "C" const char *nmoe_full_attn_error(void) { return g_err; }

extern "C" int nmoe_full_attn_append_paged(const nmoe_full_attn_weights *w, const nmoe_full_attn_shape *shape,
                                           const nmoe_paged_kv *kv, int num_seqs, int total_rows, const int32_t *cu_rows,
                                           const int32_t *kv_lens, const void *k_new, const void *v_new, int x_dtype,
                                           int64_t kv_stride, void *stream) {
    AppendArgs a;
    int rc = check_full_attn_shape(w, shape);
    if (rc == NMOE_OK) rc = check_paged_kv(kv, &a.c);
    if (rc != NMOE_OK) return rc;
    if (num_seqs < 0 || total_rows < 0) return full_attn_fail(NMOE_EINVAL, "num_seqs or total_rows is negative");
    if (num_seqs == 0 || total_rows == 0) return NMOE_OK;
    if (cu_rows == nullptr || kv_lens == nullptr || !aligned_to(cu_rows, 4) || !aligned_to(kv_lens, 4))
        return full_attn_fail(NMOE_EINVAL, "cu_rows or kv_lens is NULL or not aligned");
    const long long width = (long long)shape->kv_heads * shape->head_dim;
    a.kv_stride = kv_stride == 0 ? width : kv_stride;
    rc = check_x("k_new", k_new, x_dtype, a.kv_stride, width);
    if (rc == NMOE_OK) rc = check_x("v_new", v_new, x_dtype, a.kv_stride, width);
    int sms = 0;
    if (rc == NMOE_OK) rc = device_sm_count(&sms);
    if (rc != NMOE_OK) return rc;
    fill_rotary(shape, &a.rot);
    a.h = {nullptr, w->k_norm, shape->norm_eps};
    a.cu_rows = cu_rows;
    a.kv_lens = kv_lens;
    a.k_new = k_new;
    a.v_new = v_new;
    a.num_seqs = num_seqs;
    a.total_rows = total_rows;
    a.kv_heads = shape->kv_heads;
    a.x_bf16 = x_dtype == NMOE_DTYPE_BF16;
    rows_a_cta(total_rows / (8 * sms), &a.rows_per_cta, &a.share_log);
    const int grid = (total_rows + a.rows_per_cta - 1) / a.rows_per_cta;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (shape->head_dim == 256)
        (a.x_bf16 ? k_append_paged<256, true> : k_append_paged<256, false>)<<<grid, kAppendThreads, 0, st>>>(a);
    else
        (a.x_bf16 ? k_append_paged<128, true> : k_append_paged<128, false>)<<<grid, kAppendThreads, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? NMOE_OK : full_attn_fail(NMOE_ECUDA, "append: %s", cudaGetErrorString(e));
}

extern "C" size_t nmoe_full_attn_step_paged_workspace_bytes(const nmoe_full_attn_shape *s, int batch) {
    const nmoe_full_attn_weights none = {nullptr, nullptr};
    if (batch < 1 || check_full_attn_shape(&none, s) != NMOE_OK) return 0;
    const size_t slots = (size_t)batch * s->kv_heads + kMaxCtas;
    return slots * (s->q_heads / s->kv_heads) * (s->head_dim + 4) * sizeof(float);
}

extern "C" int nmoe_full_attn_step_paged(const nmoe_full_attn_weights *w, const nmoe_full_attn_shape *shape,
                                         const nmoe_paged_kv *kv, int batch, const int32_t *kv_lens, const void *q,
                                         int64_t q_stride, const void *k_new, const void *v_new, int64_t kv_stride,
                                         int x_dtype, float scale, void *out, int out_dtype, void *workspace,
                                         void *stream) {
    StepArgs a;
    int rc = check_full_attn_shape(w, shape);
    if (rc == NMOE_OK) rc = check_paged_kv(kv, &a.c);
    if (rc != NMOE_OK) return rc;
    if (batch < 0) return full_attn_fail(NMOE_EINVAL, "batch is negative");
    if (batch == 0) return NMOE_OK;
    if ((long long)batch * shape->kv_heads > 2147483647ll - kMaxCtas)
        return full_attn_fail(NMOE_EINVAL, "batch %d is too large", batch);
    if (kv_lens == nullptr || !aligned_to(kv_lens, 4)) return full_attn_fail(NMOE_EINVAL, "kv_lens is NULL or not aligned");
    const long long qw = (long long)shape->q_heads * shape->head_dim * (shape->gated ? 2 : 1);
    const long long width = (long long)shape->kv_heads * shape->head_dim;
    a.q_stride = q_stride == 0 ? qw : q_stride;
    a.kv_stride = kv_stride == 0 ? width : kv_stride;
    rc = check_x("q", q, x_dtype, a.q_stride, qw);
    if (rc == NMOE_OK && (k_new == nullptr) != (v_new == nullptr))
        rc = full_attn_fail(NMOE_EINVAL, "k_new and v_new go together");
    if (rc == NMOE_OK && k_new != nullptr) {
        rc = check_x("k_new", k_new, x_dtype, a.kv_stride, width);
        if (rc == NMOE_OK) rc = check_x("v_new", v_new, x_dtype, a.kv_stride, width);
    }
    if (rc != NMOE_OK) return rc;
    if (out_dtype != NMOE_DTYPE_F32 && out_dtype != NMOE_DTYPE_BF16)
        return full_attn_fail(NMOE_EINVAL, "out_dtype %d: NMOE_DTYPE_F32 or NMOE_DTYPE_BF16", out_dtype);
    if (out == nullptr || workspace == nullptr || !aligned_to(out, 16) || !aligned_to(workspace, 16))
        return full_attn_fail(NMOE_EINVAL, "out or workspace is NULL or not 16-byte aligned");
    if (!(scale >= 0.f && scale <= 3.0e38f)) return full_attn_fail(NMOE_EINVAL, "scale must be finite and not negative");
    int sms = 0;
    if ((rc = device_sm_count(&sms)) != NMOE_OK) return rc;
    fill_rotary(shape, &a.rot);
    a.h = {w->q_norm, w->k_norm, shape->norm_eps};
    a.kv_lens = kv_lens;
    a.q = q;
    a.k_new = k_new;
    a.v_new = v_new;
    a.part = static_cast<float *>(workspace);
    a.out = out;
    a.scale = (scale == 0.f ? 1.0f / sqrtf((float)shape->head_dim) : scale) * 1.4426950408889634f;
    a.tries = wait_tries();
    a.batch = batch;
    a.kv_heads = shape->kv_heads;
    a.group = shape->q_heads / shape->kv_heads;
    a.gated = shape->gated;
    a.x_bf16 = x_dtype == NMOE_DTYPE_BF16;
    a.out_bf16 = out_dtype == NMOE_DTYPE_BF16;
    // boxes of 16 rows and all columns: 16 positions lie in one page
    const int d = shape->head_dim;
    a.boxed = a.c.page_size % 16 == 0 && page_map(&a.k_map, a.c, a.c.k, d, a.kv_heads, 16, d / 64) &&
              page_map(&a.v_map, a.c, a.c.v, d, a.kv_heads, 16, d / 64);
    const long long most = (long long)batch * shape->kv_heads * ((a.c.capacity + 63) / 64);
    a.ctas = (int)(most < sms ? most : sms);
    if (a.ctas > kMaxCtas) a.ctas = kMaxCtas;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (shape->head_dim == 256) return a.out_bf16 ? launch_step<256, 2>(a, st) : launch_step<256, 3>(a, st);
    return a.out_bf16 ? launch_step<128, 2>(a, st) : launch_step<128, 3>(a, st);
}
