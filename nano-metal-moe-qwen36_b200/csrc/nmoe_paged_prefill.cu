// nmoe_paged_prefill.cu -- causal attention of packed prompts over a paged bf16 cache.
//
// out_i = sigmoid(gate_i) * sum_{p <= pos_i} softmax_p(scale q_i . k_p) v_p, 4 head_dim flops per
// visible pair of a query row and a position: the bound is the tensor cores, once a prompt has a
// few hundred rows.
//
// Tile: a pair of CTAs (cta_group::2, M = 256) takes 256 query rows of one KV head, each CTA 128 of
// them (a row is a token's query head; the heads of a group share the rows' keys and values), and
// walks over the positions in tiles of 128. S = Q K^T (Q in shared memory) and O += P V (P in tensor
// memory) are tcgen05 MMAs issued by one thread of the first CTA; each CTA holds half of every K
// tile (64 positions) and half of every V tile (head_dim / 2 columns), so a tile crosses from L2
// once per 256 rows. At head_dim 256, O takes half of the tensor memory and two S tiles the other
// half; a CTA of its own with M = 128 would have to read 62 bytes a cycle from L2 and 160 a cycle
// from shared memory to keep the tensor cores busy, the pair 31 and 95.
//
// Softmax: two threads per query row (warps 0-7, 64 columns each) read its 128 scores from tensor
// memory, keep the running maximum and sum (Milakov and Gimelshein 2018) in fp32, and write P back as bf16 over the scores. Queries and P are
// rounded to bf16, the type of the pages, since an MMA's operands have one type: the output is off by 0.0025 of its
// norm, of which its own rounding is 0.0017; two bf16 parts of either would double the products. O is rescaled only
// when a row's maximum has grown by more than 2^8 since the last time: O and the sum carry the same
// reference, so the result does not depend on which one it is. While S of tile j is in the softmax,
// the tensor cores run S of tile j + 1 and P V of tile j - 1. Measured: a prompt of 16384 rows, 16 query and 2 KV heads
// of 256: 1.77 ms held for seconds, under the power limit, 1.24 PFLOP/s (of the visible pairs; the tiles on the diagonal
// are computed whole); one call alone 1.54 ms, 1.42 PFLOP/s. Pages that no box fits (below): 4096 rows 870 us with 7
// rows a page, 198 us with 16.
//
// Pages: a warp of each CTA copies boxes of page rows by TMA (the rows of a box lie in one page, as
// a tile's 64 positions may lie in many). Positions behind a sequence's end, and pages that are
// none, are masked in the scores, and their V rows are set to zero in shared memory before the MMA
// reads them: 0 * NaN is NaN. Page sizes that are no multiple of 16 rows are copied by the warp
// itself.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "nmoe_gemm.cuh"
#include "nmoe_paged.cuh"

namespace cg = cooperative_groups;

namespace nmoe {
namespace {

struct PrefillArgs {
    CUtensorMap k_map, v_map;   // pages as 5D tensors (page_map), boxes of box_rows rows and one or more panels of 64 columns
    CUtensorMap q_map;          // prepared queries, boxes of 64 columns x 128 rows
    uint16_t *q_ready;
    int prep_rows, share_log;
    PagedDev c;
    RotaryDev rot;
    HeadDev h;
    const int *cu_rows, *kv_lens;
    const void *q;
    long long q_stride;
    uint16_t *out;
    float scale;   // softmax scale times log2(e)
    int num_seqs, total_rows, kv_heads, group, gated, x_bf16;
    int box_rows, box_shift;   // rows of a TMA box: 16, 32 or 64, or 0: no TMA
    uint32_t tries, nap;       // of a wait before it gives up, and the ns that each may take
};

constexpr int kThreads = 352;   // warps 0-7 softmax, 8 copies Q and K, 9 MMA, 10 copies V
constexpr int kRows = 128;      // query rows of a CTA
constexpr int kTile = 128;      // positions of a tile
constexpr int kInfo = 8;        // ring of tile masks

struct Shared {
    uint64_t full[10], empty[10], landed, s_full[2], p_ready[2][2], o_done, done, q_ready;
    uint32_t info[kInfo][5];          // valid positions of a tile, then whether all are
    int scan[kThreads / 32], unit_off, unit_seq;
    float row_max[2][2][kRows];       // of a row's two halves, by the parity of the tile
    uint32_t tmem;
    int stop;                         // a bounded wait has run out
};

template <int D>
struct Cfg {
    static constexpr int kQB = kRows * D * 2;
    static constexpr int kStageB = 64 * D * 2;              // half a K or V tile
    // A step is what goes through the softmax at a time: at head_dim 256 a tile, at 128 half of one (32 of each
    // CTA's 64 positions). Two steps' scores lie in tensor memory, so that the next one's product runs beside the
    // softmax. At 256 a CTA has the SM; at 128 a step's products take a quarter of that time and its softmax, a chain
    // of waits, is what lasts: two CTAs share the SM (at 80 registers a thread, 32 bytes of which are spilled).
    // Seven packed prompts of 1 to 3000 rows, 24 query and 4 KV heads, behind up to 8191 positions: 252 us; when
    // these were compared, at 250, with whole tiles, one at a time, 265 us, and with one CTA an SM 331 us
    static constexpr int kCtas = D == 256 ? 1 : 2, kHalves = D == 256 ? 1 : 2;
    static constexpr int kCols = 64 / kHalves, kStep = 2 * kCols;   // columns of a thread, of a step
    static constexpr int kStages = D == 256 ? 5 : 4;
    static constexpr int kRing = kQB, kShared = kQB + kStages * kStageB;   // offsets in shared memory
    static constexpr int kSmem = kShared + (int)sizeof(Shared);
    static_assert(kSmem <= (kCtas == 1 ? 232448 : 115712), "shared memory of a CTA");
    static constexpr uint32_t kO = 0, kS = D;               // TMEM columns: O, then two steps' scores
    static constexpr uint32_t kTmem = D + 2 * kStep;
    static_assert(kTmem * kCtas == 512, "tensor memory of the SM");
    static constexpr int kOutB = D * 4 + 16;                // a row of O on its way out
    static_assert(kRows * kOutB <= kQB + kStages * kStageB, "the output rows reuse the queries and the ring");
    // the stage that holds K tile j, V tile j of n, in the order in which they are read: K 0, K 1, V 0, K 2, V 1, .. by
    // steps of a tile, K 0, V 0, K 1, V 1, .. by halves
    __device__ static uint32_t k_stage(int j) { return kHalves == 2 ? 2 * j : j == 0 ? 0 : 2 * j - 1; }
    __device__ static uint32_t v_stage(int j, int n) { return kHalves == 2 || j == n - 1 ? 2 * j + 1 : 2 * j + 2; }
};

__device__ __forceinline__ uint32_t cluster_addr(const void *p, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
// After writes to shared memory that the pair's MMAs read.
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Where no generic write has to be seen by the other CTA: P goes through tensor memory, ordered by the
// tcgen05 fences, and copies complete on the barrier themselves. A release at cluster scope takes 1200
// cycles here, in every tile's critical path.
__device__ __forceinline__ void signal_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_tx_cluster(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                 : "memory");
}
// Bounded wait: a barrier that never completes sets `stop` in both CTAs of the pair, which depend on each other, and
// lets every later wait of theirs go at once.
__device__ __forceinline__ bool wait_bar(uint64_t *bar, uint32_t parity, volatile int *stop, uint32_t tries, uint32_t nap) {
    for (uint32_t n = 0; n < tries; ++n) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(nap)
            : "memory");
        if (ok) return true;
        if (*stop) return false;
    }
    for (int r = 0; r < 2; ++r)
        asm volatile("st.shared::cluster.u32 [%0], 1;" ::"r"(cluster_addr(const_cast<int *>(stop), r)) : "memory");
    return false;
}
// A box of page rows: coordinates (column 0, row, panel of 64 columns, head, page).
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap *map, int panel, int row, int head, int page,
                                        uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(map), "r"(0), "r"(row), "r"(panel), "r"(head), "r"(page), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap *map, int col, int row, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(dst),
        "l"(map), "r"(col), "r"(row), "r"(bar)
        : "memory");
}
// The MMAs and commits are executed by a whole warp, of which one lane (`one` != 0) issues: operands
// that are the same in all lanes stay in uniform registers. In a branch of one lane each MMA took 85
// cycles to issue, more than the 64 that it runs.
__device__ __forceinline__ void mma2_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one)
        : "memory");
}
__device__ __forceinline__ void mma2_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one)
        : "memory");
}
// All MMAs issued so far have completed: one arrival at the barrier of both CTAs.
__device__ __forceinline__ void commit2(uint64_t *bar, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3), "r"(one)
        : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
// [row][64 columns] panels, 128-byte swizzle, 8 rows apart 1024 bytes. K-major: the columns are the
// sum's index. MN-major: the rows are, and 64-column panels lie `panel` bytes apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) { return sw128_desc(addr); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t panel) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)(panel >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint32_t idesc2(int n, int b_mn) {   // bf16 x bf16 -> fp32, M = 256
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | (16u << 24);
}
__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The two warps of a row quarter.
__device__ __forceinline__ void pair_sync(int quad) { asm volatile("bar.sync %0, 64;" ::"r"(quad + 1) : "memory"); }
__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The prepared, scaled queries in bf16, [KV head][row][head of the group][D], so that the rows of a
// tile lie together: a kernel of its own (and launch), since the tiles' kernel has one warp a
// scheduler and would spend tens of microseconds a unit on it. One (cos, sin) table a row, a warp
// per (row, head).
constexpr int kPrepThreads = 256, kPrepRows = 8;

template <int D, bool kBf16>
__global__ void __launch_bounds__(kPrepThreads) k_prefill_queries(const __grid_constant__ PrefillArgs a) {
    constexpr int E = D / 32, kAtOnce = 4;
    __shared__ __align__(16) float2 cs[kPrepRows][128];
    __shared__ int at[kPrepRows], live[kPrepRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, half = a.rot.half;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int row0 = blockIdx.x * a.prep_rows, rows = min(a.prep_rows, a.total_rows - row0);
    const int heads = a.kv_heads * a.group;
    // 8 / prep_rows (a power of two) warps share a row
    const int share_log = a.share_log, share = 1 << share_log, mine = warp >> share_log, first = warp & (share - 1);
    float next[kAtOnce][E], w[E];
    const long long src = (long long)(row0 + min(mine, rows - 1)) * a.q_stride + E * lane;
    const int step = a.gated ? 2 * D : D;
    auto load = [&](int h0) {   // a warp's next heads, on their way together
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x)
            load_typed<E, kBf16>(a.q, src + (long long)min(h0 + (x << share_log), heads - 1) * step, next[x]);
    };
    load(first);
    load_weight<E>(a.h.q_norm, lane, w);
    const double freq = half > 0 ? rotary_freq(a.rot, tid & (half - 1)) : 0.0;
    if (tid < rows) {
        const int r = row0 + tid, b = find_sequence(a.cu_rows, a.num_seqs, r);
        live[tid] = b >= 0;
        at[tid] = b >= 0 ? (int)((long long)a.kv_lens[b] - a.cu_rows[b + 1] + r) : 0;
    }
    __syncthreads();
    if (half > 0)
        for (int r = tid / half; r < rows; r += kPrepThreads / half) cs[r][tid & (half - 1)] = rotary_cs(freq, at[r]);
    __syncthreads();
    if (mine >= rows || !live[mine]) return;
    for (int h0 = first; h0 < heads; h0 += kAtOnce << share_log) {
        float v[kAtOnce][E];
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x)
#pragma unroll
            for (int i = 0; i < E; ++i) v[x][i] = next[x][i];
        if (h0 + (kAtOnce << share_log) < heads) load(h0 + (kAtOnce << share_log));
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
            const int h = h0 + (x << share_log);
            if (h >= heads) break;
            prepare_head<E>(v[x], w, a.h.q_norm != nullptr, a.h.eps, cs[mine], half, lane);
#pragma unroll
            for (int i = 0; i < E; ++i) v[x][i] *= a.scale;
            const int kvh = h / a.group;
            store_bf16<E>(a.q_ready + (((long long)kvh * a.total_rows + row0 + mine) * a.group + (h - kvh * a.group)) * D + E * lane,
                          v[x]);
        }
    }
}

// A warp that copies one unit's K tiles, or its V tiles, into the ring. The ring's stages are taken
// in the order of the MMAs (Cfg::k_stage, v_stage), so each of the two warps knows its stages.
template <int D>
struct Copier {
    const PrefillArgs &a;
    Shared *S;
    uint8_t *ring;
    int b, kvh, rank, lane, len;   // len: positions that exist
    int page = -1, row = 0;        // this lane's box of the current tile (TMA)
    int next_page = -1, next_row = 0;
    uint32_t boxes = 0;

    __device__ __forceinline__ int lookup(int p, int *in_page) const {
        const int slot = (unsigned)p / (unsigned)a.c.page_size;
        *in_page = p - slot * a.c.page_size;
        return slot < a.c.max_pages ? a.c.table[(long long)b * a.c.table_stride + slot] : -1;
    }
    __device__ __forceinline__ int checked(int page_id) const {
        return page_id >= 0 && page_id < a.c.num_pages ? page_id : -1;
    }
    // The boxes of tile `tile` become current; those of the next tile are looked up meanwhile.
    __device__ __forceinline__ void look_ahead(int tile) {
        next_page = -1;
        if (lane < kTile / a.box_rows && tile * kTile + lane * a.box_rows < len)
            next_page = lookup(tile * kTile + lane * a.box_rows, &next_row);
    }
    __device__ __forceinline__ void begin(int tile, bool more) {
        if (a.box_rows == 0) return;
        page = checked(next_page), row = next_row;
        boxes = __ballot_sync(0xffffffffu, page >= 0);
        if (more) look_ahead(tile + 1);
    }
    // The mask of the tile's positions for the softmax.
    __device__ __forceinline__ void mask(int tile) {
        uint32_t *info = S->info[tile % kInfo];
        if (a.box_rows > 0) {
            const int n = kTile / a.box_rows;
            if (lane < 4) {
                uint32_t w = 0;
                for (int i = 0; i < 32; i += min(32, a.box_rows))
                    if (boxes >> ((32 * lane + i) >> a.box_shift) & 1u)
                        w |= (a.box_rows >= 32 ? 0xffffffffu : ((1u << a.box_rows) - 1u) << i);
                info[lane] = w;
            }
            if (lane == 4) info[4] = boxes == (1u << n) - 1u;
        } else {
            uint32_t all = 0xffffffffu;
            for (int i = 0; i < 4; ++i) {
                int r;
                const uint32_t w = __ballot_sync(0xffffffffu, checked(lookup(tile * kTile + 32 * i + lane, &r)) >= 0);
                all &= w;
                if (lane == 0) info[i] = w;
            }
            if (lane == 0) info[4] = all == 0xffffffffu;
        }
        __syncwarp();
    }
    __device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity) const {
        return __all_sync(0xffffffffu, wait_bar(bar, parity, &S->stop, a.tries, a.nap));
    }
    __device__ __forceinline__ bool acquire(uint32_t n, uint32_t *s) const {   // the n-th stage filled
        *s = n % Cfg<D>::kStages;
        return wait(&S->empty[*s], ((n / Cfg<D>::kStages) & 1) ^ 1);
    }
    // Positions p0 .. p0 + n - 1, columns c0 .. c0 + 64 panels - 1, by the warp's own loads and stores.
    __device__ __forceinline__ void by_hand(const uint16_t *src, uint8_t *dst, int p0, int n, int c0, int panels,
                                            bool zero) const {
        const int per = panels * 8;   // 16-byte pieces of a row
        for (int base = 0; base < n; base += 32) {
            int in_page;
            const int p = p0 + base + lane, pg = p < len ? checked(lookup(p, &in_page)) : -1;
            const long long mine = pg < 0 ? -1
                                          : (long long)pg * a.c.page_stride + (long long)in_page * a.c.row_stride +
                                                (long long)kvh * a.c.head_stride;
#pragma unroll 4
            for (int i = lane; i < 32 * per; i += 32) {
                const int r = i / per, x = i - r * per, panel = x >> 3, chunk = x & 7;
                const long long off = __shfl_sync(0xffffffffu, mine, r);
                uint4 u = make_uint4(0, 0, 0, 0);
                if (off >= 0) u = *reinterpret_cast<const uint4 *>(src + off + c0 + 8 * x);
                if (off >= 0 || zero) *reinterpret_cast<uint4 *>(dst + panel * n * 128 + sw128_off(base + r, chunk)) = u;
            }
            __syncwarp();
        }
        fence_async_smem();
        __syncwarp();
    }
    // This CTA's 64 positions of the tile's K: panels of [64 rows][64 columns]. False: a wait has run out, and nothing
    // more may be copied.
    __device__ __forceinline__ bool keys(int tile, uint32_t n) {
        mask(tile);
        uint32_t s;
        if (!acquire(n, &s)) return false;
        uint8_t *dst = ring + s * Cfg<D>::kStageB;
        const uint32_t bar = cluster_addr(&S->full[s], 0);
        if (a.box_rows == 0) {
            by_hand(a.c.k, dst, tile * kTile + 64 * rank, 64, 0, D / 64, false);
            if (lane == 0) arrive_cluster(bar);
            return true;
        }
        const int per = 64 >> a.box_shift, first = rank * per;
        const uint32_t mine = (boxes >> first) & ((1u << per) - 1u);
        if (lane == 0) arrive_tx_cluster(bar, __popc(mine) * a.box_rows * D * 2);
        __syncwarp();
        if (lane >= first && lane < first + per && page >= 0) {
            const uint32_t at = smem_u32(dst) + (lane - first) * a.box_rows * 128;
            if (a.box_rows == 64) {   // all panels in one copy
                tma_box(at, &a.k_map, 0, row, kvh, page, bar);
            } else {
                for (int p = 0; p < D / 64; ++p) tma_box(at + p * 8192, &a.k_map, p, row, kvh, page, bar);
            }
        }
        return true;
    }
    // This CTA's half of the columns of all of the tile's V. One copy a box: [box][panel][rows][64].
    __device__ __forceinline__ bool values(int tile, uint32_t n) {
        uint32_t s;
        if (!acquire(n, &s)) return false;
        uint8_t *dst = ring + s * Cfg<D>::kStageB;
        const uint32_t bar = cluster_addr(&S->full[s], 0);
        constexpr int kPanels = D / 128;
        if (a.box_rows == 0) {
            by_hand(a.c.v, dst, tile * kTile, kTile, rank * (D / 2), kPanels, true);
            if (lane == 0) arrive_cluster(bar);
            return true;
        }
        const bool clean = __popc(boxes) == kTile >> a.box_shift && (tile + 1) * kTile <= len;
        const uint32_t bytes = __popc(boxes) * a.box_rows * 128 * kPanels;
        const uint32_t to = clean ? bar : cluster_addr(&S->landed, rank);
        if (lane == 0) arrive_tx_cluster(to, bytes);
        __syncwarp();
        if (page >= 0)
            tma_box(smem_u32(dst) + lane * a.box_rows * 128 * kPanels, &a.v_map, rank * kPanels, row, kvh, page, to);
        if (!clean) {
            if (!wait(&S->landed, landed & 1)) return false;
            ++landed;
            // rows that are no positions: a box's rows [exist, box_rows), or all of them
            for (int i = 0; i < kTile >> a.box_shift; ++i) {
                const int exist = (boxes >> i & 1u) ? max(0, min(a.box_rows, len - tile * kTile - i * a.box_rows)) : 0;
                uint8_t *box = dst + i * a.box_rows * 128 * kPanels;
                for (int x = lane; x < (a.box_rows - exist) * 8 * kPanels; x += 32) {
                    const int panel = kPanels == 1 ? 0 : x & 1, y = x / kPanels;
                    *reinterpret_cast<uint4 *>(box + panel * a.box_rows * 128 + exist * 128 + y * 16) = make_uint4(0, 0, 0, 0);
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) arrive_cluster(bar);
        }
        return true;
    }
    uint32_t landed = 0;
};

template <int D>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, Cfg<D>::kCtas) k_prefill_pairs(const __grid_constant__ PrefillArgs a) {
    using C = Cfg<D>;
    extern __shared__ __align__(1024) uint8_t raw[];   // the only shared memory: queries, ring, the rest
    cg::cluster_group cluster = cg::this_cluster();
    uint8_t *q_smem = raw, *ring = raw + C::kRing;
    Shared &S = *reinterpret_cast<Shared *>(raw + C::kShared);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)cluster.block_rank();
    const int per_cta = kRows / a.group, per_unit = 2 * per_cta;   // tokens

    // ---- the unit: (sequence, query tile, KV head). Units are handed to SMs as these become free, so a long one that
    // begins last would run alone. Up to 32 sequences, a lane each: in the order of how many tiles of positions they
    // walk over, the most first. The length of this one by bisection over how many units are at least as long, each
    // sequence's by one division; by every warp for itself. More sequences: by sequence, the last tiles (the
    // longest) first, since a bisection over them costs every unit microseconds.
    const int unit = blockIdx.x >> 1, kvh = unit % a.kv_heads, want = unit / a.kv_heads;
    auto rows_of = [&](int b) { return max(0, min(a.total_rows, a.cu_rows[b + 1]) - max(0, a.cu_rows[b])); };
    auto units_of = [&](int rows) { return (int)(((unsigned)rows + per_unit - 1) / per_unit); };
    if (tid == 0) {
        S.unit_seq = -1;
        S.stop = 0;
    }
    if (a.num_seqs == 1) {   // its last units are its longest
        const int units = units_of(rows_of(0));
        if (tid == 0 && want < units) {
            S.unit_seq = 0;
            S.unit_off = units - 1 - want;
        }
    } else if (a.num_seqs <= 32) {
        const bool own = lane < a.num_seqs;
        const int rows = own ? rows_of(lane) : 0, units = units_of(rows);
        const long long len = own ? a.kv_lens[lane] : 0, there = max(0ll, min(len, (long long)a.c.capacity));
        auto from = [&](int tiles) {   // of this lane's units, the first that walks over `tiles` tiles or more (they grow)
            if (tiles <= 0 || units == 0) return 0;
            const long long need = (long long)(tiles - 1) * kTile + 1;   // positions
            if (there < need) return units;
            const long long r = need - (len - rows);   // of the sequence's rows, that many
            return r <= 0 ? 0 : min(units_of((int)r) - 1, units - 1);
        };
        auto at_least = [&](int tiles) { return (int)__reduce_add_sync(0xffffffffu, units - from(tiles)); };
        if (at_least(0) > want) {
            // at_least(lo) > want >= at_least(hi) = longer
            int lo = 0, hi = ((int)__reduce_max_sync(0xffffffffu, (int)there) + kTile - 1) / kTile + 1, longer = 0;
            while (hi - lo > 1) {
                const int mid = lo + (hi - lo) / 2, n = at_least(mid);
                if (n > want)
                    lo = mid;
                else
                    hi = mid, longer = n;
            }
            // of the units of length lo, the (want - longer)-th
            const int k = from(lo), same = from(lo + 1) - k;
            int before = same;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += v;
            }
            before -= same;
            const int nth = want - longer - before;
            if (warp == 0 && nth >= 0 && nth < same) {
                S.unit_seq = lane;
                S.unit_off = k + nth;
            }
        }
    } else {
        const int per = (a.num_seqs + kThreads - 1) / kThreads;
        const int first = min(a.num_seqs, tid * per), last = min(a.num_seqs, first + per);
        int own = 0;
        for (int b = first; b < last; ++b) own += units_of(rows_of(b));
        int before = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += v;
        }
        if (lane == 31) S.scan[warp] = before;
        __syncthreads();
        before -= own;
        for (int w = 0; w < warp; ++w) before += S.scan[w];
        if (want >= before && want < before + own)
            for (int b = first; b < last; ++b) {
                const int n = units_of(rows_of(b));
                if (want < before + n) {
                    S.unit_seq = b;
                    S.unit_off = n - 1 - (want - before);
                    break;
                }
                before += n;
            }
    }
    __syncthreads();
    const int b = S.unit_seq;
    if (b < 0) {   // both CTAs of the pair: there are fewer units than the grid has room for
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const int lo = max(0, a.cu_rows[b]), rows_b = min(a.total_rows, a.cu_rows[b + 1]) - lo;
    const int tok0 = S.unit_off * per_unit;          // first token of the pair in the sequence
    const long long len64 = a.kv_lens[b];
    const long long seq0 = len64 - rows_b;                // position of the sequence's first row
    const int len = (int)max(0ll, min(len64, (long long)a.c.capacity));
    const long long last_pos = min((long long)len, seq0 + min(rows_b, tok0 + per_unit)) - 1;
    const int n_tiles = last_pos < 0 ? 0 : (int)(last_pos / kTile) + 1;   // both CTAs alike
    const int my_tok0 = tok0 + rank * per_cta;            // this CTA's tokens
    const int my_rows = max(0, min(per_cta, rows_b - my_tok0));

    // ---- barriers and tensor memory
    if (tid == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&S.full[s], 2);    // one arrival of each CTA's copier (the first CTA's barrier is used)
            mbar_init(&S.empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&S.s_full[s], 1);
            mbar_init(&S.p_ready[s][0], 16);   // the softmax warps of both CTAs
            mbar_init(&S.p_ready[s][1], 16);
        }
        mbar_init(&S.landed, 1);
        mbar_init(&S.o_done, 1);
        mbar_init(&S.done, 1);
        mbar_init(&S.q_ready, 2);
        mbar_fence_init();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S.tmem)), "n"(C::kTmem));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    tc_fence_before();
    cluster.sync();
    tc_fence_after();
    const uint32_t tmem = S.tmem;

    if (warp == 8) {
        if (n_tiles > 0) {
            Copier<D> cp{a, &S, ring, b, kvh, rank, lane, len};
            if (a.box_rows > 0) cp.look_ahead(0);
            for (int j = 0; j < n_tiles; ++j) {
                cp.begin(j, j + 1 < n_tiles);
                if (!cp.keys(j, C::k_stage(j))) break;
                if (j == 0) {
                    asm volatile("griddepcontrol.wait;" ::: "memory");   // the prepared queries
                    if (lane == 0) {
                        const uint32_t bar = cluster_addr(&S.q_ready, 0);
                        arrive_tx_cluster(bar, C::kQB);
                        for (int p = 0; p < D / 64; ++p)
                            tma_rows(smem_u32(q_smem) + p * (kRows * 128), &a.q_map, 64 * p,
                                     (kvh * a.total_rows + lo + my_tok0) * a.group, bar);
                    }
                    __syncwarp();
                }
            }
        }
        // Every CTA waits, those that need no queries too, so that this launch never ends before the one that
        // prepares them: a call behind this one may use the workspace
        asm volatile("griddepcontrol.wait;" ::: "memory");
    } else if (warp == 10) {
        Copier<D> cp{a, &S, ring, b, kvh, rank, lane, len};
        if (a.box_rows > 0 && n_tiles > 0) cp.look_ahead(0);
        for (int j = 0; j < n_tiles; ++j) {
            cp.begin(j, j + 1 < n_tiles);
            if (!cp.values(j, C::v_stage(j, n_tiles))) break;
        }
    } else if (warp == 9) {
        if (rank == 0 && n_tiles > 0) {
            // every value below is the same in all lanes, and the compiler can see it (votes, shuffles)
            const uint32_t one = elect_one();
            const uint32_t q_at = smem_u32(q_smem), ring_at = smem_u32(ring);
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const int n = __shfl_sync(0xffffffffu, n_tiles, 0);
            const uint32_t id_s = idesc2(C::kStep, 0), id_o = idesc2(D, 1);
            const int steps = n * C::kHalves;
            // V in shared memory: [box][panel][rows][64], one box when the warp copies
            const uint32_t v_rows = a.box_rows > 0 ? a.box_rows : kTile, v_shift = a.box_rows > 0 ? a.box_shift - 4 : 3;
            auto wait = [&](uint64_t *bar, uint32_t parity) {
                return __all_sync(0xffffffffu, wait_bar(bar, parity, &S.stop, a.tries, a.nap));
            };
            // the stages that the next K and V tile are read from, and the parity of their filling
            uint32_t k_at = 0, k_round = 0, v_at = C::v_stage(0, n), v_round = 0;
            auto advance = [&](uint32_t &at, uint32_t &round, uint32_t by) {
                at += by;
                if (at >= C::kStages) at -= C::kStages, round ^= 1;
            };
            // S of step t: of its tile (half x)
            auto qk = [&](int t) {
                const int j = t / C::kHalves, x = t % C::kHalves;
                const uint32_t at = ring_at + k_at * C::kStageB + x * 32 * 128;
#pragma unroll
                for (uint32_t i = 0; i < D / 16; ++i)
                    mma2_ss(tm + C::kS + (t & 1) * C::kStep, desc_k(q_at + (i >> 2) * (kRows * 128) + (i & 3) * 32),
                            desc_k(at + (i >> 2) * 8192 + (i & 3) * 32), id_s, i > 0 ? 1u : 0u, one);
                if (x == C::kHalves - 1) {
                    commit2(&S.empty[k_at], one);
                    advance(k_at, k_round, C::k_stage(j + 1) - C::k_stage(j));
                }
                commit2(&S.s_full[t & 1], one);
            };
            // P V of step t, in the 32 positions of each CTA's half that the softmax hands over together. The 16
            // positions i of P lie over the scores that they were made of
            auto pv = [&](int t) {
                const int j = t / C::kHalves, x = t % C::kHalves;
                const uint32_t at = ring_at + v_at * C::kStageB;
                const uint32_t p = tm + C::kS + (t & 1) * C::kStep;
#pragma unroll
                for (uint32_t h = 0; h < 2 / C::kHalves; ++h) {
                    if (!wait(&S.p_ready[t & 1][h], t >> 1 & 1)) return false;
                    tc_fence_after();
#pragma unroll
                    for (uint32_t y = 0; y < 4; ++y) {
                        const uint32_t i = 2 * (C::kHalves == 2 ? x : h) + (y & 1) + 4 * (y >> 1);
                        mma2_ts(tm + C::kO, p + C::kCols * (y >> 1) + 32 * h + 8 * (y & 1),
                                desc_mn(at + (i >> v_shift) * (v_rows * D) + (i & ((1u << v_shift) - 1)) * 2048, v_rows * 128),
                                id_o, (t > 0 || h + y > 0) ? 1u : 0u, one);
                    }
                }
                if (x == C::kHalves - 1) {
                    commit2(&S.empty[v_at], one);
                    advance(v_at, v_round, C::v_stage(j + 1, n) - C::v_stage(j, n));
                }
                commit2(&S.o_done, one);
                return true;
            };
            // S 0, S 1, P V 0, S 2, P V 1, ..: S of step t + 1 runs while step t is in the softmax. What was
            // copied is waited for ahead of P, so that P V t and S t + 2 follow it at once.
            bool ok = wait(&S.q_ready, 0);
            for (int t = -2; t < steps && ok; ++t) {
                if (t >= 0 && t % C::kHalves == 0) ok = wait(&S.full[v_at], v_round);
                if (t + 2 < steps && (t + 2) % C::kHalves == 0) ok = ok && wait(&S.full[k_at], k_round);
                tc_fence_after();
                if (t >= 0 && ok) ok = pv(t);
                if (t + 2 < steps && ok) qk(t + 2);
            }
            if (ok) commit2(&S.done, one);
        }
    } else {
        // ---- softmax: two threads a row, 64 columns each; warps w and w + 4 hold the same 32 rows
        const int wg = warp >> 2, quad = warp & 3, r_cta = quad * 32 + lane;
        const int token = r_cta / a.group;
        const bool live = token < my_rows;
        const long long pos64 = seq0 + my_tok0 + token;
        // position up to which this row sees; -1: nothing
        const int pos = live && pos64 >= 0 ? (int)min(pos64, (long long)len - 1) : -1;
        float m = -INFINITY, l = 0.f;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        if (n_tiles > 0) {
            const uint32_t p_bar = cluster_addr(&S.p_ready[0][0], 0);
            // the first position that some row of this warp does not see
            const int seen = __reduce_min_sync(0xffffffffu, live ? pos + 1 : 0x7fffffff);
            for (int t = 0; t < n_tiles * C::kHalves; ++t) {
                const int j = t / C::kHalves, x0 = t % C::kHalves;
                wait_bar(&S.s_full[t & 1], t >> 1 & 1, &S.stop, a.tries, a.nap);
                tc_fence_after();
                const uint32_t st = tmem + lanes + C::kS + (t & 1) * C::kStep + C::kCols * wg;
                float s[C::kCols];
#pragma unroll
                for (int c = 0; c < C::kCols / 32; ++c) tc_ld32(st + 32 * c, reinterpret_cast<uint32_t *>(s) + 32 * c);
                tc_wait_ld();
                const uint32_t *info = S.info[j % kInfo];
                if ((j + 1) * kTile > seen || !info[4]) {
                    const int n = pos - j * kTile - 64 * wg - 32 * x0;   // columns 0..n of this thread's are seen
#pragma unroll
                    for (int c = 0; c < C::kCols / 32; ++c) {
                        const int k = n - 32 * c;
                        const uint32_t w = info[2 * wg + x0 + c] & (k >= 31 ? 0xffffffffu : k < 0 ? 0u : (2u << k) - 1u);
#pragma unroll
                        for (int i = 0; i < 32; ++i) s[32 * c + i] = w >> i & 1u ? s[32 * c + i] : -INFINITY;
                    }
                }
                float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i < C::kCols - 4; i += 8)
#pragma unroll
                    for (int x = 0; x < 4; ++x) mx[x] = max3(mx[x], s[i + x], s[i + 4 + x]);
#pragma unroll
                for (int x = 0; x < 4; ++x) mx[x] = fmaxf(mx[x], s[C::kCols - 4 + x]);
                float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                S.row_max[t & 1][wg][r_cta] = top;
                pair_sync(quad);   // the other part's maximum
                top = fmaxf(top, S.row_max[t & 1][wg ^ 1][r_cta]);
                const bool grow = top > m + 8.0f || (m == -INFINITY && top > m);
                const float mn = grow ? top : m;
                const float base = mn == -INFINITY ? 0.f : mn;
                const bool scale_o = t > 0 && __any_sync(0xffffffffu, grow);
                const float c = grow ? ex2f(m - base) : 1.0f;
                l *= c;
                m = mn;
                if (scale_o) {
                    // P V of step t - 1 is the last that added to O; that of step t - 2 is complete, since S of
                    // step t, issued after it, is
                    wait_bar(&S.o_done, (t - 1) & 1, &S.stop, a.tries, a.nap);
                    tc_fence_after();
#pragma unroll 1
                    for (int x = wg * (D / 2); x < (wg + 1) * (D / 2); x += 32) {
                        uint32_t o[32];
                        tc_ld32(tmem + lanes + C::kO + x, o);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * c);
                        tc_st16(tmem + lanes + C::kO + x, o);
                        tc_st16(tmem + lanes + C::kO + x + 16, o + 16);
                    }
                }
                const uint64_t neg = pack_f32x2(-base, -base);
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (int x = 0; x < C::kCols / 32; ++x) {   // 32 columns at a time into the MMAs' hands
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float e0, e1;
                        unpack_f32x2(add_f32x2(pack_f32x2(s[32 * x + 2 * i], s[32 * x + 2 * i + 1]), neg), e0, e1);
                        e0 = ex2f(e0), e1 = ex2f(e1);
                        sum[i & 1] = add_f32x2(sum[i & 1], pack_f32x2(e0, e1));
                        p[i] = pack2_bf16(e0, e1);
                    }
                    tc_st16(st + 32 * x, p);
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) signal_cluster(p_bar + (t & 1) * 16 + x * 8);
                }
                float s0, s1;
                unpack_f32x2(add_f32x2(sum[0], sum[1]), s0, s1);
                l += s0 + s1;
            }
            wait_bar(&S.done, 0, &S.stop, a.tries, a.nap);
            tc_fence_after();
            float(*sums)[kRows] = S.row_max[n_tiles * C::kHalves & 1];   // the parity that the last step left alone
            sums[wg][r_cta] = l;
            pair_sync(quad);
            l += sums[wg ^ 1][r_cta];
        }
        // ---- O / l through shared memory (the MMAs have read the queries and the ring for the last
        // time), so that a warp gates and stores a row of D at a time
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        uint8_t *rows_out = q_smem + quad * 32 * C::kOutB;
        if (n_tiles > 0) {
            uint8_t *to = rows_out + lane * C::kOutB;
#pragma unroll 1
            for (int x = wg * (D / 2); x < (wg + 1) * (D / 2); x += 32) {
                uint32_t o[32];
                tc_ld32(tmem + lanes + C::kO + x, o);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = inv == 0.f ? 0u : __float_as_uint(__uint_as_float(o[i]) * inv);
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                    *reinterpret_cast<uint4 *>(to + (x + i) * 4) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
            pair_sync(quad);
        }
        constexpr int E = D / 32;
        const int heads = a.kv_heads * a.group, first = wg * 16;   // this warp's 16 of the pair's 32 rows
        const int mine = min(first + 16, my_rows * a.group - quad * 32);
        constexpr int kAtOnce = 8;   // rows whose gates are on their way together
        auto store_rows = [&](auto bf16) {
            for (int i0 = first; i0 < mine; i0 += kAtOnce) {
                float g[kAtOnce][E];
                long long at[kAtOnce];
#pragma unroll
                for (int y = 0; y < kAtOnce; ++y) {
                    const int rr = quad * 32 + min(i0 + y, mine - 1), tok = rr / a.group, h = kvh * a.group + rr - tok * a.group;
                    const long long r = (long long)lo + my_tok0 + tok;
                    at[y] = (r * heads + h) * D + E * lane;
                    if (a.gated) load_typed<E, decltype(bf16)::value>(a.q, r * a.q_stride + (long long)h * 2 * D + D + E * lane, g[y]);
                }
#pragma unroll
                for (int y = 0; y < kAtOnce; ++y) {
                    if (i0 + y >= mine) break;
                    float v[E];
#pragma unroll
                    for (int x = 0; x < E; ++x) v[x] = 0.f;
                    if (n_tiles > 0) {
                        const float4 *src = reinterpret_cast<const float4 *>(rows_out + (i0 + y) * C::kOutB + E * lane * 4);
#pragma unroll
                        for (int x = 0; x < E / 4; ++x) {
                            const float4 f = src[x];
                            v[4 * x] = f.x, v[4 * x + 1] = f.y, v[4 * x + 2] = f.z, v[4 * x + 3] = f.w;
                        }
                    }
                    if (a.gated)
#pragma unroll
                        for (int x = 0; x < E; ++x) v[x] = __fdividef(v[x], 1.0f + __expf(-g[y][x]));
                    store_bf16<E>(a.out + at[y], v);
                }
            }
        };
        if (a.x_bf16)
            store_rows(std::true_type{});
        else
            store_rows(std::false_type{});
        if (*static_cast<volatile int *>(&S.stop)) {   // a copy or product that never came must not pass for an answer
            __syncwarp();
            for (int i = first; i < mine; ++i) {
                const int rr = quad * 32 + i, tok = rr / a.group, h = kvh * a.group + rr - tok * a.group;
                for (int d = lane; d < D; d += 32) a.out[(((long long)lo + my_tok0 + tok) * heads + h) * D + d] = 0x7fc0;
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (S.stop && warp == 8) {
        // what is in flight lands before the shared and the tensor memory go: of either parity of each barrier, as
        // one of them is in flight; bounded too
        auto settle = [&](uint64_t *bar) {
            for (int p = 0; p < 2; ++p)
                for (int n = 0; n < 1000 && !mbar_try_wait_sleep(bar, p, 1000); ++n) {}
        };
        for (int s = 0; s < C::kStages; ++s) settle(&S.full[s]), settle(&S.empty[s]);
        settle(&S.landed);
        settle(&S.q_ready);
        settle(&S.o_done);
    }
    cluster.sync();   // neither CTA leaves while the other may still signal it
    tc_fence_after();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::kTmem));
}

bool query_map(CUtensorMap *m, const uint16_t *base, int d, long long rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)d * 2};
    const cuuint32_t box[2] = {64, kRows}, es[2] = {1, 1};
    const TensorMapEncode fn = tensor_map_encode();
    return fn != nullptr &&
           fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<uint16_t *>(base), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
cudaError_t launch(const PrefillArgs &a, long long units, cudaStream_t st) {
    static SmemOnce once;
    cudaError_t e = once.set(k_prefill_pairs<D>, Cfg<D>::kSmem);
    if (e != cudaSuccess) return e;
    (a.x_bf16 ? k_prefill_queries<D, true> : k_prefill_queries<D, false>)
        <<<(a.total_rows + a.prep_rows - 1) / a.prep_rows, kPrepThreads, 0, st>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    // the tiles' kernel sets up and reads K while the queries are prepared
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * units));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg<D>::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_prefill_pairs<D>, a);
}

}  // namespace
}  // namespace nmoe

using namespace nmoe;

extern "C" size_t nmoe_full_attn_prefill_paged_workspace_bytes(const nmoe_full_attn_shape *s, int num_seqs,
                                                               int total_rows) {
    const nmoe_full_attn_weights none = {nullptr, nullptr};
    if (num_seqs < 1 || total_rows < 1 || check_full_attn_shape(&none, s) != NMOE_OK) return 0;
    return (size_t)total_rows * s->q_heads * s->head_dim * sizeof(uint16_t);
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
    if (out == nullptr || workspace == nullptr || !aligned_to(out, 16) || !aligned_to(workspace, 16))
        return full_attn_fail(NMOE_EINVAL, "out or workspace is NULL or not 16-byte aligned");
    if ((long long)total_rows * shape->q_heads > 2147483647ll) return full_attn_fail(NMOE_EINVAL, "too many rows");
    if (!(scale >= 0.f && scale <= 3.0e38f)) return full_attn_fail(NMOE_EINVAL, "scale must be finite and not negative");
    fill_rotary(shape, &a.rot);
    a.h = {w->q_norm, nullptr, shape->norm_eps};
    a.cu_rows = cu_rows;
    a.kv_lens = kv_lens;
    a.q = q;
    a.out = out;
    a.scale = (scale == 0.f ? 1.0f / sqrtf((float)shape->head_dim) : scale) * 1.4426950408889634f;
    a.num_seqs = num_seqs;
    a.total_rows = total_rows;
    a.kv_heads = shape->kv_heads;
    a.group = shape->q_heads / shape->kv_heads;
    a.gated = shape->gated;
    a.x_bf16 = x_dtype == NMOE_DTYPE_BF16;
    a.q_ready = static_cast<uint16_t *>(workspace);
    const uint32_t tries = wait_tries();
    a.tries = tries / 64 + (tries % 64 != 0);   // of up to 20 us each
    a.nap = tries < 20000 ? tries : 20000;
    int sms = 0;
    if ((rc = device_sm_count(&sms)) != NMOE_OK) return rc;
    rows_a_cta(total_rows / (4 * sms), &a.prep_rows, &a.share_log);
    if (!query_map(&a.q_map, a.q_ready, shape->head_dim, (long long)total_rows * shape->q_heads))
        return full_attn_fail(NMOE_ECUDA, "cuTensorMapEncodeTiled failed");
    // boxes of the largest power of two of rows that divides a page, 16 to 64: an MMA's 16 positions lie
    // in one box. A page's K box takes all panels at 64 rows (the tile's rows are then 128 bytes apart).
    int box = a.c.page_size & -a.c.page_size, shift = 0;
    box = box > 64 ? 64 : box;
    while (1 << shift < box) ++shift;
    a.box_rows = box < 16 ? 0 : box;
    a.box_shift = shift;
    const int d = shape->head_dim;
    if (a.box_rows > 0 && !(page_map(&a.k_map, a.c, a.c.k, d, a.kv_heads, box, box == 64 ? d / 64 : 1) &&
                            page_map(&a.v_map, a.c, a.c.v, d, a.kv_heads, box, d / 128)))
        a.box_rows = 0;   // strides that a tensor map cannot have: the warp copies
    const int per_unit = 2 * (kRows / a.group);
    const long long units = ((long long)total_rows / per_unit + num_seqs) * a.kv_heads;
    if (2 * units > 2147483647ll) return full_attn_fail(NMOE_EINVAL, "too many rows or sequences");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = shape->head_dim == 256 ? launch<256>(a, units, st) : launch<128>(a, units, st);
    return e == cudaSuccess ? NMOE_OK : full_attn_fail(NMOE_ECUDA, "prefill: %s", cudaGetErrorString(e));
}
