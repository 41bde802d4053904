// Products of token rows with their group's weights, y[r] = x[r] W[e(r)]^T,
// on the 5th-generation tensor cores: bf16 operands, or e4m3 operands with a
// float32 scale for each token and 128 inputs (sx) and for each 128 x 128
// weights (sw):
//   y[r][n] = sum_b sx[b][r] sw[e][n / 128][b] (sum over block b of x w)
// A block's inner sum is four tcgen05.mma of 32 inputs into TMEM; the scales
// differ from block to block, so the epilogue warps read every block's sum
// back and add it, scaled, to float32 registers while the tensor core works
// on the next blocks. bf16 needs none of this: a tile's whole sum stays in
// TMEM.
//
// The groups' rows are contiguous (`off`, on the device): a tile is rows of
// one group. Rows past the group's end that a TMA box brings along belong to
// another group or are zero; they are lanes of the accumulator that are never
// stored.
//
// A tile is up to 128 tokens (the accumulator's lanes, so that a thread's
// token scale is one register) x 256 weight rows (gate/up: 128 of each), with
// two TMEM buffers. Persistent CTAs of specialised warps: warp 0 issues TMA
// copies of 128-byte rows into a ring of 128-byte-swizzled stages, warp 1
// issues the MMAs, warps 2 and 3 stage what the epilogue reads, and sixteen
// warps are the epilogue, 64 accumulator columns each. Three modes:
//   kPair    two CTAs (cta_group::2) share a tile of 256 tokens: each loads its
//            128 tokens and half of the weight rows, so a block costs a CTA 32
//            KB of L2 reads instead of 48. Many tokens a group.
//   kSingle  one CTA a tile, fewer token rows loaded when groups are small: the
//            weights' stream bounds it.
//   kSplit   few tiles: a cluster of up to 8 CTAs shares a tile's blocks; the
//            partial sums meet in distributed shared memory, added in rank
//            order.
// and kSmall, a kernel of its own with the weights on the lanes, for groups of
// a few tokens.
//
// Measured (us of device time a call, replayed from a CUDA graph, the
// quantizer included; as calls in a loop in brackets, with the host's part or
// the power cap where either is more): linear 8192 x 8192 x 4096 e4m3 304 (1.81
// PFLOP/s, 1.10 of the measured bf16 rate) [343 to 352], of 128 tokens 19.1
// [20.6], of one, 4096 x 4096, 11.3 [19]; rows grouped by 128 experts of 768 x
// 2048, bf16: 512 rows 67 (398 MB: 0.91 of the measured copy rate) [68 to 70],
// 32768 rows by Zipf's law 141 (103 GFLOP) [165]; e4m3: 43 [45] and 130 [149].
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <map>
#include <mutex>

#include "experts.cuh"
#include "gmm.cuh"
#include "stages.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace vqmoe {

namespace gm {
using namespace tc;

constexpr int kLanes = 128;                    // rows of an accumulator (MMA M)

// Whether a barrier's phase of that parity is over, without waiting
__device__ __forceinline__ bool test_bar(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
// A whole warp's wait, first without the suspending form (a barrier that is
// ready already costs the least so; `ready`: a test_bar the caller made some
// work ago). One that ran out is recorded where the caller gave a word for it,
// and every later one is skipped.
struct Waiter {
    uint32_t *err;
    bool failed = false;
    __device__ void operator()(uint64_t *bar, uint32_t parity) { (*this)(bar, parity, test_bar(bar, parity)); }
    __device__ void operator()(uint64_t *bar, uint32_t parity, bool ready) {
        if (__all_sync(0xffffffffu, ready) || failed) return;
        const uint32_t a = smem_u32(bar);
        for (int i = 0; i < kPoll; ++i) {
            uint32_t done;
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}\n"
                : "=r"(done)
                : "r"(a), "r"(parity), "r"(kSuspendNs)
                : "memory");
            if (__all_sync(0xffffffffu, done)) return;
        }
        failed = true;
        if (err) atomicExch(err, kWaitPipeline);
    }
};

// One 32-byte-deep MMA of this CTA (PAIR: of both CTAs, issued by the leader)
template <bool FP8, bool PAIR>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
#define VQMOE_MMA(GROUP, KIND)                                                                      \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                   \
                 "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), \
                 "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)                                       \
                 : "memory")
    if (FP8 && PAIR) VQMOE_MMA("2", "f8f6f4");
    else if (FP8) VQMOE_MMA("1", "f8f6f4");
    else if (PAIR) VQMOE_MMA("2", "f16");
    else VQMOE_MMA("1", "f16");
#undef VQMOE_MMA
}

// D f32, A and B e4m3 (kind::f8f6f4) or bf16 (kind::f16), both K-major
constexpr uint32_t idesc_of(bool fp8, int m, int n) {
    return (1u << 4) | (fp8 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// The MMAs issued so far arrive on `bar` when they are done (PAIR: on both
// CTAs' barrier at that place).
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t *bar) {
    if (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(
                smem_u32(bar)),
            "h"((uint16_t)3)
            : "memory");
    else
        tc_commit(bar);
}
__device__ __forceinline__ uint32_t map_cluster(uint32_t saddr, int cta) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(saddr), "r"(cta));
    return r;
}
// An arrival on a barrier of the cluster (an address from map_cluster)
__device__ __forceinline__ void arrive_at(uint32_t addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(addr) : "memory");
}
// A copy of a pair's CTA into its own shared memory that counts on the
// leader's barrier
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void *map, int c0, int c1, uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .b32 r;\n\t"
        "mapa.shared::cluster.u32 r, %2, 0;\n\t"
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
        "{%3, %4}], [r];\n\t}\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
        : "memory");
}

// Two float32 in a 64-bit register, as the packed multiply-add takes them: kept
// packed throughout, so that no moves come between it and tcgen05.ld's registers
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ void fma2(uint64_t &d, uint64_t v, uint64_t s) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;\n" : "+l"(d) : "l"(v), "l"(s));
}
__device__ __forceinline__ float lo2(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi2(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

__device__ __forceinline__ int ld_here(const int *p) {   // not sunk to its use
    int v;
    asm volatile("ld.global.nc.s32 %0, [%1];\n" : "=r"(v) : "l"(p));
    return v;
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
        "%13, %14, %15}, [%16];\n"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}

// One lane of the (converged) warp. The roles that issue copies and MMAs run
// their loops with the whole warp and elect a lane for the issue alone: the
// loop stays uniform, so descriptors and barriers are built in uniform
// registers (an MMA a lane issues from a divergent loop took 92 cycles to
// issue, 58 so: four a block, more than 128 x 16 of them need).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;\n" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void cluster_arrive_wait() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// ------------------------------------------------------- groups and tiles

struct Groups {
    int pre[kMaxGroups + 1];     // token tiles before group e
    int beg[kMaxGroups], end[kMaxGroups];
};

// Warp 0 fills the groups' rows and the running count of their token tiles.
// Whatever the offsets hold, group e has the rows between the largest of the
// first e + 1 offsets and of the first e + 2, all clamped to [0, P]: groups
// never share a row (two tiles would write it, in no order), and their tiles
// are at most the launcher's bound (a cluster of kSplit takes one tile).
__device__ __forceinline__ void build_groups(const GmmArgs &a, Groups &g, int rows_per_tile) {
    const int lane = threadIdx.x & 31;
    const int per = (a.E + 31) / 32, e0 = lane * per, e1 = min(e0 + per, a.E);
    auto tiles = [&](int e) { return (g.end[e] - g.beg[e] + rows_per_tile - 1) / rows_per_tile; };
    int sum = 0;
    bool falls = false;
    for (int e = e0; e < e1; ++e) {
        const int b = min(max(__ldg(a.off + e), 0), a.P), n = min(max(__ldg(a.off + e + 1), 0), a.P);
        falls |= n < b;
        g.beg[e] = b;
        g.end[e] = n;
        sum += (n - b + rows_per_tile - 1) / rows_per_tile;
    }
    if (__any_sync(0xffffffffu, falls)) {          // not as documented: the running maximum, by one lane
        __syncwarp();                              // (a vote orders no memory)
        if (lane == 0)
            for (int e = 0, most = g.beg[0]; e < a.E; ++e) {
                g.beg[e] = most;
                g.end[e] = most = max(most, g.end[e]);
            }
        __syncwarp();
        sum = 0;
        for (int e = e0; e < e1; ++e) sum += tiles(e);
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    int at = inc - sum;
    for (int e = e0; e < e1; ++e) {
        g.pre[e] = at;
        at += tiles(e);
    }
    if (lane == 31) g.pre[a.E] = inc;
}

struct Tile {
    int e, row0, end, nt;        // group, first row, the group's last row + 1, column tile
};

__device__ __forceinline__ Tile locate(const GmmArgs &a, const Groups &g, int tile, int ntiles, int rows_per_tile) {
    Tile t;
    const int j = tile / ntiles;
    t.nt = tile - j * ntiles;
    if (!a.off) {
        t.e = 0;
        t.row0 = j * rows_per_tile;
        t.end = a.P;
        return t;
    }
    int lo = 0, hi = a.E;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (g.pre[mid] <= j) lo = mid;
        else hi = mid;
    }
    t.e = lo;
    t.row0 = g.beg[lo] + (j - g.pre[lo]) * rows_per_tile;
    t.end = g.end[lo];
    return t;
}

// The quantizer's two numbers of a group whose largest |bf16| has the bits
// `amax`: its scale f32(a / 448), and what quantize1() divides by. a is at
// least 2^-100; a NaN or an infinity in the group makes the scale NaN.
struct QScale {
    float s, d, r;
};
__device__ __forceinline__ QScale qscale(uint32_t amax) {
    QScale q;
    const float a = fmaxf(bf16_to_f32(amax), 7.888609052210118e-31f);
    q.s = amax >= 0x7F80u ? __uint_as_float(0x7FC00000u) : __fdiv_rn(a, 448.0f);
    q.d = a * 0.001953125f;                  // a / 512, exact
    q.r = __frcp_rn(q.d);
    return q;
}
// 448 x / a, i.e. (0.875 x) / (a / 512): 0.875 x is exact, one correction of
// the product with the rounded reciprocal by its exact remainder. Where the
// quotient is half way between two e4m3 values it is a float32, and the
// corrected product is that float32; other quotients of two 8-bit numbers lie
// 2^-13 and more (relative) from any half-way point. So the e4m3 rounding
// that follows is the exact quotient's.
__device__ __forceinline__ float quotient(float x, const QScale &q) {
    const float b = 0.875f * x;
    const float y = b * q.r;
    return fmaf(fmaf(-y, q.d, b), q.r, y);
}
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// ------------------------------------------------------------- the kernel

enum Mode { kSingle = 0, kSplit = 1, kPair = 2, kSmall = 3 };

constexpr int kAccCols = 256;                  // accumulator columns: two halves of 128
constexpr int kEpiWarps = 16;                  // a warp of the accumulator's 32 lanes takes 64 columns
constexpr int kThreads = 32 * (4 + kEpiWarps); // TMA, MMA, two stagers, the epilogue
constexpr int kCtlRegs = 56, kEpiRegs = 104;   // setmaxnreg: 128 x 56 + 512 x 104 of the 640 x 96 at launch
constexpr int kGroup = 4, kSlots = 3;          // scale blocks of a staged slot, and the slots
constexpr int kMaxStages = 8;
constexpr int kRingBytes = 160 * 1024;
constexpr int kPartPitch = 260;                // floats of a row of partial sums (kSplit)
constexpr int kPatch = 2048;                   // an epilogue warp's output staging: 32 rows of 64 bytes
constexpr size_t kSmem = 1024 + kRingBytes + kEpiWarps * kPatch;

// SwiGLU / GeGLU of two columns, every step rounded to bf16: packed bf16
__device__ __forceinline__ uint32_t glu_pair(float g0, float g1, float u0, float u1, int act) {
    const uint32_t g = cvt_bf16x2(g0, g1), u = cvt_bf16x2(u0, u1);
    const uint32_t a = act == VQMOE_ACT_GEGLU ? cvt_bf16x2(gelu_tanh_f32(bf_lo(g)), gelu_tanh_f32(bf_hi(g)))
                                              : cvt_bf16x2(silu_fast(bf_lo(g)), silu_fast(bf_hi(g)));
    return cvt_bf16x2(bf_lo(a) * bf_lo(u), bf_hi(a) * bf_hi(u));
}

// What the launcher fixes beyond GmmArgs.
struct Plan {
    int bm;              // token rows a CTA loads for a tile (32, 64 or 128)
    int stages;
    int split;           // kSplit: CTAs of a cluster
    int weights_first;   // the first stages' weights may be read before the kernel's predecessor has finished
};

// The 32 rows a warp's lanes hold, through its patch of shared memory, so that
// a store instruction writes whole rows: lane `lane` puts CH 16-byte chunks of
// its row (put), and CH lanes then write each row (flush). A thread storing its
// own row, 16 bytes in each of 32 rows an instruction, took 12800 cycles of a
// 128 x 256 tile, and the tensor core waits for most of them; this takes 2300
// to 3400.
template <int CH>
struct RowStore {
    uint8_t *patch;
    int lane;
    __device__ static int at(int row, int c) {
        return row * (CH * 16) + 16 * (c ^ (CH == 4 ? (row >> 1) & 3 : (row >> 2) & 1));
    }
    __device__ void put(int c, uint32_t a, uint32_t b, uint32_t d, uint32_t e) const {
        *reinterpret_cast<uint4 *>(patch + at(lane, c)) = make_uint4(a, b, d, e);
    }
    // row of lane l to base + row_l * pitch (bytes); row_l < 0: not stored;
    // `valid` bytes of the row's CH * 16
    __device__ void flush(uint8_t *base, long long pitch, int row, int valid) const {
        __syncwarp();
        const int c = lane % CH;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const int rr = (32 / CH) * k + lane / CH;
            const int o = __shfl_sync(0xffffffffu, row, rr);
            if (o >= 0 && 16 * c < valid)
                *reinterpret_cast<uint4 *>(base + o * pitch + 16 * c) = *reinterpret_cast<const uint4 *>(patch + at(rr, c));
        }
        __syncwarp();
    }
};

template <bool GLU, bool FP8, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
    gmm_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw0,
               const __grid_constant__ CUtensorMap tw1, const GmmArgs a, const Plan p) {
    constexpr bool PAIR = MODE == kPair, SPLIT = MODE == kSplit;
    constexpr int kOutCols = GLU ? 128 : 256;      // output columns of a tile
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t s_tmem;
    __shared__ Groups s_g;
    __shared__ uint32_t s_amax[GLU ? 4 * kLanes : 1];
    // staged products of token and weight scales: [slot][block][half, or gate / up][row]
    __shared__ float s_scale[FP8 ? kSlots * kGroup * 2 * kLanes : 1];
    __shared__ uint64_t sc_full[kSlots], sc_empty[kSlots];
    // with a tile's first slot: the tile, its rows' output rows (-1: none) and their factors
    __shared__ int4 s_tile[kSlots];
    __shared__ int s_row[kSlots][kLanes];
    __shared__ float s_rs[GLU ? 1 : kSlots][kLanes];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int bm = PAIR ? kLanes : p.bm, stages = p.stages;
    const int abytes = bm * 128, stage_bytes = abytes + (PAIR ? 128 : 256) * 128;
    // rank in the cluster; a pair's leader (rank 0) owns the barriers its MMAs wait on
    const int S = PAIR ? 2 : SPLIT ? p.split : 1;
    const int rank = PAIR || SPLIT ? (int)(blockIdx.x % S) : 0;
    const int first = blockIdx.x / S, step = gridDim.x / S;
    if (tid == 0) {
        for (int i = 0; i < stages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], (PAIR ? 2 : 1) * kEpiWarps);
        }
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&sc_full[i], 2);
            mbar_init(&sc_empty[i], kEpiWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    // warp 0 uses `full` before the CTA's barrier (the early weights below), by
    // an elected lane that need not be the one that initialised it
    __syncwarp();
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem)),
                         "r"(512)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem)),
                         "r"(512)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
        }
    }
    const int ntiles = (a.N + kOutCols - 1) / kOutCols;
    const int tile_rows = PAIR ? 2 * kLanes : bm;
    const int kb0 = SPLIT ? (int)((long long)a.KB * rank / S) : 0;
    const int kb1 = SPLIT ? (int)((long long)a.KB * (rank + 1) / S) : a.KB;
    Waiter wait{a.err};
    // A stage's weights: 256 rows, in the order of the accumulator's columns;
    // a pair's CTA loads the 128 of its rank. Gate/up: a half is 64 gate rows,
    // then the same 64 up rows.
    auto load_weights = [&](uint32_t dst, int kb, int wrow, uint64_t *bar) {
        if (PAIR && GLU) {
            tma_load_2d_pair(dst, &tw0, kb * 128, wrow + 64 * rank, bar);
            tma_load_2d_pair(dst + 8192, &tw1, kb * 128, wrow + 64 * rank, bar);
        } else if (PAIR) {
            tma_load_2d_pair(dst, &tw0, kb * 128, wrow + 128 * rank, bar);
        } else if (GLU) {
            for (int h = 0; h < 2; ++h) {
                tma_load_2d(dst + h * 16384, &tw0, kb * 128, wrow + 64 * h, bar);
                tma_load_2d(dst + h * 16384 + 8192, &tw1, kb * 128, wrow + 64 * h, bar);
            }
        } else {
            tma_load_2d(dst, &tw0, kb * 128, wrow, bar);
        }
    };
    // A dense product's weights do not depend on the kernel before this one:
    // the first stages' weights are on their way before its result is waited
    // for.
    int early = 0;
    if (!PAIR && p.weights_first && warp == 0) {
        if (first < ((a.P + bm - 1) / bm) * ntiles) early = min(stages, kb1 - kb0);
        if (elect_one()) {
            for (int s = 0; s < early; ++s) {
                arrive_expect_tx(&full[s], stage_bytes);
                load_weights(sbase + s * stage_bytes + abytes, kb0 + s, (first % ntiles) * kOutCols, &full[s]);
            }
        }
        __syncwarp();
    }
    pdl_wait();
    pdl_trigger();
    if (a.off && warp == 0) build_groups(a, s_g, tile_rows);
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_arrive_wait();                // the peer's barriers and accumulators exist
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const int tiles = (a.off ? s_g.pre[a.E] : (a.P + tile_rows - 1) / tile_rows) * ntiles;
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kCtlRegs));
        if (warp == 0) {
            // ---- TMA producer
            int s = 0;
            uint32_t phase = 1;                     // an empty stage's first wait passes
            for (int tile = first; tile < tiles; tile += step) {
                const Tile t = locate(a, s_g, tile, ntiles, tile_rows);
                const int wrow = t.e * a.N + t.nt * kOutCols;
                const int row0 = t.row0 + (PAIR ? kLanes * rank : 0);
                for (int kb = kb0; kb < kb1; ++kb) {
                    const uint32_t st = sbase + s * stage_bytes;
                    wait(&empty[s], phase);
                    if (elect_one()) {
                        if (PAIR) {
                            // the leader's barrier counts both CTAs' bytes
                            if (rank == 0) arrive_expect_tx(&full[s], 2 * stage_bytes);
                            tma_load_2d_pair(st, &tx, kb * 128, row0, &full[s]);
                            load_weights(st + abytes, kb, wrow, &full[s]);
                        } else {
                            if (early <= 0) {
                                arrive_expect_tx(&full[s], stage_bytes);
                                load_weights(st + abytes, kb, wrow, &full[s]);
                            }
                            tma_load_2d(st, &tx, kb * 128, row0, &full[s]);
                        }
                    }
                    __syncwarp();
                    --early;
                    if (++s == stages) {
                        s = 0;
                        phase ^= 1;
                    }
                }
            }
            // every stage released: no commit is on its way when the CTA leaves
            for (int i = 0; i < stages; ++i) {
                wait(&empty[s], phase);
                if (++s == stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        } else if (warp == 1 && !(PAIR && rank)) {
            // ---- MMA issuer: the sum of one scale block (e4m3) or of a tile
            // (bf16) at a time. (In two halves of 128 columns, so that four
            // smaller buffers hide the epilogue's answer, the MMAs themselves
            // took 1.25 times as long.)
            constexpr uint32_t idesc = idesc_of(FP8, PAIR ? 256 : 128, kAccCols);
            int s = 0;
            uint32_t phase = 0, u = 0, uphase = 1;
            for (int tile = first; tile < tiles; tile += step) {
                for (int kb = kb0; kb < kb1; ++kb) {
                    const bool fresh = FP8 || kb == kb0, last = FP8 || kb == kb1 - 1;
                    const uint32_t st = sbase + s * stage_bytes, d = tmem + u * kAccCols;
                    wait(&full[s], phase);
                    if (fresh) wait(&acc_empty[u], uphase);
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            mma_ss<FP8, PAIR>(d, sw128_desc(st + 32 * q), sw128_desc(st + abytes + 32 * q), idesc,
                                              !fresh || q > 0);
                        commit<PAIR>(&empty[s]);
                        if (last) commit<PAIR>(&acc_full[u]);
                    }
                    __syncwarp();
                    if (++s == stages) {
                        s = 0;
                        phase ^= 1;
                    }
                    if (last) {
                        u ^= 1;
                        if (u == 0) uphase ^= 1;
                    }
                }
            }
        }
        else if (warp >= 2) {
            // ---- stagers: warps 2 and 3 find the tiles for the epilogue, a few
            // blocks ahead of it, with their output rows and (e4m3) the products
            // of the blocks' scales. (With the tiles found and the output rows
            // looked up by the epilogue a tile of six blocks took 11200 cycles,
            // so 10400. The scales' loads in the epilogue's own loop would take
            // a dozen of its registers and, with six scoreboards a warp, make
            // it wait for the youngest.)
            const int l = tid - 64;                 // rows l and l + 64
            const int NB = (a.N + kScaleBlock - 1) / kScaleBlock, units = FP8 ? kb1 - kb0 : 1;
            int slot = 0;
            uint32_t phase = 1;
            for (int tile = first; tile < tiles; tile += step) {
                const Tile t = locate(a, s_g, tile, ntiles, tile_rows);
                const int nb = GLU ? t.nt : 2 * t.nt;
                const int r = t.row0 + (PAIR ? kLanes * rank : 0) + l, r1 = r + 64;
                const bool live0 = l < bm && r < t.end, live1 = l + 64 < bm && r1 < t.end;
                int o0 = live0 ? r : -1, o1 = live1 ? r1 : -1;
                float rs0 = 1.0f, rs1 = 1.0f;
                if (!GLU) {
                    if (a.map && live0) o0 = __ldg(a.map + r);
                    if (a.map && live1) o1 = __ldg(a.map + r1);
                    if (a.row_scale && live0) rs0 = __ldg(a.row_scale + o0);
                    if (a.row_scale && live1) rs1 = __ldg(a.row_scale + o1);
                }
                const float *w0 = nullptr, *w1 = nullptr, *x0 = nullptr, *x1 = nullptr;
                if (FP8) {
                    w0 = a.sw0 + ((size_t)t.e * NB + nb) * a.KB + kb0;
                    w1 = GLU ? a.sw1 + ((size_t)t.e * NB + nb) * a.KB + kb0 : w0 + (nb + 1 < NB ? a.KB : 0);
                    x0 = a.sx + (size_t)kb0 * a.P + min(r, a.P - 1);
                    x1 = a.sx + (size_t)kb0 * a.P + min(r1, a.P - 1);
                }
                for (int i0 = 0; i0 < units; i0 += kGroup) {
                    float v[kGroup][4];
                    if (FP8)
#pragma unroll
                        for (int z = 0; z < kGroup; ++z) {
                            const int i = min(i0 + z, units - 1);
                            v[z][0] = __ldg(x0 + (size_t)i * a.P);
                            v[z][1] = __ldg(x1 + (size_t)i * a.P);
                            v[z][2] = __ldg(w0 + i);
                            v[z][3] = __ldg(w1 + i);
                        }
                    wait(&sc_empty[slot], phase);
                    if (FP8) {
                        float *to = s_scale + slot * kGroup * 2 * kLanes + l;
#pragma unroll
                        for (int z = 0; z < kGroup; ++z, to += 2 * kLanes) {
                            to[0] = v[z][0] * v[z][2];
                            to[64] = v[z][1] * v[z][2];
                            to[kLanes] = v[z][0] * v[z][3];
                            to[kLanes + 64] = v[z][1] * v[z][3];
                        }
                    }
                    if (i0 == 0) {
                        if (l == 0) s_tile[slot] = make_int4(t.e, t.row0, t.end, t.nt);
                        s_row[slot][l] = o0;
                        s_row[slot][l + 64] = o1;
                        if (!GLU) {
                            s_rs[slot][l] = rs0;
                            s_rs[slot][l + 64] = rs1;
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[slot]);
                    if (++slot == kSlots) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
            }
        }
        __syncwarp();
        if (SPLIT) {
            cluster_arrive_wait();
            cluster_arrive_wait();
        }
    } else {
        // ---- epilogue: thread = one token, a quarter of the tile's columns:
        // 64 weight rows, or (gate/up) 32 of each matrix
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kEpiRegs));
        const int q = warp & 3, part = (warp - 4) >> 2, half = part >> 1, row = 32 * q + lane;
        const bool busy = 32 * q < bm;              // lanes that hold token rows at all
        uint8_t *const patch = smem_raw + (sbase - smem_u32(smem_raw)) + kRingBytes + (warp - 4) * kPatch;
        // its accumulator columns: two pieces of 32
        const int col0 = GLU ? 128 * half + 32 * (part & 1) : 64 * part, col1 = col0 + (GLU ? 64 : 32);
        const uint32_t tq = tmem + ((uint32_t)(32 * q) << 16);
        // the accumulators' barriers for the MMA issuer, a pair's in its leader
        const uint32_t done0 = map_cluster(smem_u32(&acc_empty[0]), 0);
        uint32_t un = 0, sphase = 0;
        int slot = 0;
        bool ready = false;
        for (int tile = first; tile < tiles; tile += step) {
            Tile t{};
            int orow = -1;                          // its output row
            float rs = 1.0f;
            uint64_t acc[32];                       // 64 float32 sums
            if (FP8) {
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[j] = 0;
            }
            const int units = FP8 ? kb1 - kb0 : 1;
            for (int i0 = 0; i0 < units; i0 += kGroup) {
                wait(&sc_full[slot], sphase);
                if (i0 == 0) {
                    const int4 f = s_tile[slot];
                    t = Tile{f.x, f.y, f.z, f.w};
                    orow = s_row[slot][row];
                    if (!GLU) rs = s_rs[GLU ? 0 : slot][row];
                }
                const float *sc = s_scale + (FP8 ? slot * kGroup * 2 * kLanes + row : 0);
#pragma unroll 1
                for (int z = 0; z < kGroup; ++z) {
                    if (i0 + z >= units) break;
                    uint64_t s0 = 0, s1 = 0;
                    if (FP8) {
                        const uint32_t b = __float_as_uint(sc[(2 * z + (GLU ? 0 : half)) * kLanes]);
                        s0 = s1 = pack2(b, b);
                        if (GLU) {
                            const uint32_t c = __float_as_uint(sc[(2 * z + 1) * kLanes]);
                            s1 = pack2(c, c);
                        }
                    }
                    const uint32_t u = un & 1, td = tq + u * kAccCols;
                    wait(&acc_full[u], (un >> 1) & 1, ready);
                    ++un;
                    tc_fence_after();
                    uint32_t dv[16];
                    auto add = [&](int c) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint64_t v = pack2(dv[2 * j], dv[2 * j + 1]);
                            if (FP8) fma2(acc[8 * c + j], v, c >= 2 ? s1 : s0);
                            else acc[8 * c + j] = v;
                        }
                    };
                    if (busy) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            tmem_ld16(td + (c >= 2 ? col1 : col0) + 16 * (c & 1), dv);
                            tmem_wait_ld();
                            if (c < 3) add(c);
                        }
                    }
                    // (every lane's tcgen05.ld is done: the wait is the warp's)
                    tc_fence_before();
                    if (lane == 0) {
                        if (PAIR) arrive_at(done0 + 8 * u);
                        else mbar_arrive(&acc_empty[u]);
                    }
                    ready = test_bar(&acc_full[un & 1], (un >> 1) & 1);
                    if (busy) add(3);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sc_empty[slot]);
                if (++slot == kSlots) {
                    slot = 0;
                    sphase ^= 1;
                }
            }
            const int n0 = t.nt * kOutCols + part * (kOutCols / 4);   // its first output column
            if (SPLIT) {
                // the ring is idle: this CTA's sums, [row][column]. At a pitch
                // of 65 x 16 bytes neither the lanes' 16-byte pieces of their
                // rows nor a row's 16-byte pieces meet in a bank.
                float *sums = reinterpret_cast<float *>(smem_raw + (sbase - smem_u32(smem_raw)));
                if (row < bm) {
                    float *to = sums + row * kPartPitch;
#pragma unroll
                    for (int j = 0; j < 32; j += 2)
                        *reinterpret_cast<ulonglong2 *>(to + (j < 16 ? col0 : col1 - 32) + 2 * j) =
                            make_ulonglong2(acc[j], acc[j + 1]);
                }
            } else if (GLU) {
                // 32 activations of the token's group of 128; the largest of
                // all 128 with the other three warps of these lanes
                uint32_t m = 0, v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    v[j] = glu_pair(lo2(acc[j]), hi2(acc[j]), lo2(acc[16 + j]), hi2(acc[16 + j]), a.act);
                    if (n0 + 2 * j < a.N) m = __vmaxu2(m, v[j] & 0x7FFF7FFFu);
                }
                s_amax[part * kLanes + row] = max(m & 0xFFFFu, m >> 16);
                bar_sync(1, 32 * kEpiWarps);
                m = max(max(s_amax[row], s_amax[kLanes + row]), max(s_amax[2 * kLanes + row], s_amax[3 * kLanes + row]));
                bar_sync(1, 32 * kEpiWarps);        // read before the next tile's
                const QScale qs = qscale(m);
                const RowStore<2> rows{patch, lane};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t w[4];
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const uint32_t x0 = v[8 * c + 2 * z], x1 = v[8 * c + 2 * z + 1];
                        w[z] = cvt_e4m3x2(quotient(bf_lo(x0), qs), quotient(bf_hi(x0), qs)) |
                               (cvt_e4m3x2(quotient(bf_lo(x1), qs), quotient(bf_hi(x1), qs)) << 16);
                    }
                    rows.put(c, w[0], w[1], w[2], w[3]);
                }
                rows.flush(a.q_out + n0, a.N, orow, a.N - n0);
                if (part == 0 && orow >= 0) a.s_out[(size_t)t.nt * a.P + orow] = qs.s;
            } else {
                const RowStore<4> rows{patch, lane};
                if (a.out_f32) {
                    uint8_t *y = reinterpret_cast<uint8_t *>(static_cast<float *>(a.out) + n0);
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint64_t x0 = acc[8 * h + 2 * c], x1 = acc[8 * h + 2 * c + 1];
                            rows.put(c, (uint32_t)x0, (uint32_t)(x0 >> 32), (uint32_t)x1, (uint32_t)(x1 >> 32));
                        }
                        rows.flush(y + 64 * h, 4 * a.out_stride, orow, 4 * (a.N - n0) - 64 * h);
                    }
                } else {
                    uint8_t *y = reinterpret_cast<uint8_t *>(static_cast<uint16_t *>(a.out) + n0);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t w[4];
#pragma unroll
                            for (int z = 0; z < 4; ++z) {
                                const uint64_t x = acc[16 * h + 4 * c + z];
                                w[z] = cvt_bf16x2(lo2(x), hi2(x));
                                if (a.row_scale) w[z] = cvt_bf16x2(bf_lo(w[z]) * rs, bf_hi(w[z]) * rs);
                            }
                            rows.put(c, w[0], w[1], w[2], w[3]);
                        }
                        rows.flush(y + 64 * h, 2 * a.out_stride, orow, 2 * (a.N - n0) - 64 * h);
                    }
                }
            }
        }
        __syncwarp();
        if (SPLIT) {
            // Each CTA adds up and stores its share of the tile: a warp takes a
            // row's 128 activations (gate/up) or 128 columns of a row, a lane
            // four of them.
            cluster_arrive_wait();
            if (first < tiles) {
                const Tile t = locate(a, s_g, first, ntiles, tile_rows);
                const int np = min(bm, t.end - t.row0);
                uint32_t peer[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) peer[c] = map_cluster(sbase, min(c, S - 1));
                // the cluster's sums from N places, every load in flight before
                // the first is used
                auto sums = [&](auto &v, const auto &at) {
                    constexpr int N = sizeof(v) / sizeof(float4);
#pragma unroll
                    for (int n = 0; n < N; ++n) v[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float4 x[N][4];
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (4 * h + c < S)
#pragma unroll
                                for (int n = 0; n < N; ++n) x[n][c] = ld_cluster4(peer[4 * h + c] + 4 * at(n));
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (4 * h + c < S)
#pragma unroll
                                for (int n = 0; n < N; ++n) {
                                    v[n].x += x[n][c].x;
                                    v[n].y += x[n][c].y;
                                    v[n].z += x[n][c].z;
                                    v[n].w += x[n][c].w;
                                }
                    }
                };
                if (GLU) {
                    const int c = 4 * lane, n = t.nt * 128 + c;
                    for (int u = (warp - 4) * S + rank; u < np; u += kEpiWarps * S) {
                        float4 g[2];             // gate and up of this lane's four columns
                        sums(g, [&](int i) { return u * kPartPitch + (c >> 6) * 128 + (c & 63) + 64 * i; });
                        const uint32_t y0 = glu_pair(g[0].x, g[0].y, g[1].x, g[1].y, a.act);
                        const uint32_t y1 = glu_pair(g[0].z, g[0].w, g[1].z, g[1].w, a.act);
                        uint32_t m = n < a.N ? __vmaxu2(y0 & 0x7FFF7FFFu, y1 & 0x7FFF7FFFu) : 0u;
                        m = __reduce_max_sync(0xffffffffu, max(m & 0xFFFFu, m >> 16));
                        const QScale qs = qscale(m);
                        const size_t r = (size_t)(t.row0 + u);
                        if (n < a.N)
                            *reinterpret_cast<uint32_t *>(a.q_out + r * a.N + n) =
                                cvt_e4m3x2(quotient(bf_lo(y0), qs), quotient(bf_hi(y0), qs)) |
                                (cvt_e4m3x2(quotient(bf_lo(y1), qs), quotient(bf_hi(y1), qs)) << 16);
                        if (lane == 0) a.s_out[(size_t)t.nt * a.P + r] = qs.s;
                    }
                } else {
                    // two steps at a time
                    constexpr int kSteps = 2;
                    const int stride = kEpiWarps * S, total = 2 * np;
                    for (int u0 = (warp - 4) * S + rank; u0 < total; u0 += kSteps * stride) {
                        float4 v[kSteps];
                        sums(v, [&](int i) {
                            const int u = min(u0 + i * stride, total - 1);
                            return (u >> 1) * kPartPitch + (u & 1) * 128 + 4 * lane;
                        });
#pragma unroll
                        for (int k = 0; k < kSteps; ++k) {
                            const int u = u0 + k * stride, n = t.nt * 256 + (u & 1) * 128 + 4 * lane;
                            if (u >= total || n >= a.N) continue;
                            const int r = t.row0 + (u >> 1), o = a.map ? a.map[r] : r;
                            if (a.out_f32) {
                                *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + o * a.out_stride + n) = v[k];
                            } else {
                                uint32_t y0 = cvt_bf16x2(v[k].x, v[k].y), y1 = cvt_bf16x2(v[k].z, v[k].w);
                                if (a.row_scale) {
                                    const float rs = a.row_scale[o];
                                    y0 = cvt_bf16x2(bf_lo(y0) * rs, bf_hi(y0) * rs);
                                    y1 = cvt_bf16x2(bf_lo(y1) * rs, bf_hi(y1) * rs);
                                }
                                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + o * a.out_stride + n) =
                                    make_uint2(y0, y1);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            cluster_arrive_wait();                      // the others have read this CTA's sums
        }
    }
    tc_fence_before();
    __syncthreads();
    // neither CTA of a pair leaves while the other may signal its barriers
    if (PAIR) cluster_arrive_wait();
    if (warp == 1) {
        tc_fence_after();
        if (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ------------------------------------------ few tokens: weights on the lanes

// Groups of a few tokens leave most of a 128-token tile's lanes empty, and its
// two wide accumulators leave the tensor core waiting on the epilogue of a
// tile of a few blocks. Here 128 weight rows take the lanes and 32 tokens are
// the MMA's N: eight accumulators fit, all the lanes carry results, and the
// two epilogue warpgroups take alternate tiles, so that one stores while the
// other adds up. Each has its own accumulators and scale slots: a barrier's
// parity tells two phases apart, so whoever waits on one has to see them all.
// What bounds the kernel is the weights' stream from HBM.
constexpr int kTok = 32;
constexpr int kUnits = 4;                      // accumulators of a warpgroup
constexpr int kSmallSlots = 2;                 // slots of staged scales of a warpgroup
constexpr int kSmallThreads = 384;
constexpr int kSmallRing = 184 * 1024;
constexpr size_t kSmallSmem = 1024 + kSmallRing;

template <int NMAT, bool FP8>
__global__ void __launch_bounds__(kSmallThreads, 1)
    gmm_small_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw0,
                     const __grid_constant__ CUtensorMap tw1, const GmmArgs a, const Plan p) {
    constexpr bool GLU = NMAT == 2;
    constexpr int kStageBytes = NMAT * 16384 + kTok * 128, kStages = kSmallRing / kStageBytes;
    constexpr int kCols = NMAT * kTok, kAlloc = 2 * kUnits * kCols;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[kStages], empty[kStages], acc_full[2][kUnits], acc_empty[2][kUnits];
    __shared__ uint64_t sc_full[2][kSmallSlots], sc_empty[2][kSmallSlots];
    __shared__ uint32_t s_tmem;
    __shared__ Groups s_g;
    // products of token and weight scales: [warpgroup][slot][block][matrix][token]
    __shared__ __align__(16) float s_scale[FP8 ? 2 * kSmallSlots * kGroup * kCols : 4];
    __shared__ __align__(16) uint16_t s_out[2][kTok * kLanes];      // [warpgroup][token][weight row]
    __shared__ uint32_t s_amax[GLU ? 2 : 1][4][kTok];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2 * kUnits; ++i) {
            mbar_init(&acc_full[i / kUnits][i % kUnits], 1);
            mbar_init(&acc_empty[i / kUnits][i % kUnits], 4);
        }
        for (int i = 0; i < 2 * kSmallSlots; ++i) {
            mbar_init(&sc_full[i / kSmallSlots][i % kSmallSlots], NMAT);
            mbar_init(&sc_empty[i / kSmallSlots][i % kSmallSlots], 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem)),
                     "r"(kAlloc)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    pdl_wait();
    pdl_trigger();
    if (a.off && warp == 0) build_groups(a, s_g, kTok);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const int ntiles = (a.N + kLanes - 1) / kLanes;
    const int tiles = (a.off ? s_g.pre[a.E] : (a.P + kTok - 1) / kTok) * ntiles;
    const int units = FP8 ? a.KB : 1;              // accumulators of a tile
    Waiter wait{a.err};
    if (warp == 0) {
        // ---- TMA producer
        int s = 0;
        uint32_t phase = 1;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            const Tile t = locate(a, s_g, tile, ntiles, kTok);
            const int wrow = t.e * a.N + t.nt * kLanes;
            for (int kb = 0; kb < a.KB; ++kb) {
                const uint32_t st = sbase + s * kStageBytes;
                wait(&empty[s], phase);
                if (elect_one()) {
                    arrive_expect_tx(&full[s], kStageBytes);
                    tma_load_2d(st, &tw0, kb * 128, wrow, &full[s]);
                    if (GLU) tma_load_2d(st + 16384, &tw1, kb * 128, wrow, &full[s]);
                    tma_load_2d(st + NMAT * 16384, &tx, kb * 128, t.row0, &full[s]);
                }
                __syncwarp();
                if (++s == kStages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        // every stage released: no commit is on its way when the CTA leaves
        for (int i = 0; i < kStages; ++i) {
            wait(&empty[s], phase);
            if (++s == kStages) {
                s = 0;
                phase ^= 1;
            }
        }
    } else if (warp == 1) {
        // ---- MMA issuer
        constexpr uint32_t idesc = idesc_of(FP8, kLanes, kTok);
        int s = 0, wg = 0;
        uint32_t phase = 0, un[2] = {0, 0};        // accumulators handed to each warpgroup
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, wg ^= 1) {
            uint32_t c = wg ? un[1] : un[0];
            for (int kb = 0; kb < a.KB; ++kb) {
                const bool fresh = FP8 || kb == 0, last = FP8 || kb == a.KB - 1;
                const uint32_t u = c % kUnits, d = tmem + (wg * kUnits + u) * kCols;
                const uint32_t st = sbase + s * kStageBytes;
                wait(&full[s], phase);
                if (fresh) wait(&acc_empty[wg][u], ((c / kUnits) & 1) ^ 1);
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int m = 0; m < NMAT; ++m)
                            mma_ss<FP8, false>(d + m * kTok, sw128_desc(st + m * 16384 + 32 * q),
                                               sw128_desc(st + NMAT * 16384 + 32 * q), idesc, !fresh || q > 0);
                    tc_commit(&empty[s]);
                    if (last) tc_commit(&acc_full[wg][u]);
                }
                __syncwarp();
                if (++s == kStages) {
                    s = 0;
                    phase ^= 1;
                }
                if (last) ++c;
            }
            if (wg) un[1] = c;
            else un[0] = c;
        }
    } else if (warp < 4) {
        // ---- scales: a warp a matrix, a lane a token
        if (FP8 && warp - 2 < NMAT) {
            const int m = warp - 2;
            int wg = 0;
            uint32_t gg[2] = {0, 0};               // slots filled for each warpgroup
            for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, wg ^= 1) {
                uint32_t g = wg ? gg[1] : gg[0];
                const Tile t = locate(a, s_g, tile, ntiles, kTok);
                const float *w = (m ? a.sw1 : a.sw0) + ((size_t)t.e * ntiles + t.nt) * a.KB;
                const float *x = a.sx + min(t.row0 + lane, a.P - 1);
                for (int i0 = 0; i0 < units; i0 += kGroup, ++g) {
                    const uint32_t slot = g % kSmallSlots;
                    float v[kGroup], f[kGroup];
#pragma unroll
                    for (int z = 0; z < kGroup; ++z) {
                        const int i = min(i0 + z, units - 1);
                        v[z] = __ldg(x + (size_t)i * a.P);
                        f[z] = __ldg(w + i);
                    }
                    wait(&sc_empty[wg][slot], ((g / kSmallSlots) & 1) ^ 1);
#pragma unroll
                    for (int z = 0; z < kGroup; ++z)
                        s_scale[(((wg * kSmallSlots + slot) * kGroup + z) * NMAT + m) * kTok + lane] = v[z] * f[z];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[wg][slot]);
                }
                if (wg) gg[1] = g;
                else gg[0] = g;
            }
        }
        __syncwarp();
    } else {
        // ---- epilogue: thread = one weight row; the warpgroups take alternate tiles
        const int wg = (warp - 4) >> 2, q = warp & 3, row = 32 * q + lane;
        const uint32_t tq = tmem + ((uint32_t)(32 * q) << 16) + wg * kUnits * kCols;
        uint32_t un = 0, gg = 0;                    // accumulators and scale slots this warpgroup has read
        uint16_t *const so = s_out[wg];
        for (int tile = blockIdx.x + wg * gridDim.x; tile < tiles; tile += 2 * gridDim.x) {
            const Tile t = locate(a, s_g, tile, ntiles, kTok);
            const int np = min(kTok, t.end - t.row0), n0 = t.nt * kLanes, n = n0 + row;
            // lane's token: its output row
            int orow = -1;
            if (lane < np) orow = !GLU && a.map ? ld_here(a.map + t.row0 + lane) : t.row0 + lane;
            uint64_t acc[NMAT][kTok / 2];
#pragma unroll
            for (int m = 0; m < NMAT; ++m)
#pragma unroll
                for (int j = 0; j < kTok / 2; ++j) acc[m][j] = 0;
            for (int i0 = 0; i0 < units; i0 += kGroup, ++gg) {
                const uint32_t slot = gg % kSmallSlots;
                if (FP8) wait(&sc_full[wg][slot], (gg / kSmallSlots) & 1);
                for (int i = i0; i < min(i0 + kGroup, units); ++i, ++un) {
                    const uint32_t u = un % kUnits;
                    wait(&acc_full[wg][u], (un / kUnits) & 1);
                    tc_fence_after();
                    uint32_t dv[NMAT][32];
#pragma unroll
                    for (int m = 0; m < NMAT; ++m) tmem_ld32(tq + u * kCols + m * kTok, dv[m]);
                    tmem_wait_ld();
                    tc_fence_before();
                    if (lane == 0) mbar_arrive(&acc_empty[wg][u]);
#pragma unroll
                    for (int m = 0; m < NMAT; ++m) {
                        const ulonglong2 *sc = reinterpret_cast<const ulonglong2 *>(
                            s_scale + (((wg * kSmallSlots + slot) * kGroup + i - i0) * NMAT + m) * kTok);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if (FP8) {
                                const ulonglong2 s = sc[j];
                                fma2(acc[m][2 * j], pack2(dv[m][4 * j], dv[m][4 * j + 1]), s.x);
                                fma2(acc[m][2 * j + 1], pack2(dv[m][4 * j + 2], dv[m][4 * j + 3]), s.y);
                            } else {
                                acc[m][2 * j] = pack2(dv[m][4 * j], dv[m][4 * j + 1]);
                                acc[m][2 * j + 1] = pack2(dv[m][4 * j + 2], dv[m][4 * j + 3]);
                            }
                        }
                    }
                }
                if (FP8) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_empty[wg][slot]);
                }
            }
            if (!GLU && a.out_f32) {
#pragma unroll
                for (int j = 0; j < kTok; ++j) {
                    const int o = __shfl_sync(0xffffffffu, orow, j);
                    const float v = j & 1 ? hi2(acc[0][j >> 1]) : lo2(acc[0][j >> 1]);
                    if (o >= 0 && n < a.N) static_cast<float *>(a.out)[o * a.out_stride + n] = v;
                }
                continue;
            }
            const float rs = !GLU && a.row_scale && orow >= 0 ? a.row_scale[orow] : 1.0f;
            uint32_t most = 0;
#pragma unroll
            for (int j = 0; j < kTok / 2; ++j) {
                uint32_t w;
                if (GLU) {
                    w = glu_pair(lo2(acc[0][j]), hi2(acc[0][j]), lo2(acc[NMAT - 1][j]), hi2(acc[NMAT - 1][j]), a.act);
                    const uint32_t m = n < a.N ? w & 0x7FFF7FFFu : 0u;
                    const uint32_t m0 = __reduce_max_sync(0xffffffffu, m & 0xFFFFu);
                    const uint32_t m1 = __reduce_max_sync(0xffffffffu, m >> 16);
                    if (lane == 2 * j) most = m0;
                    if (lane == 2 * j + 1) most = m1;
                } else {
                    w = cvt_bf16x2(lo2(acc[0][j]), hi2(acc[0][j]));
                    if (a.row_scale)
                        w = cvt_bf16x2(bf_lo(w) * __shfl_sync(0xffffffffu, rs, 2 * j),
                                       bf_hi(w) * __shfl_sync(0xffffffffu, rs, 2 * j + 1));
                }
                so[2 * j * kLanes + row] = (uint16_t)w;
                so[(2 * j + 1) * kLanes + row] = (uint16_t)(w >> 16);
            }
            if (GLU) s_amax[GLU ? wg : 0][q][lane] = most;
            bar_sync(1 + wg, 128);
            // eight tokens a warp, sixteen lanes a token's 128 values
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int tok = 8 * q + 2 * k + (lane >> 4), c = 8 * (lane & 15);
                const int o = __shfl_sync(0xffffffffu, orow, tok);
                if (o < 0 || n0 + c >= a.N) continue;
                const uint4 v = *reinterpret_cast<const uint4 *>(so + tok * kLanes + c);
                if (GLU) {
                    const uint32_t *am = &s_amax[GLU ? wg : 0][0][tok];
                    const QScale qs = qscale(max(max(am[0], am[kTok]), max(am[2 * kTok], am[3 * kTok])));
                    const uint32_t lo = cvt_e4m3x2(quotient(bf_lo(v.x), qs), quotient(bf_hi(v.x), qs)) |
                                        (cvt_e4m3x2(quotient(bf_lo(v.y), qs), quotient(bf_hi(v.y), qs)) << 16);
                    const uint32_t hi = cvt_e4m3x2(quotient(bf_lo(v.z), qs), quotient(bf_hi(v.z), qs)) |
                                        (cvt_e4m3x2(quotient(bf_lo(v.w), qs), quotient(bf_hi(v.w), qs)) << 16);
                    *reinterpret_cast<uint2 *>(a.q_out + (size_t)o * a.N + n0 + c) = make_uint2(lo, hi);
                    if (c == 0) a.s_out[(size_t)t.nt * a.P + o] = qs.s;
                } else {
                    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + o * a.out_stride + n0 + c) = v;
                }
            }
            bar_sync(1 + wg, 128);                  // read before this warpgroup's next tile
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kAlloc) : "memory");
    }
}

// ---------------------------------------------------------------- host

// The epilogue warps take registers that the block's other warps gave up. A
// build that launches with fewer than the two shares' sum would wait for them
// without end: refused (looked up once per kernel and device).
static vqmoe_status check_registers(const void *fn) {
    static std::mutex mu;
    static std::map<std::pair<const void *, int>, int> regs;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("gmm_kernel");
    std::lock_guard<std::mutex> lock(mu);
    int &n = regs[{fn, dev}];
    if (!n) {
        cudaFuncAttributes at{};
        if (cudaFuncGetAttributes(&at, fn) != cudaSuccess) return check_launch("gmm_kernel");
        n = at.numRegs;
    }
    if (n * kThreads < 128 * kCtlRegs + 32 * kEpiWarps * kEpiRegs)
        return set_error(VQMOE_LAUNCH_FAILED, "gmm_kernel: built with %d registers a thread", n);
    return VQMOE_OK;
}

static bool byte_map(CUtensorMap *m, const void *base, size_t rows, size_t row_bytes, size_t pitch, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)row_bytes, (cuuint64_t)rows};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    return encode_tma_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, dims, pitch, box) == CUDA_SUCCESS;
}

// How many clusters of `size` CTAs of the kernel run at a time (each CTA takes
// an SM, and a cluster stays inside one GPC), looked up once per device: every
// kSplit kernel asks for the same threads, registers and dynamic shared memory,
// one CTA an SM, so the first one's answer is the others' too.
static int max_clusters(const void *fn, int size) {
    static std::atomic<int> known[64][9];          // the number + 1
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (const int n = known[dev][size].load(std::memory_order_relaxed)) return n - 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (ensure_dynamic_smem(fn, kSmem, "gmm_kernel") != VQMOE_OK ||
        cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    known[dev][size].store(n + 1, std::memory_order_relaxed);
    return n;
}

template <int MODE>
static const void *kernel_of(bool glu, bool fp8) {
    return glu   ? reinterpret_cast<const void *>(&gmm_kernel<true, true, MODE>)
           : fp8 ? reinterpret_cast<const void *>(&gmm_kernel<false, true, MODE>)
                 : reinterpret_cast<const void *>(&gmm_kernel<false, false, MODE>);
}

}  // namespace gm

vqmoe_status launch_gmm(const void *x, size_t x_pitch, const void *w0, const void *w1, size_t row_bytes, bool fp8,
                        const GmmArgs &a, cudaStream_t stream, bool pdl_weights) {
    using namespace gm;
    const bool glu = w1 != nullptr;
    if (a.P <= 0) return VQMOE_OK;
    if (a.E <= 0 || a.E > kMaxGroups || (!a.off && a.E != 1))
        return set_error(VQMOE_BAD_SHAPE, "grouped product: %d groups (1..%d)", a.E, kMaxGroups);
    if ((long long)a.E * a.N > 0x7FFFFFFFLL - 256 || (long long)a.KB * 128 > 0x7FFFFFFFLL)
        return set_error(VQMOE_BAD_SHAPE, "grouped product: %d groups of %d rows", a.E, a.N);
    const int sms = sm_count();
    // groups that can have rows, and the tiles of `rows` token rows (a bound, with ragged groups)
    const int groups = std::min(a.E, a.P);
    const long long ntiles = (a.N + (glu ? 127 : 255)) / (glu ? 128 : 256);
    auto tiles_of = [&](int rows) {
        return ntiles * (a.off ? std::min<long long>(a.P, a.P / rows + groups) : (a.P + rows - 1) / rows);
    };
    // Which mode: the least estimated time, waves of tiles times their blocks,
    // from measured microseconds of a 128-byte block, a tile's other work and,
    // for a split tile, bringing the sums together (fixed, and by its rows).
    const int small_cols = (int)(((a.N + kLanes - 1) / kLanes + ntiles - 1) / ntiles);   // kSmall's column tiles of one here
    const double unit = fp8 ? 1.0 : 0.8;
    Plan p{};
    int mode = kSingle;
    double best = 1e30;
    auto consider = [&](int m, int bm, int split, double block, double other, int slots) {
        const long long tiles = tiles_of(m == kPair ? 2 * bm : bm) * (m == kSmall ? small_cols : 1);
        const double cost = (double)((tiles + slots - 1) / slots) * ((a.KB + split - 1) / split * block * unit + other);
        if (cost < best) {
            best = cost;
            mode = m;
            p.bm = bm;
            p.split = split;
        }
    };
    if (a.off) {
        // Ragged: the host knows the mean alone, so the tile goes by that.
        // Measured at 128 groups of 768 x 2048 (us; kSmall / kSingle with 64 /
        // with 128 rows / kPair), even groups, then Zipf-distributed ones: mean
        // 4 e4m3 42 / 43 / 44 / 66, 36 / 34 / 35 / 47, bf16 69 / 69 / 73 / 82,
        // 57 / 55 / 56 / 58; mean 16 e4m3 46 / 47 / 48 / 69, 51 / 46 / 48 / 71,
        // bf16 72 / 72 / 75 / 86, 80 / 71 / 74 / 84; mean 32 e4m3 58 / 51 / 51 /
        // 72, 65 / 60 / 51 / 73; mean 256 (128 rows / kPair) e4m3 136 / 141, 146 /
        // 147, bf16 146 / 126, 149 / 135; mean 512 e4m3 247 / 232, bf16 235 / 192.
        // e4m3 gate/up with down: mean 4 124 / 143 / 148 / 203, mean 32 156 / 156 /
        // 162 (gate/up by kSmall, down by 128 rows: 148), mean 48 188 / 167 / 166.
        // The points below are those of the even groups at this one shape: other
        // widths were not measured against each other, and under Zipf the even
        // groups' choice can be behind (e4m3 mean 16: kSmall 51, 64 rows 46).
        const int mean = (a.P + groups - 1) / groups;
        if (mean <= (glu ? 40 : fp8 ? 20 : 6)) consider(kSmall, kTok, 1, glu ? 0.74 : 0.37, 0.7, sms);
        else if (mean <= 24) consider(kSingle, 64, 1, 0.55, 3.0, sms);
        else if (mean < (fp8 ? 640 : 192)) consider(kSingle, 128, 1, 0.6, 3.0, sms);
        else consider(kPair, 128, 1, 0.6, 3.0, sms / 2);
    } else {
        consider(kPair, 128, 1, 0.58, 2.0, sms / 2);
        consider(kSingle, 128, 1, 0.60, 2.0, sms);
        consider(kSingle, 64, 1, 0.55, 2.0, sms);
        consider(kSingle, 32, 1, 0.45, 2.0, sms);
    }
    // Splitting pays while a wave of tiles leaves SMs idle: one wave of clusters
    // then, at least two blocks a CTA. (4096 x 4096 e4m3, one token: 1 x 16
    // CTAs 19.5 us, clusters of 4 11.5, of 6 10.7, of 8, which do not all fit at
    // once, 18.)
    for (int bm = 32; bm <= 128; bm *= 2)
        for (int s = 2; s <= 8 && 2 * s <= a.KB; ++s)
            if (tiles_of(bm) * s <= sms) {
                const int slots = max_clusters(kernel_of<kSplit>(glu, fp8), s);
                if (tiles_of(bm) <= slots)
                    consider(kSplit, bm, s, bm == 32 ? 0.45 : bm == 64 ? 0.5 : 0.55,
                             3.5 + 0.01 * bm + 0.006 * bm * s, slots);
            }
    const int stage = p.bm * 128 + (mode == kPair ? 128 : 256) * 128;
    p.stages = std::min(kMaxStages, kRingBytes / stage);
    const int box = mode == kSmall ? kLanes : glu ? 64 : mode == kPair ? 128 : 256;
    p.weights_first = pdl_weights && !a.off && mode != kPair;
    const int cluster = mode == kPair ? 2 : p.split;
    const long long tiles = std::min<long long>(tiles_of(mode == kPair ? 256 : p.bm) * (mode == kSmall ? small_cols : 1),
                                                1 << 20);
    const int grid = mode == kSplit ? (int)tiles * p.split
                     : mode == kPair ? 2 * (int)std::min<long long>(tiles, sms / 2)
                                     : (int)std::min<long long>(tiles, sms);
    CUtensorMap mx, m0, m1;
    const size_t wrows = (size_t)a.E * a.N;
    if (!byte_map(&mx, x, a.P, row_bytes, x_pitch, p.bm) || !byte_map(&m0, w0, wrows, row_bytes, row_bytes, box) ||
        !byte_map(&m1, glu ? w1 : w0, wrows, row_bytes, row_bytes, box))
        return set_error(VQMOE_LAUNCH_FAILED, "grouped product: tensor map");
    const void *fn = mode == kPair    ? kernel_of<kPair>(glu, fp8)
                     : mode == kSplit ? kernel_of<kSplit>(glu, fp8)
                     : mode == kSmall ? (glu   ? reinterpret_cast<const void *>(&gmm_small_kernel<2, true>)
                                         : fp8 ? reinterpret_cast<const void *>(&gmm_small_kernel<1, true>)
                                               : reinterpret_cast<const void *>(&gmm_small_kernel<1, false>))
                                      : kernel_of<kSingle>(glu, fp8);
    const size_t smem = mode == kSmall ? kSmallSmem : kSmem;
    vqmoe_status s;
    if ((mode != kSmall && (s = check_registers(fn)) != VQMOE_OK) ||
        (s = ensure_dynamic_smem(fn, smem, "gmm_kernel")) != VQMOE_OK)
        return s;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(mode == kSmall ? kSmallThreads : kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    void *params[5] = {&mx, &m0, &m1, const_cast<GmmArgs *>(&a), &p};
    if (cudaLaunchKernelExC(&cfg, fn, params) != cudaSuccess) return check_launch("gmm_kernel");
    return VQMOE_OK;
}

// -------------------------------------------------------------- quantizer

namespace gm {

// Eight lanes a group of 128, 16 values each; a thread has kQuantAhead groups'
// loads in flight (a row's bytes are read and written once: HBM-bound). The
// largest |bf16| by integer comparison of the bits: a NaN compares above an
// infinity, and both above every finite value.
constexpr int kQuantAhead = 2;
template <bool ORDER>
__global__ void __launch_bounds__(256)
    quantize_kernel(const uint16_t *__restrict__ x, uint32_t total, uint32_t groups, int cols, long long x_stride,
                    uint8_t *__restrict__ q, float *__restrict__ s, long long s_row, long long s_group,
                    const QuantOrder o) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 7;
    const uint32_t slots = gridDim.x * 32, slot = blockIdx.x * 32 + (threadIdx.x >> 3);
    // every lane of a warp makes the same trips (the shuffles need all of them)
    const uint32_t trips = (total + slots - 1) / slots;
    const int k = ORDER && !o.per_pair ? o.k : 1;
    // the places of pairs y0 .. y0 + 7 of a row (-1: no such expert, no place)
    auto places = [&](int (&at)[8], uint32_t row, int y0) {
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            const size_t p = (size_t)row * k + min(y0 + y, k - 1);
            const int rk = __ldg(o.rank + p), e = __ldg(o.inds + p);
            at[y] = y0 + y < k && rk >= 0 ? __ldg(o.off + e) + rk : -1;
        }
    };
    for (uint32_t i0 = 0; i0 < trips; i0 += kQuantAhead) {
        uint4 v[kQuantAhead][2];
        uint32_t row[kQuantAhead];
        int c[kQuantAhead];
        bool in[kQuantAhead];
        int at[ORDER ? kQuantAhead : 1][8];
#pragma unroll
        for (int z = 0; z < kQuantAhead; ++z) {
            const uint32_t g = slot + (i0 + z) * slots;
            in[z] = i0 + z < trips && g < total;
            row[z] = in[z] ? g / groups : 0;
            c[z] = in[z] ? (int)(g - row[z] * groups) * kScaleBlock + lane * 16 : 0;
            v[z][0] = v[z][1] = make_uint4(0, 0, 0, 0);
            if (in[z] && c[z] < cols) {
                const uint4 *p = reinterpret_cast<const uint4 *>(x + row[z] * x_stride + c[z]);
                v[z][0] = __ldcs(p);
                v[z][1] = __ldcs(p + 1);
            }
            if (ORDER && in[z]) places(at[ORDER ? z : 0], row[z], 0);   // beside the values' own load
        }
#pragma unroll
        for (int z = 0; z < kQuantAhead; ++z) {
            const uint32_t w[8] = {v[z][0].x, v[z][0].y, v[z][0].z, v[z][0].w,
                                   v[z][1].x, v[z][1].y, v[z][1].z, v[z][1].w};
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
#pragma unroll
            for (int d = 4; d > 0; d >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, d));
            const QScale qs = qscale(max(m & 0xFFFFu, m >> 16));
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                b[j] = cvt_e4m3x2(quotient(bf_lo(w[2 * j]), qs), quotient(bf_hi(w[2 * j]), qs)) |
                       (cvt_e4m3x2(quotient(bf_lo(w[2 * j + 1]), qs), quotient(bf_hi(w[2 * j + 1]), qs)) << 16);
            if (!in[z]) continue;
            const uint4 r = make_uint4(b[0], b[1], b[2], b[3]);
            const bool live = c[z] < cols;
            const long long grp = c[z] / kScaleBlock;
            if (!ORDER) {
                if (live) *reinterpret_cast<uint4 *>(q + (size_t)row[z] * cols + c[z]) = r;
                if (lane == 0) s[row[z] * s_row + grp * s_group] = qs.s;
            } else {
                for (int y0 = 0; y0 < k; y0 += 8) {
                    int (&to)[8] = at[ORDER ? z : 0];
                    if (y0) places(to, row[z], y0);
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        if (to[y] < 0) continue;
                        if (live) *reinterpret_cast<uint4 *>(q + (size_t)to[y] * cols + c[z]) = r;
                        if (lane == 0) s[to[y] * s_row + grp * s_group] = qs.s;
                    }
                }
            }
        }
    }
}

}  // namespace gm

vqmoe_status launch_quantize_fp8(const void *x, long long rows, int cols, long long x_stride, uint8_t *q, float *s,
                                 long long s_row, long long s_group, const QuantOrder *order, cudaStream_t stream) {
    if (rows <= 0) return VQMOE_OK;
    const uint32_t groups = (cols + kScaleBlock - 1) / kScaleBlock;
    const long long total = rows * groups;
    if (total > 0x7FFFFFFFLL) return set_error(VQMOE_BAD_SHAPE, "quantize: %lld rows of %d", rows, cols);
    const int grid = (int)std::min<long long>((total + 31) / 32, (long long)sm_count() * 8);
    const uint16_t *xp = static_cast<const uint16_t *>(x);
    if (order) {
        if (launch_pdl(gm::quantize_kernel<true>, dim3(grid), dim3(256), 0, stream, xp, (uint32_t)total, groups, cols,
                       x_stride, q, s, s_row, s_group, *order) != cudaSuccess)
            return check_launch("quantize_kernel");
        return VQMOE_OK;
    }
    gm::quantize_kernel<false><<<grid, 256, 0, stream>>>(xp, (uint32_t)total, groups, cols, x_stride, q, s, s_row,
                                                         s_group, QuantOrder{});
    return check_launch("quantize_kernel");
}


// ---------------------------------------------- routed experts, C ABI

static size_t quantized_bytes(size_t rows, int in) {
    return align_up(rows * in, 256) + align_up(rows * ((in + kScaleBlock - 1) / kScaleBlock) * sizeof(float), 256);
}
size_t fp8_rows_bytes(int rows, int in) { return quantized_bytes((size_t)rows, in); }

static GmmArgs fp8_args(const RoutedIO &r, const vqmoe_linear *w0, const vqmoe_linear *w1, uint32_t *err) {
    GmmArgs a{};
    a.off = r.off;
    a.E = r.E;
    a.P = r.P;
    a.N = w0->out_features;
    a.KB = (w0->in_features + kScaleBlock - 1) / kScaleBlock;
    a.sw0 = static_cast<const float *>(w0->scales);
    a.sw1 = w1 ? static_cast<const float *>(w1->scales) : nullptr;
    a.err = err;
    return a;
}

// The routed experts with block-scaled e4m3 weights: the inputs quantized
// into expert order, gate/up with its activations quantized in the epilogue
// (r1, may be null), then w2. r1->out holds the quantized activations: I
// bytes and ceil(I / 128) floats a pair fit the 2 I bytes it has (I >= 16).
vqmoe_status launch_experts_fp8(const vqmoe_linear *gate, const vqmoe_linear *up, const RoutedIO *r1,
                                const vqmoe_linear *w2, const RoutedIO &r2, uint32_t *err, cudaStream_t stream,
                                cudaEvent_t after_permute) {
    const RoutedIO &in = r1 ? *r1 : r2;
    const vqmoe_linear *w = r1 ? gate : w2;
    const int P = in.P, IN = w->in_features;
    uint8_t *q = static_cast<uint8_t *>(in.xq);
    float *s = reinterpret_cast<float *>(q + align_up((size_t)P * IN, 256));
    const QuantOrder o{in.inds, in.rank, in.off, in.E, in.k, in.x_per_pair};
    vqmoe_status st = launch_quantize_fp8(in.x, in.x_per_pair ? P : P / in.k, IN, IN, q, s, 1, P, &o, stream);
    if (st != VQMOE_OK) return st;
    if (after_permute && cudaEventRecord(after_permute, stream) != cudaSuccess) return check_launch("event");
    if (r1) {
        GmmArgs a = fp8_args(*r1, gate, up, err);
        uint8_t *qa = static_cast<uint8_t *>(r1->out);
        float *sa = reinterpret_cast<float *>(qa + (size_t)P * a.N);
        a.sx = s;
        a.q_out = qa;
        a.s_out = sa;
        a.act = r1->act;
        if ((st = launch_gmm(q, IN, gate->weight, up->weight, IN, true, a, stream)) != VQMOE_OK) return st;
        q = qa;
        s = sa;
    }
    GmmArgs a = fp8_args(r2, w2, nullptr, err);
    a.sx = s;
    a.out = r2.out;
    a.out_stride = a.N;
    a.map = r2.list;
    a.row_scale = r2.pair_scale;
    return launch_gmm(q, w2->in_features, w2->weight, nullptr, w2->in_features, true, a, stream);
}

}  // namespace vqmoe

using namespace vqmoe;

extern "C" {

vqmoe_status vqmoe_quantize_fp8(const void *x, int64_t rows, int32_t cols, int64_t x_stride, void *q, float *scales,
                                void *stream) {
    if (rows < 0 || rows > (1LL << 31) - 1 || cols <= 0 || cols % 16 || x_stride < cols || x_stride % 8)
        return set_error(VQMOE_BAD_SHAPE,
                         "quantize_fp8: %lld rows of %d (a multiple of 16) at a pitch of %lld (a multiple of 8)",
                         (long long)rows, cols, (long long)x_stride);
    if (rows == 0) return VQMOE_OK;
    if (!x || !aligned16(x) || !q || !aligned16(q) || !scales)
        return set_error(VQMOE_BAD_POINTER, "quantize_fp8: x / q / scales null or not 16-byte aligned");
    const int groups = (cols + kScaleBlock - 1) / kScaleBlock;
    return launch_quantize_fp8(x, rows, cols, x_stride, static_cast<uint8_t *>(q), scales, groups, 1, nullptr,
                               static_cast<cudaStream_t>(stream));
}

size_t vqmoe_grouped_linear_workspace_size(const vqmoe_linear *w, int32_t rows) {
    if (!w || rows <= 0 || w->format != VQMOE_FMT_FP8_BLOCK || w->in_features <= 0) return 0;
    return quantized_bytes((size_t)rows, w->in_features);
}

vqmoe_status vqmoe_grouped_linear(const vqmoe_linear *w, const void *x, int32_t rows, int64_t x_stride,
                                  const int32_t *offsets, void *out, int32_t out_dtype, void *workspace,
                                  size_t workspace_bytes, uint32_t *status, void *stream) {
    vqmoe_status s = check_linear(w, "grouped_linear");
    if (s != VQMOE_OK) return s;
    const bool fp8 = w->format == VQMOE_FMT_FP8_BLOCK;
    if (!fp8 && w->format != VQMOE_FMT_DENSE_BF16)
        return set_error(VQMOE_BAD_FORMAT, "grouped_linear: format %d (bf16 or block-scaled e4m3)", w->format);
    const int E = w->num_experts, K = w->in_features, N = w->out_features;
    if (rows < 0 || rows > (1 << 26) || x_stride < K || x_stride % 8)
        return set_error(VQMOE_BAD_SHAPE, "grouped_linear: %d rows at a pitch of %lld", rows, (long long)x_stride);
    if (E > kMaxGroups) return set_error(VQMOE_BAD_SHAPE, "grouped_linear: %d groups (<= %d)", E, kMaxGroups);
    if (!offsets && E != 1) return set_error(VQMOE_BAD_POINTER, "grouped_linear: %d groups without offsets", E);
    if (out_dtype != VQMOE_OUT_BF16 && out_dtype != VQMOE_OUT_F32)
        return set_error(VQMOE_BAD_FORMAT, "grouped_linear: out_dtype %d", out_dtype);
    if (rows == 0) return VQMOE_OK;
    if (!x || !aligned16(x) || !out || !aligned16(out))
        return set_error(VQMOE_BAD_POINTER, "grouped_linear: x / out null or not 16-byte aligned");
    GmmArgs a{};
    a.off = offsets;
    a.E = E;
    a.P = rows;
    a.N = N;
    a.out = out;
    a.out_stride = N;
    a.out_f32 = out_dtype == VQMOE_OUT_F32;
    a.err = status;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!fp8) {
        a.KB = (2 * K + 127) / 128;
        return launch_gmm(x, (size_t)x_stride * 2, w->weight, nullptr, (size_t)K * 2, false, a, st);
    }
    const size_t need = vqmoe_grouped_linear_workspace_size(w, rows);
    if (!workspace || !aligned16(workspace))
        return set_error(VQMOE_BAD_POINTER, "grouped_linear: workspace null or not 16-byte aligned");
    if (workspace_bytes < need)
        return set_error(VQMOE_WORKSPACE_TOO_SMALL, "grouped_linear: workspace %zu < %zu bytes", workspace_bytes, need);
    uint8_t *q = static_cast<uint8_t *>(workspace);
    float *sx = reinterpret_cast<float *>(q + align_up((size_t)rows * K, 256));
    if ((s = launch_quantize_fp8(x, rows, K, x_stride, q, sx, 1, rows, nullptr, st)) != VQMOE_OK) return s;
    a.KB = (K + kScaleBlock - 1) / kScaleBlock;
    a.sx = sx;
    a.sw0 = static_cast<const float *>(w->scales);
    return launch_gmm(q, K, w->weight, nullptr, K, true, a, st, true);
}

}  // extern "C"
